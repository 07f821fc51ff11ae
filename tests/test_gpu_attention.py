"""GPU tests of attention on the fused QKV tensor (through the C ABI, llmq_amd.kernels) against the formulas in 64 bits.

Bars, with u = 2^-8 (half a step of a bf16 rounding, relative to the value).  Forward: the scores are fp32, each probability is
rounded to bf16 once (u of itself) and the result once more, so |err| <= u |out| + u sum_k p |v| plus fp32 terms: scores of
head_dim products lose at most head_dim 2^-24 sum |q k| scale, which moves every probability by that factor, and the
exponential and the sums 2^-20 together.  Backward: D comes from the forward's out, so it is off by sum_d |dout| err(out); p and ds
are rounded once each, so  |err(dv)| <= u |dv| + u sum p |dout|;  |err(ds)| <= u |ds| + p err(D);  dq, dk from the sums of those
times |k|, |q|, plus one rounding of the result.  Each bar is computed from the data below (`bars`), with the products of errors:
the rounding of a value that is off by e is off by u (|x| + e)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from llmq_amd import kernels
    return kernels


def make(B, T, Nq, Nkv, HD, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(1000 * T + HD + seed)
    qkv = (torch.randn((B, T, (Nq + 2 * Nkv) * HD), device="cuda", generator=g) * std).to(torch.bfloat16)
    dout = torch.randn((B, T, Nq * HD), device="cuda", generator=g).to(torch.bfloat16)
    return qkv, dout


def first_keys(kind, B, T):
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    if kind == "none":
        return None
    if kind == "window":
        f = (t - 36).expand(B, T)                      # negative values count as 0
    elif kind == "docs":
        f = torch.stack([(t // (37 + 64 * b)) * (37 + 64 * b) for b in range(B)])
    elif kind == "ones":
        f = t.expand(B, T)                             # every token a document
    elif kind == "pad":
        pad = min(T, 33)
        f = torch.where(t < pad, torch.full_like(t, 2 ** 31 - 1), torch.full_like(t, pad)).expand(B, T)
    elif kind == "empty":
        f = (t + 1).expand(B, T)
    elif kind == "mixed":                              # not monotone, some rows empty
        g = torch.Generator(device="cuda").manual_seed(T)
        f = torch.randint(-5, T + 3, (B, T), device="cuda", generator=g, dtype=torch.int32)
    return f.contiguous()


def allowed_of(first, B, T):
    t = torch.arange(T, device="cuda")
    a = (t[None, :] <= t[:, None]).expand(B, T, T)
    return a if first is None else a & (t[None, None, :] >= first.long()[:, :, None])


def exact(qkv, dout, Nq, Nkv, first, scale=None):
    """The formulas in 64 bits, and the bars of the header."""
    B, T, C = qkv.shape
    HD, G = C // (Nq + 2 * Nkv), Nq // Nkv
    scale = HD ** -0.5 if scale is None else scale
    x = qkv.double().view(B, T, Nq + 2 * Nkv, HD).permute(0, 2, 1, 3)
    q, k, v = x[:, :Nq], x[:, Nq:Nq + Nkv].repeat_interleave(G, 1), x[:, Nq + Nkv:].repeat_interleave(G, 1)
    do = dout.double().view(B, T, Nq, HD).permute(0, 2, 1, 3)
    mask = allowed_of(first, B, T)[:, None]
    mm = lambda a, b: torch.matmul(a.contiguous(), b.contiguous())  # noqa: E731
    s = (mm(q, k.transpose(2, 3)) * scale).masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    out = mm(p, v)
    dp = mm(do, v.transpose(2, 3))
    D = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - D)
    heads = lambda y: y.view(B, Nkv, G, T, HD).sum(2)  # noqa: E731
    grads = [mm(ds, k) * scale, heads(mm(ds.transpose(2, 3), q)) * scale, heads(mm(p.transpose(2, 3), do))]
    # bars.  w: relative change of a probability by the fp32 evaluation of its score, its row's lse and the exponential
    w = (HD * 2.0 ** -24 * scale * mm(q.norm(dim=-1, keepdim=True), k.norm(dim=-1, keepdim=True).transpose(2, 3)) + 2.0 ** -18)
    w = torch.where(mask, w + w.masked_fill(~mask, 0).amax(-1, keepdim=True), 0.0)
    # a rounding is one of the value with its errors so far: u (|x| + e), so e becomes e (1 + u) + u |x|
    ep = p * (w * (1 + U) + U)
    bar_out = mm(ep, v.abs()) * (1 + U) + U * out.abs()
    eds = ds.abs() * (w * (1 + U) + U) + p * (1 + w) * (1 + U) * ((do.abs() * bar_out).sum(-1, keepdim=True) + HD * 2.0 ** -23 * mm(do.abs(), v.abs().transpose(2, 3)))
    bars = [mm(eds, k.abs()) * scale, heads(mm(eds.transpose(2, 3), q.abs())) * scale, heads(mm(ep.transpose(2, 3), do.abs()))]
    bars = [b * (1 + U) + U * y.abs() for b, y in zip(bars, grads)]
    join = lambda ys: torch.cat([y.permute(0, 2, 1, 3) for y in ys], 2).reshape(B, T, C)  # noqa: E731
    flat = lambda y: y.permute(0, 2, 1, 3).reshape(B, T, Nq * HD)  # noqa: E731
    return dict(out=flat(out), lse=lse, grad=join(grads), bar_out=flat(bar_out), bar_lse=w.amax(-1), bar_grad=join(bars))


def forward(K, qkv, Nq, Nkv, first=None, scale=None, abs_max=None):
    B, T, C = qkv.shape
    HD = C // (Nq + 2 * Nkv)
    out = torch.full((B, T, Nq * HD), float("nan"), dtype=torch.bfloat16, device="cuda")
    lse = torch.full((B, Nq, T), float("nan"), device="cuda")
    K.attention_forward(out, lse, qkv, abs_max, Nq, Nkv, first, scale)
    return out, lse


def backward(K, qkv, dout, out, lse, Nq, Nkv, first=None, scale=None):
    B, T, C = qkv.shape
    size = K.get_attention_backward_scratch_size(B, T, Nq, Nkv, C // (Nq + 2 * Nkv))
    scratch = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    dqkv = torch.full_like(qkv, float("nan"))
    K.attention_backward(dqkv, dout, out, lse, qkv, scratch[:size], Nq, Nkv, first, scale)
    assert bool((scratch[size:] == 0xFF).all())
    return dqkv


def check(K, qkv, dout, Nq, Nkv, first=None, scale=None):
    e = exact(qkv, dout, Nq, Nkv, first, scale)
    am = torch.full((1,), 9e9, device="cuda")
    out, lse = forward(K, qkv, Nq, Nkv, first, scale, am)
    assert torch.isfinite(out).all()
    worst = ((out.double() - e["out"]).abs() / (e["bar_out"] + 1e-30)).max().item()
    assert worst <= 1, "out: %.3f of the bar" % worst
    empty = e["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    off = torch.where(empty, 0.0, (lse.double() - e["lse"]).abs() - e["bar_lse"] - 2.0 ** -22 * e["lse"].abs())
    assert off.max().item() <= 0
    ref = torch.zeros(1, device="cuda")
    K.abs_max(ref, out)
    assert am.item() == ref.item()
    dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first, scale)
    assert torch.isfinite(dqkv).all()
    worst = ((dqkv.double() - e["grad"]).abs() / (e["bar_grad"] + 1e-30)).max().item()
    assert worst <= 1, "dqkv: %.3f of the bar" % worst
    return out, lse, dqkv


# (B, T, Nq, Nkv, HD): one token, both sides of the 32 / 64 / 128 tiles, the head layouts of the 0.5B, 1.5B and 7B models
SHAPES = [(1, 1, 2, 1, 64), (1, 2, 1, 1, 128), (2, 31, 4, 2, 32), (1, 33, 3, 1, 8), (1, 40, 14, 2, 64), (2, 64, 2, 2, 128),
          (3, 65, 6, 3, 24), (1, 127, 4, 4, 80), (2, 128, 12, 2, 128), (1, 129, 28, 4, 128), (2, 200, 4, 1, 96), (1, 257, 14, 2, 64),
          (1, 700, 6, 2, 128), (2, 515, 4, 4, 64), (1, 1100, 7, 1, 64)]


@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_the_formulas(K, shape):
    B, T, Nq, Nkv, HD = shape
    qkv, dout = make(*shape)
    check(K, qkv, dout, Nq, Nkv)


@pytest.mark.parametrize("kind", ["window", "docs", "ones", "pad", "empty", "mixed"])
@pytest.mark.parametrize("shape", [(2, 1, 2, 1, 64), (2, 65, 4, 2, 64), (2, 300, 6, 2, 128), (1, 777, 4, 1, 40)])
def test_attention_masks(K, kind, shape):
    B, T, Nq, Nkv, HD = shape
    qkv, dout = make(*shape, seed=7)
    first = first_keys(kind, B, T)
    out, lse, dqkv = check(K, qkv, dout, Nq, Nkv, first)
    empty = (first.long().clamp_min(0) > torch.arange(T, device="cuda"))
    assert (out[empty] == 0).all() and (dqkv.view(B, T, Nq + 2 * Nkv, HD)[:, :, :Nq][empty] == 0).all()


@pytest.mark.parametrize("scale,std", [(0.3, 1.0), (1.0, 1.0), (0.02, 4.0), (None, 6.0)])
def test_attention_scales_and_large_scores(K, scale, std):
    for shape in ((2, 190, 4, 2, 64), (1, 333, 3, 1, 128)):
        qkv, dout = make(*shape, seed=3, std=std)
        check(K, qkv, dout, shape[2], shape[3], first_keys("docs", shape[0], shape[1]), scale)


def by_rows(qkv, dout, out, Nq, Nkv, first):
    """Outputs and gradients in 64 bits, a row of the probabilities at a time over the keys it may look at, so that nothing else
    can reach them.  `out`: the rounded outputs the backward pass is given."""
    B, T, C = qkv.shape
    HD, G = C // (Nq + 2 * Nkv), Nq // Nkv
    x, do, o = (y.double().cpu() for y in (qkv.view(B, T, -1, HD), dout.view(B, T, Nq, HD), out.view(B, T, Nq, HD)))
    f = torch.zeros((B, T), dtype=torch.long) if first is None else first.long().cpu().clamp_min(0)
    want, grad, scale = torch.zeros_like(o), torch.zeros_like(x), HD ** -0.5
    for b in range(B):
        for h in range(Nq):
            k, v = x[b, :, Nq + h // G], x[b, :, Nq + Nkv + h // G]
            for t in range(T):
                if f[b, t] > t:
                    continue
                a, q, g = slice(int(f[b, t]), t + 1), x[b, t, h], do[b, t, h]
                p = torch.softmax((k[a] * q).sum(1) * scale, 0)
                want[b, t, h] = (p[:, None] * v[a]).sum(0)
                ds = p * ((v[a] * g).sum(1) - (g * o[b, t, h]).sum())
                grad[b, t, h] = (ds[:, None] * k[a]).sum(0) * scale
                grad[b, a, Nq + h // G] += ds[:, None] * q * scale
                grad[b, a, Nq + Nkv + h // G] += p[:, None] * g
    return want.view(B, T, -1).cuda(), grad.view(B, T, C).cuda()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("shape", [(2, 150, 4, 2, 64), (1, 300, 2, 1, 128), (1, 200, 3, 1, 40)])
def test_values_that_are_not_finite_reach_what_they_enter_and_nothing_else(K, shape, value):
    """One such value in the second document, in a query, a key, a value or an output gradient: what the formulas keep finite is
    finite and within its bar, what they do not is not."""
    B, T, Nq, Nkv, HD = shape
    first = first_keys("docs", B, T)
    at = {"q": 1, "k": Nq, "v": Nq + Nkv}
    for name in ("q", "k", "v", "dout"):
        qkv, dout = make(*shape, seed=11)
        clean = exact(qkv, dout, Nq, Nkv, first)
        if name == "dout":
            dout.view(B, T, Nq, HD)[0, 80, Nq - 1, 5] = value
        else:
            qkv.view(B, T, -1, HD)[0, 80, at[name], 5] = value
        am, ref = torch.full((1,), 9e9, device="cuda"), torch.zeros(1, device="cuda")
        out, lse = forward(K, qkv, Nq, Nkv, first, None, am)
        K.abs_max(ref, out)
        assert torch.equal(am, ref)
        dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first)
        want, grad = by_rows(qkv, dout, out, Nq, Nkv, first)
        assert torch.equal(torch.isfinite(out), torch.isfinite(want)), name
        assert torch.equal(torch.isfinite(dqkv), torch.isfinite(grad)), name
        for got, ref, bar in ((out, clean["out"], clean["bar_out"]), (dqkv, clean["grad"], clean["bar_grad"])):
            other = torch.ones((B, T), dtype=torch.bool, device="cuda")
            other[0, 74:111] = False                                         # the document of the value
            assert ((got.double() - ref).abs() <= bar + 1e-30)[other].all(), name


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("shape", [(2, 300, 4, 2, 64), (1, 777, 2, 1, 128)])
def test_padding_may_hold_anything(K, shape, value):
    """Rows without keys, which nobody looks at: whatever their tensors hold, their results are zeros and the others' as ever."""
    B, T, Nq, Nkv, HD = shape
    first = first_keys("pad", B, T)
    qkv, dout = make(*shape, seed=5)
    e = exact(qkv, dout, Nq, Nkv, first)
    qkv[:, :33], dout[:, :33] = value, value
    out, lse = forward(K, qkv, Nq, Nkv, first)
    dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first)
    assert ((out.double() - e["out"]).abs() <= e["bar_out"] + 1e-30).all() and (out[:, :33] == 0).all()
    assert (lse[..., :33] == -math.inf).all()
    assert ((lse.double() - e["lse"]).abs() <= e["bar_lse"] + 2.0 ** -22 * e["lse"].abs())[..., 33:].all()
    assert ((dqkv.double() - e["grad"]).abs() <= e["bar_grad"] + 1e-30).all() and (dqkv[:, :33] == 0).all()


def test_rows_whose_scores_are_all_minus_infinity(K):
    qkv, _ = make(1, 3, 2, 1, 64)
    qkv.view(3, 4, 64)[:, :2, 0] = 1.0
    qkv.view(3, 4, 64)[:2, 2, 0] = -math.inf
    out, lse = forward(K, qkv, 2, 1)
    assert (out[0, :2] == 0).all() and (lse[0, :, :2] == -math.inf).all()
    assert torch.equal(out.view(3, 2, 64)[2], qkv.view(3, 4, 64)[2, 3:].expand(2, 64)) and torch.isfinite(lse[0, :, 2]).all()


def test_gradient_against_differences(K):
    """The loss sum(dout out) of the formulas in 64 bits, stepped along random directions; the kernel's gradient is off by its bars."""
    B, T, Nq, Nkv, HD = 1, 70, 4, 2, 64
    qkv, dout = make(B, T, Nq, Nkv, HD, seed=9)
    first = first_keys("window", B, T)
    out, lse = forward(K, qkv, Nq, Nkv, first)
    dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first).double()
    bar = exact(qkv, dout, Nq, Nkv, first)["bar_grad"]
    g = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(3):
        step = torch.randn(qkv.shape, device="cuda", generator=g, dtype=torch.float64)
        eps = 1e-5
        loss = [(exact(qkv.double() + e * step, dout, Nq, Nkv, first)["out"] * dout.double()).sum() for e in (eps, -eps)]
        diff = ((loss[0] - loss[1]) / (2 * eps)).item()
        # eps^2 times third derivatives of order 1e3 and 2^-52 of the loss over eps are far below the bars
        assert abs(diff - (dqkv * step).sum().item()) <= (bar * step.abs()).sum().item() + 1e-4


@pytest.mark.parametrize("shape", [(1, 1, 4, 2, 64), (2, 129, 14, 2, 64), (1, 700, 4, 1, 128)])
def test_results_repeat_and_streams_and_graphs_agree(K, shape):
    """The same bits from call to call, on another stream, and from every replay of a captured forward and backward pass, with
    the program's own work on the same tensors between the replays."""
    B, T, Nq, Nkv, HD = shape
    qkv, dout = make(*shape)
    first = first_keys("docs", B, T)
    out, lse = forward(K, qkv, Nq, Nkv, first)
    dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = forward(K, qkv, Nq, Nkv, first)
        d2 = backward(K, qkv, dout, o2, l2, Nq, Nkv, first)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o2, out) and torch.equal(l2, lse) and torch.equal(d2, dqkv)
    am = torch.zeros(1, device="cuda")
    scratch = torch.empty(K.get_attention_backward_scratch_size(B, T, Nq, Nkv, HD), dtype=torch.uint8, device="cuda")

    def step():
        K.attention_forward(o2, l2, qkv, am, Nq, Nkv, first)
        K.attention_backward(d2, dout, o2, l2, qkv, scratch, Nq, Nkv, first)

    step()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]                      # which share their scratch
    for g in graphs:
        with torch.cuda.graph(g):
            step()
    data = qkv.clone()
    for turn in range(4):
        qkv.copy_(data if turn % 2 == 0 else data * 0.5)
        want = forward(K, qkv, Nq, Nkv, first)
        want = (*want, backward(K, qkv, dout, *want, Nq, Nkv, first))
        o2.fill_(math.nan), d2.fill_(math.nan), scratch.fill_(0xFF), am.fill_(-1.0)
        graphs[turn // 2].replay()
        assert all(torch.equal(a, b) for a, b in zip((o2, l2, d2), want))
        assert am.item() == o2.abs().max().item()
        step()
        assert torch.equal(d2, want[2])


def test_nothing_is_written_behind_the_tensors(K):
    """Tensors that begin and end inside a larger buffer, of batches and lengths that do not fill a tile."""
    B, T, Nq, Nkv, HD = 2, 77, 4, 2, 24
    qkv, dout = make(B, T, Nq, Nkv, HD)
    want = forward(K, qkv, Nq, Nkv)
    want = (*want, backward(K, qkv, dout, *want, Nq, Nkv))
    bufs = [torch.full((y.numel() + 128,), 7.0, dtype=y.dtype, device="cuda") for y in want]
    inner = [b[64:-64].view(y.shape) for b, y in zip(bufs, want)]
    K.attention_forward(inner[0], inner[1], qkv, None, Nq, Nkv)
    scratch = torch.empty(K.get_attention_backward_scratch_size(B, T, Nq, Nkv, HD), dtype=torch.uint8, device="cuda")
    K.attention_backward(inner[2], dout, inner[0], inner[1], qkv, scratch, Nq, Nkv)
    for b, i, y in zip(bufs, inner, want):
        assert torch.equal(i, y) and (b[:64] == 7).all() and (b[-64:] == 7).all()


def test_tensors_of_more_than_four_gibibytes(K):
    """The last sequence of a batch whose tensors pass 2^32 bytes equals the same sequence alone: bit for bit forward and dq; dk
    and dv are summed in another split, which moves a bf16 result by one step at most (and fp32 roundings of sums near zero)."""
    B, T, Nq, Nkv, HD = 120, 4096, 28, 4, 128
    C = (Nq + 2 * Nkv) * HD
    one, g1 = make(1, T, Nq, Nkv, HD)
    qkv, dout = one.expand(B, T, C).contiguous(), g1.expand(B, T, Nq * HD).contiguous()
    qkv[:-1] *= 0.5
    first = (torch.arange(T, device="cuda", dtype=torch.int32) - 200).expand(B, T).contiguous()
    out, lse = forward(K, qkv, Nq, Nkv, first)
    dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first)
    o1, l1 = forward(K, one, Nq, Nkv, first[:1])
    d1 = backward(K, one, g1, o1, l1, Nq, Nkv, first[:1])
    assert torch.equal(out[-1], o1[0]) and torch.equal(lse[-1], l1[0]) and torch.equal(dqkv[-1, :, :Nq * HD], d1[0, :, :Nq * HD])
    a, b = dqkv[-1].float(), d1[0].float()
    assert ((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -14).all()


def test_empty_calls(K):
    am = torch.full((1,), 3.0, device="cuda")
    for B, T in ((0, 5), (2, 0)):
        qkv = torch.empty((B, T, 4 * 64), dtype=torch.bfloat16, device="cuda")
        out, lse = qkv[..., :128].contiguous(), torch.empty((B, 2, T), device="cuda")
        K.attention_forward(out, lse, qkv, am, 2, 1)
        assert am.item() == 0
        assert K.get_attention_backward_scratch_size(B, T, 2, 1, 64) == 0
        K.attention_backward(torch.empty_like(qkv), out, out, lse, qkv, torch.empty(0, dtype=torch.uint8, device="cuda"), 2, 1)


def test_refusals_on_device_tensors(K):
    B, T, Nq, Nkv, HD = 1, 8, 2, 1, 64
    qkv, dout = make(B, T, Nq, Nkv, HD)
    out, lse = forward(K, qkv, Nq, Nkv)
    size = K.get_attention_backward_scratch_size(B, T, Nq, Nkv, HD)
    scratch, first = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros((B, T), dtype=torch.int32, device="cuda")
    keep = out.clone(), lse.clone()

    def refused(call, *a, **k):
        with pytest.raises(ValueError):
            call(*a, **k)

    f, b = K.attention_forward, K.attention_backward
    refused(f, out, lse, qkv.half(), None, Nq, Nkv)
    refused(f, out, lse, qkv.float(), None, Nq, Nkv)
    refused(f, out, lse.double(), qkv, None, Nq, Nkv)
    refused(f, out[:, :7], lse, qkv, None, Nq, Nkv)
    refused(f, out, lse[..., :7], qkv, None, Nq, Nkv)
    refused(f, out, lse, qkv, None, 3, 2)
    refused(f, out, lse, qkv, None, 2, 0)
    refused(f, out, lse, qkv, None, Nq, Nkv, first.long())
    refused(f, out, lse, qkv, None, Nq, Nkv, first[0])
    refused(f, out, lse, qkv, None, Nq, Nkv, None, 0.0)
    refused(f, out, lse, qkv, None, Nq, Nkv, None, -1.0)
    refused(f, out, lse, qkv, None, Nq, Nkv, None, math.nan)
    refused(f, out, lse, qkv, None, Nq, Nkv, None, math.inf)
    refused(f, out, lse, qkv.cpu(), None, Nq, Nkv)
    refused(f, out, lse, torch.zeros((1, 8, 512), dtype=torch.bfloat16, device="cuda")[..., ::2], None, Nq, Nkv)
    wide = torch.zeros((1, 8, 4 * 136), dtype=torch.bfloat16, device="cuda")
    refused(f, wide[..., :272].contiguous(), lse, wide, None, 2, 1)                  # head_dim 136
    odd = torch.zeros((1, 8, 4 * 12), dtype=torch.bfloat16, device="cuda")
    refused(f, odd[..., :24].contiguous(), lse, odd, None, 2, 1)                     # head_dim 12
    flat = torch.zeros(qkv.numel() + 1, dtype=torch.bfloat16, device="cuda")
    refused(f, out, lse, flat[1:].view(qkv.shape), None, Nq, Nkv)                    # 2-byte aligned
    d = torch.empty_like(qkv)
    refused(b, d, dout, out, lse, qkv, scratch[:size - 16], Nq, Nkv)
    refused(b, d, dout, out, lse, qkv, scratch.new_empty(size + 1)[1:], Nq, Nkv)
    refused(b, d, dout, out, lse, qkv, None, Nq, Nkv)
    refused(b, qkv, dout, out, lse, qkv, scratch, Nq, Nkv)
    refused(b, d[:, :7], dout, out, lse, qkv, scratch, Nq, Nkv)
    refused(b, d, dout[:, :7], out, lse, qkv, scratch, Nq, Nkv)
    refused(b, d, dout, out, lse, qkv, scratch, Nq, Nkv, None, -0.5)
    assert torch.equal(out, keep[0]) and torch.equal(lse, keep[1])


def test_registered_operators(K):
    import llmq_amd.ops  # noqa: F401
    B, T, Nq, Nkv, HD = 2, 50, 4, 2, 64
    qkv, dout = make(B, T, Nq, Nkv, HD)
    first = first_keys("docs", B, T)
    for scale in (0.0, 0.2):
        out, lse = forward(K, qkv, Nq, Nkv, first, scale or None)
        dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, first, scale or None)
        o2, l2, d2, am = torch.empty_like(out), torch.empty_like(lse), torch.empty_like(qkv), torch.zeros(1, device="cuda")
        scratch = torch.empty(K.get_attention_backward_scratch_size(B, T, Nq, Nkv, HD), dtype=torch.uint8, device="cuda")
        torch.ops.llmq.attention_forward(o2, l2, qkv, am, Nq, Nkv, first, scale)
        torch.ops.llmq.attention_backward(d2, dout, o2, l2, qkv, scratch, Nq, Nkv, first, scale)
        assert torch.equal(o2, out) and torch.equal(l2, lse) and torch.equal(d2, dqkv) and am.item() == out.abs().max().item()
