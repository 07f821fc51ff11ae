"""GPU tests of attention on the fused QKV tensor (through the C ABI, llmq_amd.kernels) against the formulas in 64 bits.

Bars, with u = 2^-8 (half a step of a bf16 rounding, relative to the value).  Forward: the scores are fp32, each probability is
rounded to bf16 once (u of itself) and the result once more, so |err| <= u |out| + u sum_k p |v| plus fp32 terms: scores of
head_dim products lose at most head_dim 2^-24 sum |q k| scale, which moves every probability by that factor, and the
exponential and the sums 2^-20 together.  Backward: with the forward's rounded out, D is off by u sum_d |dout out|; p and ds are
rounded once each, so  |err(dv)| <= u |dv| + u sum p |dout|;  |err(ds)| <= u |ds| + p (u sum_d |dout out|);  dq, dk from the sums
of those times |k|, |q|, plus one rounding of the result.  Each bar is computed from the data below (`bars`)."""
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
    ep = p * (U + w)
    bar_out = U * out.abs() * (1 + U) + mm(ep, v.abs())
    eds = ds.abs() * (U + w) + p * (1 + U) * (U * (do * out).abs().sum(-1, keepdim=True) + HD * 2.0 ** -23 * mm(do.abs(), v.abs().transpose(2, 3)))
    bars = [mm(eds, k.abs()) * scale, heads(mm(eds.transpose(2, 3), q.abs())) * scale, heads(mm(ep.transpose(2, 3), do.abs()))]
    bars = [b + U * (1 + U) * y.abs() for b, y in zip(bars, grads)]
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
