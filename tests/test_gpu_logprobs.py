"""GPU tests of token_logprobs and its gradient (through the C ABI, llmq_amd.kernels) against the formulas in 64 bits.

Bars.  lse = r + ln s: d = (x - r) log2 e is off by 2 roundings of |d| 2^-24, a term by that and the exponential's ulp (2^-22),
terms far below the reference weigh nothing, and V terms are summed in chains of at most V / 256 + 20 fp32 additions: with
|d| <= 60 where it matters, the relative error of s is below 60 2^-22 + (V / 256 + 20) 2^-24 =: ES, and lse and logp are off by
ES + 2^-23 (|lse| + |x|).  entropy adds the same relative error of sum p (x - r), whose terms are at most 60: 61 ES + 2^-22.  The gradient is rounded once to
its type (u = 2^-8 for bf16, 2^-24 for fp32) and off by the relative error of p, (|x - lse| + 4) 2^-23 + the error of the given
lse (taken as given), times |dlogp| + |dentropy| (|x - lse| + entropy + 1), where |x - lse| <= 90 if p is not 0 in fp32."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from llmq_amd import kernels
    return kernels


def make(N, V, P, dtype, seed=0, std=3.0, banned=0.0):
    g = torch.Generator(device="cuda").manual_seed(N * 7 + V + seed)
    x = torch.randn((N, P), device="cuda", generator=g) * std
    t = torch.randint(0, V, (N,), device="cuda", generator=g, dtype=torch.int32)
    x.scatter_add_(1, t.long()[:, None], torch.full((N, 1), 7.0, device="cuda"))
    if banned:
        x.masked_fill_(torch.rand((N, P), device="cuda", generator=g) < banned, -math.inf)
        x.scatter_(1, t.long()[:, None], 1.0)
    if N > 3:
        t[1], t[2], t[3] = -100, V, -1
    return x.to(dtype), t


def forward(K, x, t, V, k=0, entropy=True):
    N = x.shape[0]
    new = lambda *s: torch.full(s, float("nan"), device="cuda")  # noqa: E731
    logp, lse, ent = new(N), new(N), new(N) if entropy else None
    top, ids = (new(N, k), torch.full((N, k), -7, dtype=torch.int32, device="cuda")) if k else (None, None)
    size = K.get_token_logprobs_scratch_size(N, V, k)
    scratch = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    K.token_logprobs(logp, ent, lse, top, ids, x, t, scratch[:size] if size else None, V)
    assert bool((scratch[size:] == 0xFF).all())
    return logp, ent, lse, top, ids


def exact(x, t, V):
    x = x[:, :V].double()
    lse = torch.logsumexp(x, 1)
    given = (t >= 0) & (t < V)
    xt = x.gather(1, torch.where(given, t, 0).long()[:, None])[:, 0]
    d = x - lse[:, None]
    p = d.exp()
    ent = -torch.where(p > 0, p * d, 0.0).sum(1)
    return torch.where(given, xt - lse, 0.0), ent, lse, xt, given, p, d


def es(V):
    return 60 * 2.0 ** -22 + (V / 256 + 20) * 2.0 ** -24


def check_forward(K, x, t, V, k):
    logp, ent, lse, top, ids = forward(K, x, t, V, k)
    elogp, eent, else_, xt, given, _, _ = exact(x, t, V)
    bar = es(V) + 2.0 ** -23 * (else_.abs() + xt.abs())
    assert ((lse - else_).abs() <= bar).all()
    assert ((logp - elogp).abs()[given] <= bar[given]).all() and (logp[~given] == 0).all()
    assert ((ent - eent).abs() <= 61 * es(V) + 2.0 ** -22 * (1 + eent)).all()
    if k:
        val, at = torch.sort(x[:, :V].float(), dim=1, descending=True, stable=True)
        n = min(k, V)
        assert torch.equal(ids[:, :n], at[:, :n].int())
        want = val[:, :n] - lse[:, None]
        assert torch.equal(top[:, :n], want)                        # one fp32 subtraction
        assert (ids[:, n:] == -1).all() and (top[:, n:] == -math.inf).all()
    return logp, ent, lse


# (N, V, P): one logit, odd sizes, rows that begin anywhere in a granule, split rows (few rows, long) and whole ones
SHAPES = [(1, 1, 1), (3, 2, 5), (5, 63, 63), (4, 64, 64), (7, 1000, 1001), (2, 4097, 4099), (1, 50257, 50257), (9, 32001, 32003),
          (1100, 517, 520), (1025, 4100, 4100), (1, 151936, 151936), (40, 131072, 131072)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_logprobs_match_the_formulas(K, shape, dtype):
    N, V, P = shape
    x, t = make(N, V, P, dtype)
    for k in (0, 1, 7, 32):
        check_forward(K, x, t, V, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_top_tokens_of_rows_with_ties_and_orders(K, dtype):
    """Equal logits go by token, whatever lane, granule or share of the row holds them."""
    V = 70001
    i = torch.arange(V, device="cuda")
    rows = [torch.zeros(V, device="cuda"),                                   # all equal
            (i // 16).float() % 256,                                         # rising steps, exact in bf16
            (255 - (i // 300) % 256).float(),                                # falling steps
            (i % 2048 == 5).float() + (i % 4096 == 4101).float(),            # one lane holds all the large ones
            torch.where(i % 2048 < 8, 200.0 - (i // 2048) % 100, 0.0),       # a lane with many large granules
            torch.where(i == 69999, -0.0, torch.where(i < 30, -1.0, 0.0)),   # both zeros
            torch.where(i % 3 == 0, -math.inf, -2.0),
            torch.where(i == 12345, 1.0, -math.inf)]
    for n in (1, 1200):                                                      # split rows, whole rows
        x = torch.stack(rows)[torch.arange(n, device="cuda") % 8 if n > 1 else slice(0, 8)].to(dtype)
        for k in (1, 5, 32):
            for part in (x, x[:, :64007].contiguous()):
                Vp = part.shape[1]
                _, _, lse, top, ids = forward(K, part, torch.zeros(len(part), dtype=torch.int32, device="cuda"), Vp, k)
                val, at = torch.sort(part[:8].float(), dim=1, descending=True, stable=True)
                val, at = val[:, :k].repeat(len(part) // 8, 1), at[:, :k].repeat(len(part) // 8, 1)
                assert torch.equal(ids, at.int())
                assert torch.equal(top, torch.where(val == -math.inf, val, val - lse[:, None]))


def test_top_tokens_of_rising_logits(K):
    """Logits that rise along the row: every later granule lies above any earlier bound."""
    V = 500009
    x = torch.arange(V, device="cuda").float()[None] / 1024
    for n in (1, 600):
        _, _, lse, top, ids = forward(K, x.repeat(n, 1), torch.full((n,), 3, dtype=torch.int32, device="cuda"), V, 32)
        assert torch.equal(ids, (V - 1 - torch.arange(32, device="cuda", dtype=torch.int32)).expand(n, 32))
        assert torch.equal(top, x[:, -32:].flip(1) - lse[:, None])


def test_top_tokens_when_the_chosen_lanes_hold_too_many(K):
    """More logits between the bound and the k-th best than the list holds: one lane's granules large in every turn."""
    V = 8 * 256 * 200
    i = torch.arange(V, device="cuda")
    lane = (i // 8) % 256
    x = torch.where(lane < 31, 100.0 + (i % 8), torch.where(lane == 40, 50.0, 0.0))
    x[(i == V - 1)] = 101.0
    x = x[None].repeat(1030, 1).to(torch.bfloat16)
    val, at = torch.sort(x[:1].float(), dim=1, descending=True, stable=True)
    _, _, lse, top, ids = forward(K, x, torch.zeros(1030, dtype=torch.int32, device="cuda"), V, 32)
    assert torch.equal(ids, at[:, :32].int().expand(1030, 32)) and torch.equal(top, val[:, :32] - lse[:, None])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n", [2, 1300])
def test_rows_of_masks_and_non_finite_logits(K, dtype, n):
    V, P = 9001, 9003
    lowest = torch.finfo(dtype).min
    for name in ("empty", "lowest", "one lowest", "nan", "inf", "half"):
        x, t = make(n, V, P, dtype, seed=3)
        x[:, V:] = math.nan                                                  # the padded columns are not looked at
        t[:] = 17
        if name == "empty":
            x[0, :V] = -math.inf
        elif name == "lowest":
            x[0, :V] = lowest
        elif name == "one lowest":
            x[0, :V] = -math.inf
            x[0, 8000] = lowest
        elif name == "nan":
            x[0, 4000] = math.nan
        elif name == "inf":
            x[0, 4000] = math.inf
        else:
            x[0, :4500] = lowest
        logp, ent, lse, top, ids = forward(K, x, t, V, 4)
        assert torch.isfinite(torch.stack([logp[1:], ent[1:], lse[1:]])).all() and torch.isfinite(top[1:]).all()
        row = (logp[0].item(), ent[0].item(), lse[0].item())
        if name == "empty":
            assert row == (-math.inf, 0.0, -math.inf) and (top[0] == -math.inf).all() and ids[0].tolist() == [0, 1, 2, 3]
        elif name == "lowest":
            assert row[0] == 0 and row[2] == lowest and abs(row[1] - math.log(V)) < 1e-4 and ids[0].tolist() == [0, 1, 2, 3]
        elif name == "one lowest":
            assert row == (-math.inf, 0.0, lowest) and ids[0].tolist() == [8000, 0, 1, 2] and top[0, 0] == 0
        elif name in ("nan", "inf"):
            assert all(math.isnan(v) for v in row)
        else:
            check_forward(K, x[:, :V].contiguous(), t, V, 4)
        grad = torch.full_like(x, 7.0)
        ones = torch.ones(n, device="cuda")
        K.token_logprobs_backward(grad, ones, ones, x, t, lse, ent, None, V)
        assert (grad[:, V:] == 0).all() and torch.isfinite(grad[1:]).all()
        if name == "empty":
            assert (grad[0] == 0).all()
        if name in ("nan", "inf"):
            assert torch.isnan(grad[0, 4000])
            am = torch.zeros(1, device="cuda")                               # no gradient enters: zeros, whatever the row holds
            ones[0] = 0
            K.token_logprobs_backward(grad, ones, ones, x, t, lse, ent, am, V)
            assert (grad[0] == 0).all() and math.isfinite(am.item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2, 5), (5, 63, 63), (7, 1000, 1001), (2, 4097, 4099), (300, 517, 520), (3, 50257, 50257),
                                   (2, 151936, 151936)])
@pytest.mark.parametrize("entropy", [False, True])
def test_gradient_matches_the_formula(K, shape, dtype, entropy):
    N, V, P = shape
    x, t = make(N, V, P, dtype, banned=0.2 if V > 10 else 0.0)
    _, ent, lse, _, _ = forward(K, x, t, V)
    g = torch.Generator(device="cuda").manual_seed(5)
    dlogp, dent = (torch.randn(N, device="cuda", generator=g) for _ in range(2))
    lse64, ent64 = lse.double(), ent.double()
    given = (t >= 0) & (t < V)
    d = x[:, :V].double() - lse64[:, None]
    p = d.exp()
    gl = torch.where(given, dlogp.double(), 0.0)[:, None]
    h = dent.double()[:, None] if entropy else torch.zeros((N, 1), device="cuda", dtype=torch.float64)
    want = -gl * p - h * torch.where(p > 0, p * (d + ent64[:, None]), 0.0)
    want.scatter_add_(1, torch.where(given, t, 0).long()[:, None], gl)
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    far = d.abs().clamp_max(90)
    bar = want.abs() * u + p * ((far + 8) * 2.0 ** -22) * (gl.abs() + h.abs() * (far + ent64[:, None] + 1)) + 2.0 ** -23 * gl.abs() * p + 1e-36
    got = torch.full((N, P), float("nan"), dtype=dtype, device="cuda")
    am = torch.full((1,), 9e9, device="cuda")
    K.token_logprobs_backward(got, dlogp, dent if entropy else None, x, t, lse, ent if entropy else None, am, V)
    assert ((got[:, :V].double() - want).abs() <= bar * (1 + u)).all() and (got[:, V:] == 0).all()
    ref = torch.zeros(1, device="cuda")
    K.abs_max(ref, got)
    assert am.item() == ref.item()
    K.token_logprobs_backward(x, dlogp, dent if entropy else None, x, t, lse, ent if entropy else None, None, V)     # in place
    assert torch.equal(x, got)


def test_gradient_against_differences(K):
    """The loss sum(c logp + h entropy) of fp32 logits, stepped along random directions, in 64 bits."""
    N, V = 6, 4001
    x, t = make(N, V, V, torch.float32, std=1.5)
    g = torch.Generator(device="cuda").manual_seed(8)
    c, h = (torch.randn(N, device="cuda", generator=g) for _ in range(2))
    _, ent, lse, _, _ = forward(K, x, t, V)
    grad = torch.empty_like(x)
    K.token_logprobs_backward(grad, c, h, x, t, lse, ent, None, V)

    def loss(y):
        logp, e, *_ = exact(y, t, V)
        return (c * logp + h * e).sum().item()

    for _ in range(3):
        step = torch.randn((N, V), device="cuda", generator=g, dtype=torch.float64)
        eps = 1e-4
        diff = (loss(x.double() + eps * step) - loss(x.double() - eps * step)) / (2 * eps)
        # central differences: eps^2 / 6 of a third derivative of order sum |step|^3 p; fp32 roundings of the gradient
        assert abs(diff - (grad.double() * step).sum().item()) <= 1e-5 * (1 + grad.abs().double().mul(step.abs()).sum().item())


def test_results_repeat_and_streams_and_graphs_agree(K):
    """The same bits from call to call, on another stream, and from every replay of captured calls that share their scratch, with
    the program's own work on the same tensors between the replays."""
    for N, V, k in ((1, 70001, 20), (2, 4100, 0), (700, 1003, 5)):
        x, t = make(N, V, V, torch.bfloat16)
        data = x.clone()
        side = torch.cuda.Stream()
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        logp, ent, lse, grad, am = new(N), new(N), new(N), torch.empty_like(x), new(1)
        top, ids = (new(N, k), torch.empty((N, k), dtype=torch.int32, device="cuda")) if k else (None, None)
        scratch = torch.empty(K.get_token_logprobs_scratch_size(N, V, k) + 16, dtype=torch.uint8, device="cuda")
        ones = torch.ones(N, device="cuda")

        def step():
            K.token_logprobs(logp, ent, lse, top, ids, x, t, scratch, V)
            K.token_logprobs_backward(grad, ones, ones, x, t, lse, ent, am, V)

        step()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for g in graphs:
            with torch.cuda.graph(g):
                step()
        for turn in range(4):
            x.copy_(data if turn % 2 == 0 else data * 0.5)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                want = [y for y in forward(K, x, t, V, k) if y is not None]
                dx = torch.empty_like(x)
                K.token_logprobs_backward(dx, ones, ones, x, t, want[2], want[1], None, V)
            torch.cuda.current_stream().wait_stream(side)
            for y in (logp, ent, lse, grad, am):
                y.fill_(math.nan)
            scratch.fill_(0xFF)
            graphs[turn // 2].replay()
            got = [y for y in (logp, ent, lse, top, ids) if y is not None]
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(grad, dx)
            assert am.item() == grad.abs().max().item()
            step()
            assert torch.equal(grad, dx)


def test_logits_of_more_than_four_gibibytes(K):
    """The last rows of logits that pass 2^32 bytes equal the same rows alone, bit for bit (a row is summed by one workgroup from
    256 rows on)."""
    N, V, tail = 15000, 151936, 600
    x = torch.zeros((N, V), dtype=torch.bfloat16, device="cuda")
    part, t1 = make(tail, V, V, torch.bfloat16)
    x[-tail:] = part
    t = torch.zeros(N, dtype=torch.int32, device="cuda")
    t[-tail:] = t1
    got, want = forward(K, x, t, V, 3), forward(K, part, t1, V, 3)
    assert all(torch.equal(a[-tail:], b) for a, b in zip(got, want))
    assert torch.allclose(got[2][:-tail], torch.full((), math.log(V), device="cuda"), rtol=1e-6, atol=0)
    ones = torch.ones(N, device="cuda")
    dpart = torch.empty_like(part)
    K.token_logprobs_backward(dpart, ones[:tail], ones[:tail], part, t1, want[2], want[1], None, V)
    K.token_logprobs_backward(x, ones, ones, x, t, got[2], got[1], None, V)
    assert torch.equal(x[-tail:], dpart)


def test_empty_calls(K):
    x, t = torch.empty((0, 9), device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    e, am = torch.empty(0, device="cuda"), torch.full((1,), 3.0, device="cuda")
    K.token_logprobs(e, e, e, None, None, x, t, None)
    K.token_logprobs_backward(x, e, e, x, t, e, e, am)
    assert am.item() == 0 and K.get_token_logprobs_scratch_size(0, 9, 4) == 0


def test_leading_dimensions_and_registered_operators(K):
    import llmq_amd.ops  # noqa: F401
    x, t = make(12, 1003, 1010, torch.bfloat16)
    want = forward(K, x, t, 1003, 3)
    x3, t3 = x.view(3, 4, 1010), t.view(3, 4)
    logp, ent, lse = (torch.empty((3, 4), device="cuda") for _ in range(3))
    top, ids = torch.empty((3, 4, 3), device="cuda"), torch.empty((3, 4, 3), dtype=torch.int32, device="cuda")
    torch.ops.llmq.token_logprobs(logp, ent, lse, top, ids, x3, t3, None, 1003)
    for a, b in zip((logp, ent, lse, top, ids), want):
        assert torch.equal(a.view(b.shape), b)
    g, g3, ones, am = torch.empty_like(x), torch.empty_like(x3), torch.ones((3, 4), device="cuda"), torch.zeros(1, device="cuda")
    K.token_logprobs_backward(g, ones.view(12), None, x, t, want[2], None, None, 1003)
    torch.ops.llmq.token_logprobs_backward(g3, ones, None, x3, t3, lse, None, am, 1003)
    assert torch.equal(g3.view(12, 1010), g) and am.item() == g.abs().max().item()


def test_nothing_is_written_behind_the_tensors(K):
    for dtype in (torch.bfloat16, torch.float32):
        N, V, P = 5, 1001, 1003
        x, t = make(N, V, P, dtype)
        _, ent, lse, _, _ = forward(K, x, t, V)
        buf = torch.full((N * P + 64,), 7.0, dtype=dtype, device="cuda")
        ones = torch.ones(N, device="cuda")
        K.token_logprobs_backward(buf[32:-32].view(N, P), ones, ones, x, t, lse, ent, None, V)
        assert (buf[:32] == 7).all() and (buf[-32:] == 7).all() and torch.isfinite(buf).all()
        outs = torch.full((6, N + 2), 7.0, device="cuda")
        top, ids = torch.full((N + 2, 4), 7.0, device="cuda"), torch.full((N + 2, 4), 7, dtype=torch.int32, device="cuda")
        K.token_logprobs(outs[0, 1:-1], outs[1, 1:-1], outs[2, 1:-1], top[1:-1], ids[1:-1], x, t, None, V)
        assert (outs[:3, 0] == 7).all() and (outs[:3, -1] == 7).all() and (outs[3:] == 7).all()
        assert (top[[0, -1]] == 7).all() and (ids[[0, -1]] == 7).all() and torch.equal(outs[2, 1:-1], lse)


def test_refusals_on_device_tensors(K):
    x, t = make(2, 70000, 70001, torch.bfloat16)
    x = x[:, :70000].contiguous()
    o = lambda *s: torch.zeros(s or (2,), device="cuda")  # noqa: E731
    ids = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    need = K.get_token_logprobs_scratch_size(2, 70000, 3)
    assert need > 0
    s = torch.empty(need, dtype=torch.uint8, device="cuda")
    logp, ent, lse, top = o(), o(), o(), o(2, 3)

    def refused(call, *a, **k):
        with pytest.raises(ValueError):
            call(*a, **k)

    f, b = K.token_logprobs, K.token_logprobs_backward
    refused(f, logp, ent, lse, top, ids, x.half(), t, s)
    refused(f, logp, ent, lse, top, ids, x.double(), t, s)
    refused(f, logp, ent, lse, top, ids, x, t.long(), s)
    refused(f, logp, ent, lse, top, ids, x, t[:1], s)
    refused(f, logp, ent, lse, top, None, x, t, s)
    refused(f, logp, ent, lse, top, ids[:, :2], x, t, s)
    refused(f, logp, ent, lse, o(2, 33), torch.zeros((2, 33), dtype=torch.int32, device="cuda"), x, t, s)
    refused(f, logp, ent, lse, top, ids, x, t, None)
    refused(f, logp, ent, lse, top, ids, x, t, s[:-16])
    refused(f, logp, ent, lse, top, ids, x, t, s, 70001)
    refused(f, logp, ent, lse, top, ids, x, t, s, 0)
    refused(f, logp, ent, lse, top, ids, x[:, ::2], t, s)
    refused(f, logp, ent, lse, top, ids, x[0], t, s)
    refused(f, None, ent, lse, top, ids, x, t, s)
    refused(f, logp.double(), ent, lse, top, ids, x, t, s)
    flat = torch.zeros(140001, dtype=torch.bfloat16, device="cuda")
    refused(f, logp, ent, lse, top, ids, flat[1:].view(2, 70000), t, s)
    d = torch.empty_like(x)
    refused(b, d[:1], logp, None, x, t, lse, None, None)
    refused(b, d, logp, ent, x, t, lse, None, None)
    refused(b, d.float(), logp, None, x, t, lse, None, None)
    refused(b, d, o(3), None, x, t, lse, None, None)
    refused(b, d, logp, None, x, t, lse, None, None, 70001)
    refused(b, flat[1:].view(2, 70000), logp, None, x, t, lse, None, None)
    assert all((y == 0).all() for y in (logp, ent, lse, top, ids))
