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
