"""GPU tests of token_logprobs on finite logits of any size: masks of -1e4 to -1e29 in place of -inf, rows with a common offset, one
very large logit.  Against the formulas in 64 bits on the stored logits, with the bars of test_gpu_logprobs: they follow from
exponents that are off by 2 |d| 2^-24, d = (x - r) log2 e, whatever the size of r; lse itself is fp32, so lse and logp carry
2^-23 (|lse| + |x|)."""
import math

import pytest
import torch

from test_gpu_logprobs import es, forward, make

pytestmark = pytest.mark.gpu
V, P = 9001, 9003


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from llmq_amd import kernels
    return kernels


def gradient_within_its_bar(K, x, t, lse, ent, entropy):
    N = x.shape[0]
    g = torch.Generator(device="cuda").manual_seed(5)
    dlogp, dent = (torch.randn(N, device="cuda", generator=g) for _ in range(2))
    given = (t >= 0) & (t < V)
    d = x[:, :V].double() - lse.double()[:, None]
    p = d.exp()
    gl = torch.where(given, dlogp.double(), 0.0)[:, None]
    h = dent.double()[:, None] if entropy else torch.zeros((N, 1), device="cuda", dtype=torch.float64)
    e64 = ent.double()[:, None]
    want = -gl * p - h * torch.where(p > 0, p * (d + e64), 0.0)
    want.scatter_add_(1, torch.where(given, t, 0).long()[:, None], gl)
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    far = d.abs().clamp_max(90)
    bar = want.abs() * u + p * ((far + 8) * 2.0 ** -22) * (gl.abs() + h.abs() * (far + e64 + 1)) + 2.0 ** -23 * gl.abs() * p + 1e-36
    got = torch.full_like(x, math.nan)
    K.token_logprobs_backward(got, dlogp, dent if entropy else None, x, t, lse, ent if entropy else None, None, V)
    assert ((got[:, :V].double() - want).abs() <= bar * (1 + u)).all() and (got[:, V:] == 0).all()


def exact(x, t):
    """The formulas in 64 bits of the logits less their largest: beside 1e20, 64 bits lose ln V too."""
    x = x[:, :V].double()
    m = x.amax(1)
    y = x - m[:, None]
    total = torch.logsumexp(y, 1)
    given = (t >= 0) & (t < V)
    at = torch.where(given, t, 0).long()[:, None]
    d = y - total[:, None]
    p = d.exp()
    ent = -torch.where(p > 0, p * d, 0.0).sum(1)
    return torch.where(given, d.gather(1, at)[:, 0], 0.0), ent, m + total, x.gather(1, at)[:, 0], given


def check(K, x, t):
    elogp, eent, else_, xt, given = exact(x, t)
    bar = es(V) + 2.0 ** -23 * (else_.abs() + xt.abs())
    val, at = torch.sort(x[:, :V].float(), dim=1, descending=True, stable=True)
    for k in (0, 4):
        for entropy in (False, True):
            logp, ent, lse, top, ids = forward(K, x, t, V, k, entropy)
            assert ((lse - else_).abs() <= bar).all()
            assert ((logp - elogp).abs()[given] <= bar[given]).all() and (logp[~given] == 0).all()
            if entropy:
                assert ((ent - eent).abs() <= 61 * es(V) + 2.0 ** -22 * (1 + eent)).all()
            if k:
                assert torch.equal(ids, at[:, :k].int()) and torch.equal(top, val[:, :k] - lse[:, None])
    for entropy in (False, True):
        gradient_within_its_bar(K, x, t, lse, ent, entropy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n", [2, 1300])                                     # split rows, whole rows
@pytest.mark.parametrize("mask", [-1e4, -65504.0, -1e8, -1e9, -1e10, -1e11, -1e12, -1e15, -1e20, -1e29, -1e30, -3e38])
def test_rows_masked_by_a_large_finite_value(K, dtype, n, mask):
    for where in ("all", "first half", "last half", "all but one", "a third"):
        x, t = make(n, V, P, dtype, seed=3)
        x[:, V:] = math.nan
        t[:] = 17
        if where == "all":
            x[0, :V] = mask
        elif where == "first half":
            x[0, :4500] = mask
            t[:] = 5000
        elif where == "last half":
            x[0, 4500:V] = mask
        elif where == "all but one":
            keep = x[0, 8000].clone()
            x[0, :V] = mask
            x[0, 8000] = keep
            t[:] = 8000
        else:
            g = torch.Generator(device="cuda").manual_seed(2)
            x[:, :V].masked_fill_(torch.rand((n, V), device="cuda", generator=g) < 1 / 3, mask)
        check(K, x, t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n", [2, 1300])
def test_rows_with_a_common_offset_and_single_large_logits(K, dtype, n):
    for offset in (1e2, -1e2, 1e3, -1e3, 4090.0, -4099.0, 1e5, -1e5, 1e7, -1e9):
        x, t = make(n, V, P, torch.float32, seed=9)
        check(K, (x + offset).to(dtype), t)
    for large in (1e4, 1e8, 1e10, 1e20, 1e29, 1e38):
        for at in (0, 3, 4000, V - 1):
            x, t = make(n, V, P, dtype, seed=4)
            x[0, at] = large
            t[0] = at
            check(K, x, t)
            x[0, :2000] = -large                                             # and masked ones beside it
            x[0, at] = large
            check(K, x, t)


def test_logits_that_rise_by_orders_of_magnitude(K):
    """The reference follows from -1e30 to 1e30 along a row, through both forms of the exponent, in every lane."""
    i = torch.arange(V, device="cuda", dtype=torch.float64)
    for sign in (1.0, -1.0):
        x = sign * torch.sign(i - V / 2) * 10.0 ** ((i - V / 2).abs() / 150.0)
        x = torch.cat([x, torch.full((P - V,), math.nan, device="cuda", dtype=torch.float64)]).float()
        for n in (1, 700):
            for dtype in (torch.float32, torch.bfloat16):
                y = x.expand(n, P).to(dtype).contiguous()
                check(K, y, torch.full((n,), V - 1 if sign > 0 else 0, dtype=torch.int32, device="cuda"))
