"""GPU tests of attention on finite scores of any size that fp32 holds.

Queries and keys have one dimension, powers of two times small whole numbers, so that scores are exact and the softmax is known:
one key a row, or a mean over equal keys.  Bars, with u = 2^-8 (half a step of bf16).  Forward: the chosen keys' probabilities are
equal but not always 1 before the division, so each is rounded by u: u mean |v|, and the mean by u: u |out|; sums and the keys that
weigh e^-64 at most are within T 2^-22 max |v|; lse is fp32: 2^-22 |lse| + 2^-20.  Backward, for the out and the targets it is given:
the exponent may be off by 2^-8 where lse is large, so p by 2^-8 ln 2, and rounded by u: 2^-7 in all of p and of ds; ds = p (dp - D) of
two fp32 sums of HD products each: HD 2^-22 sum |dout v|.  The other keys, 1.6e-28 at the nearest steps, add less than 1e-20."""
import math

import pytest
import torch

from test_gpu_attention import U, backward, exact, first_keys, forward, make

pytestmark = pytest.mark.gpu

SCALE = 0.125
SHAPES = [(2, 150, 4, 2, 64), (1, 250, 2, 1, 128), (1, 200, 3, 1, 40)]
# exponents of two of a step between scores; at the last q.k, before the scale, is 250 2^119 = 1.7e38 of the 3.4e38 that fp32 holds
STEPS = [6, 9, 12, 15, 20, 25, 30, 34, 50, 80, 116]


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from llmq_amd import kernels
    return kernels


def steps_of(number, step, shape):
    """qkv and dout whose scores are number[t] 2^step SCALE / 2^-3, with random values."""
    B, T, Nq, Nkv, HD = shape
    qkv, dout = make(*shape, seed=13)
    x = qkv.view(B, T, Nq + 2 * Nkv, HD)
    x[:, :, :Nq + Nkv] = 0
    x[:, :, :Nq, 1] = 2.0 ** (step // 2)
    x[:, :, Nq:Nq + Nkv, 1] = (number.float() * 2.0 ** (step - step // 2 + 3))[None, :, None]
    assert torch.equal(x[0, :, Nq, 1].float(), number.float() * 2.0 ** (step - step // 2 + 3))
    return qkv, dout, x


def chosen(number, first, B, T):
    """Truth values [B, T, T]: the keys with the largest score among those that the query may look at."""
    t = torch.arange(T, device="cuda")
    a = (t[None, :] <= t[:, None]).expand(B, T, T)
    if first is not None:
        a = a & (t[None, None, :] >= first.long()[:, :, None])
    s = number.double()[None, None].expand(B, T, T).masked_fill(~a, -math.inf)
    m = s.amax(-1, keepdim=True)
    return a & (s == m), m[..., 0]


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_largest_scores_share_and_the_rest_is_nothing(K, shape, step, sign):
    B, T, Nq, Nkv, HD = shape
    t = torch.arange(T, device="cuda")
    for number in (t // 2, -(t // 2), t % 3 - 5, torch.full_like(t, 201)):
        qkv, dout, x = steps_of(sign * number, step, shape)
        for first in (None, first_keys("docs", B, T)):
            c, top = chosen(sign * number, first, B, T)
            n = c.sum(-1)
            out, lse = forward(K, qkv, Nq, Nkv, first, SCALE)
            v = x[:, :, Nq + Nkv:].double().repeat_interleave(Nq // Nkv, 2).permute(0, 2, 1, 3).contiguous()
            mean = lambda y: (torch.matmul(c.double()[:, None].expand(B, Nq, T, T).contiguous(), y) / n[:, None, :, None]).permute(0, 2, 1, 3)  # noqa: E731
            want = mean(v)
            got = out.double().view(B, T, Nq, HD)
            assert ((got - want).abs() <= U * want.abs() + U * (1 + U) * mean(v.abs()) + T * 2.0 ** -22 * v.abs().amax()).all()
            elog = (top * 2.0 ** step + n.double().log())[:, None].expand(B, Nq, T)
            assert ((lse.double() - elog).abs() <= 2.0 ** -22 * elog.abs() + 2.0 ** -20).all()
            assert torch.isfinite(backward(K, qkv, dout, out, lse, Nq, Nkv, first, SCALE)).all()


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_gradient_where_one_key_has_all(K, shape, step, sign):
    """The last key of a row (rising scores) or its first one (falling) has all of the probability."""
    B, T, Nq, Nkv, HD = shape
    G = Nq // Nkv
    number = torch.arange(T, device="cuda") + 1
    for number in (number, -number):
        qkv, dout, x = steps_of(sign * number, step, shape)
        for first in (None, first_keys("docs", B, T)):
            c, _ = chosen(sign * number, first, B, T)
            out, lse = forward(K, qkv, Nq, Nkv, first, SCALE)
            got = backward(K, qkv, dout, out, lse, Nq, Nkv, first, SCALE).double().view(B, T, Nq + 2 * Nkv, HD)
            do = dout.double().view(B, T, Nq, HD).permute(0, 2, 1, 3)
            v = x[:, :, Nq + Nkv:].double().repeat_interleave(G, 2).permute(0, 2, 1, 3).contiguous()
            back = c.double().transpose(1, 2)[:, None].expand(B, Nq, T, T).contiguous()           # [key, query]
            heads = lambda y: y.view(B, Nkv, G, T, -1).sum(2).permute(0, 2, 1, 3)  # noqa: E731
            dv, adv = heads(torch.matmul(back, do.contiguous())), heads(torch.matmul(back, do.abs().contiguous()))
            assert ((got[:, :, Nq + Nkv:] - dv).abs() <= U * dv.abs() + (2.0 ** -7 + T * G * 2.0 ** -23) * adv + 1e-20).all()
            at = c.double()[:, None].expand(B, Nq, T, T).contiguous()
            vc = torch.matmul(at, v)                                                              # the chosen key's value
            ds = (do * (vc - out.double().view(B, T, Nq, HD).permute(0, 2, 1, 3))).sum(-1, keepdim=True)
            eds = 2.0 ** -7 * ds.abs() + (1 + 2.0 ** -7) * HD * 2.0 ** -22 * (do * vc).abs().sum(-1, keepdim=True)
            kx = x[:, :, Nq:Nq + Nkv].double().repeat_interleave(G, 2).permute(0, 2, 1, 3).contiguous()
            qx = x[:, :, :Nq].double().permute(0, 2, 1, 3)
            kc = torch.matmul(at, kx)
            dq, edq = ((y * SCALE).permute(0, 2, 1, 3) for y in (ds * kc, eds * kc.abs()))
            dk, edk = (heads(torch.matmul(back, y.contiguous())) * SCALE for y in (ds * qx, (eds + T * G * 2.0 ** -23 * ds.abs()) * qx.abs()))
            for y, want, e in ((got[:, :, :Nq], dq, edq), (got[:, :, Nq:Nq + Nkv], dk, edk)):
                assert ((y - want).abs() <= U * want.abs() + (1 + U) * e + 1e-20).all()


@pytest.mark.parametrize("size", [10, 20, 30, 34, 60, 100, 123])
@pytest.mark.parametrize("shape", SHAPES)
def test_very_negative_scores_before_ordinary_ones(K, shape, size):
    """The first keys' scores are all about -201 / 128 2^size, the others' ordinary: rows that see both are those of the later keys alone."""
    B, T, Nq, Nkv, HD = shape
    cut = 100
    qkv, dout = make(*shape, seed=17)
    x = qkv.view(B, T, Nq + 2 * Nkv, HD)
    x[:, :, :Nq, 1] = 2.0 ** (size // 2)
    x[:, :, Nq:Nq + Nkv, 1] = 0
    x[:, :cut, Nq:Nq + Nkv, 1] = -201 * 2.0 ** (size - size // 2 + 3 - 7)
    out, lse = forward(K, qkv, Nq, Nkv, None, SCALE)
    dqkv = backward(K, qkv, dout, out, lse, Nq, Nkv, None, SCALE).double().view(B, T, Nq + 2 * Nkv, HD)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all() and torch.isfinite(dqkv).all()
    assert ((lse[..., :cut].double() + 201 * 2.0 ** (size - 7)).abs() <= 2.0 ** -20 * 2.0 ** size + 64).all()
    plain = qkv.clone()                      # the same for the later keys, whose dimension 1 is 0
    plain.view(x.shape)[:, :, :Nq, 1] = 1.0
    first = torch.full((B, T), cut, dtype=torch.int32, device="cuda")
    e = exact(plain, dout, Nq, Nkv, first, SCALE)
    rows = slice(cut, T)
    assert ((out.double() - e["out"]).abs() <= e["bar_out"] + 1e-30)[:, rows].all()
    assert ((lse.double() - e["lse"]).abs() <= e["bar_lse"] + 2.0 ** -22 * e["lse"].abs())[..., rows].all()
    grad, bar = (e[n].view(B, T, Nq + 2 * Nkv, HD)[:, rows].clone() for n in ("grad", "bar_grad"))
    for y in (grad, bar):
        y[:, :, Nq:Nq + Nkv, 1] *= 2.0 ** (size // 2)
    assert ((dqkv[:, rows] - grad).abs() <= bar + 1e-30).all()


def test_scores_of_every_size_in_one_row(K):
    """A row's reference follows scores from -8e37 to 8e37 over both forms of the exponent."""
    for HD in (64, 128):
        T = 240
        t = torch.arange(T, device="cuda", dtype=torch.float64)
        number = torch.sign(t - T / 2 + 0.5) * 2.0 ** ((t - T / 2 + 0.5).abs() - 0.5)     # exact in bf16, -2^119 .. 2^119
        qkv, dout = make(1, T, 2, 1, HD, seed=2)
        x = qkv.view(1, T, 4, HD)
        x[:, :, :3] = 0
        x[:, :, :2, 1] = 8.0
        x[:, :, 2, 1] = number.to(torch.bfloat16)
        out, lse = forward(K, qkv, 2, 1, None, SCALE)
        s = number[None].expand(T, T).masked_fill(t[None, :] > t[:, None], -math.inf)
        want, el = torch.softmax(s, -1) @ x[0, :, 3].double(), torch.logsumexp(s, -1)
        assert ((out[0].double().view(T, 2, HD) - want[:, None]).abs() <= 3 * U * x[0, :, 3].double().abs().amax()).all()
        assert ((lse[0].double() - el).abs() <= 2.0 ** -22 * el.abs() + 2.0 ** -20).all()
        assert torch.isfinite(backward(K, qkv, dout, out, lse, 2, 1, None, SCALE)).all()


@pytest.mark.parametrize("shape", SHAPES)
def test_values_near_the_largest_of_their_type(K, shape):
    """A mean of values is no larger than they are: sums of probabilities that are not yet divided may not be either.  Bars of `exact`."""
    B, T, Nq, Nkv, HD = shape
    for first in (None, first_keys("docs", B, T)):
        for power in (100, 120, 124):
            qkv, dout = make(*shape, seed=19)
            x = qkv.view(B, T, Nq + 2 * Nkv, HD)
            x[:, :, Nq + Nkv:] *= 2.0 ** power
            assert torch.isfinite(qkv).all()
            e = exact(qkv, dout, Nq, Nkv, first)
            am, ref = torch.full((1,), 0.0, device="cuda"), torch.zeros(1, device="cuda")
            out, lse = forward(K, qkv, Nq, Nkv, first, None, am)
            assert ((out.double() - e["out"]).abs() <= e["bar_out"]).all()
            assert ((lse.double() - e["lse"]).abs() <= e["bar_lse"] + 2.0 ** -22 * e["lse"].abs()).all()
            K.abs_max(ref, out)
            assert torch.equal(am, ref)
