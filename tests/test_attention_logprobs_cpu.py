"""What attention and the token log probabilities refuse and how much scratch they ask for, without a GPU: the library checks
every argument before it touches the device."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def capi():
    from llmq_amd import capi
    return capi


@pytest.fixture(scope="module")
def p():
    buf = (C.c_char * (1 << 20))()   # never read: every call below is refused or empty
    p.buf = buf
    return (C.addressof(buf) + 15) & ~15


def test_attention_forward_refuses(capi, p):
    f = capi.lib.llmq_attention_forward_bf16

    def rc(out=p, lse=p + 8192, qkv=p + 16384, first=None, am=None, scale=0.125, B=1, T=8, Nq=4, Nkv=2, HD=64):
        return f(out, lse, qkv, first, am, scale, B, T, Nq, Nkv, HD, None)

    bad = [dict(out=None), dict(lse=None), dict(qkv=None), dict(out=p + 2), dict(qkv=p + 8), dict(out=p + 16384), dict(out=p + 24560),
           dict(out=p + 12320), dict(lse=p + 4080), dict(lse=p + 16380), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=float("nan")), dict(scale=float("inf")), dict(B=-1), dict(T=-1), dict(Nq=0), dict(Nkv=0), dict(Nq=5), dict(Nkv=-2), dict(HD=0),
           dict(HD=4), dict(HD=12), dict(HD=136), dict(HD=-64), dict(Nq=65536, Nkv=1), dict(T=(1 << 30) + 1), dict(B=1 << 20, T=1 << 20),
           dict(B=1 << 20, Nq=32, Nkv=1)]
    for a in bad:
        assert rc(**a) == capi.LLMQ_ERR_INVALID_ARGUMENT, a
        assert capi.lib.llmq_last_error().startswith(b"attention_forward"), a
    for a in (dict(B=0), dict(T=0), dict(B=0, out=None, lse=None, qkv=None)):
        assert rc(**a) == capi.LLMQ_OK


def test_attention_backward_refuses(capi, p):
    f = capi.lib.llmq_attention_backward_bf16
    need = capi.lib.llmq_attention_backward_scratch_bytes(1, 8, 4, 2, 64)
    assert need > 0

    k = 8192   # bytes of dqkv and qkv: 8 tokens of 8 heads of 64

    def rc(d=p, dout=p + k, out=p + 2 * k, lse=p + 3 * k, qkv=p + 4 * k, first=None, s=p + 5 * k, n=need, scale=0.125, B=1, T=8, Nq=4, Nkv=2, HD=64):
        return f(d, dout, out, lse, qkv, first, s, n, scale, B, T, Nq, Nkv, HD, None)

    bad = [dict(d=None), dict(dout=None), dict(out=None), dict(lse=None), dict(qkv=None), dict(s=None), dict(d=p + 2), dict(dout=p + 68), dict(out=p + 130),
           dict(qkv=p + 258), dict(s=p + 520), dict(n=need - 1), dict(n=0), dict(d=p + 4 * k), dict(d=p + 16), dict(d=p + 2 * k - 16),
           dict(d=p + 2 * k), dict(d=p + 3 * k - 16), dict(s=p + 4 * k), dict(s=p + 5 * k - 16), dict(s=p), dict(s=p + k - 16), dict(scale=0.0),
           dict(scale=float("nan")), dict(B=-1), dict(Nq=5), dict(HD=12), dict(HD=136)]
    for a in bad:
        assert rc(**a) == capi.LLMQ_ERR_INVALID_ARGUMENT, a
        assert capi.lib.llmq_last_error().startswith(b"attention_backward"), a
    assert rc(B=0) == capi.LLMQ_OK and rc(T=0, d=None, s=None, n=0) == capi.LLMQ_OK


def test_attention_scratch(capi):
    f = capi.lib.llmq_attention_backward_scratch_bytes
    for bad in ((0, 8, 4, 2, 64), (1, 0, 4, 2, 64), (1, 8, 5, 2, 64), (1, 8, 4, 0, 64), (-1, 8, 4, 2, 64), (1, 8, 4, 2, 0), (1, -8, 4, 2, 64)):
        assert f(*bad) == 0, bad
    for B, T, Nq, Nkv, HD in ((1, 1, 1, 1, 8), (1, 40, 14, 2, 64), (1, 8192, 28, 4, 128), (8, 1024, 28, 4, 128), (300, 1, 2, 2, 64)):
        n = f(B, T, Nq, Nkv, HD)
        assert n % 256 == 0 and n >= 2 * 4 * B * Nq * T
        # two statistics a row, and at most 16 partial sums of the key and value gradients
        assert n <= 2 * 4 * B * Nq * T + 16 * 4 * B * T * Nkv * 2 * HD + 8 * B * T + 4 * 16 * B * Nkv * (T // 128 + 1) + 2048


@pytest.mark.parametrize("ty", ["bf16", "f32"])
def test_token_logprobs_refuse(capi, p, ty):
    f, b = getattr(capi.lib, "llmq_token_logprobs_" + ty), getattr(capi.lib, "llmq_token_logprobs_backward_" + ty)
    need = capi.lib.llmq_token_logprobs_scratch_bytes(1, 1 << 17, 5)
    assert need > 0

    def rc(logp=p, ent=p, lse=p, top=p, ids=p, x=p, t=p, s=p, n=need, N=1, V=1 << 17, P=1 << 17, k=5):
        return f(logp, ent, lse, top, ids, x, t, s, n, N, V, P, k, None)

    bad = [dict(logp=None), dict(lse=None), dict(top=None), dict(ids=None), dict(x=None), dict(t=None), dict(s=None), dict(n=need - 1), dict(x=p + 4),
           dict(s=p + 8), dict(N=-1), dict(N=1 << 24), dict(V=0), dict(V=-5), dict(P=(1 << 17) - 1), dict(P=(1 << 28) + 1), dict(k=-1), dict(k=33)]
    for a in bad:
        assert rc(**a) == capi.LLMQ_ERR_INVALID_ARGUMENT, a
        assert capi.lib.llmq_last_error().startswith(b"token_logprobs"), a
    assert rc(N=0) == capi.LLMQ_OK

    def rcb(d=p, g=p, h=None, x=p, t=p, lse=p, ent=None, am=None, N=1, V=64, P=64):
        return b(d, g, h, x, t, lse, ent, am, N, V, P, None)

    bad = [dict(d=None), dict(g=None), dict(x=None), dict(t=None), dict(lse=None), dict(h=p), dict(d=p + 2), dict(x=p + 2), dict(d=p + 16), dict(N=-1), dict(N=1 << 24),
           dict(V=0), dict(V=65), dict(P=(1 << 28) + 1), dict(N=(1 << 24) - 1, P=1 << 20)]
    for a in bad:
        assert rcb(**a) == capi.LLMQ_ERR_INVALID_ARGUMENT, a
        assert capi.lib.llmq_last_error().startswith(b"token_logprobs_backward"), a
    assert rcb(N=0) == capi.LLMQ_OK


def test_token_logprobs_scratch(capi):
    f = capi.lib.llmq_token_logprobs_scratch_bytes
    for bad in ((0, 9, 1), (-1, 9, 1), (1 << 24, 9, 1), (1, 0, 1), (1, 9, -1), (1, 9, 33)):
        assert f(*bad) == 0, bad
    assert f(1, 1000, 20) == 0 and f(4096, 151936, 5) == 0       # short rows, many rows: not split
    assert 0 < f(1, 151936, 0) < f(1, 151936, 20) <= 64 * (32 + 20 * 8) + 16


def test_wrappers_refuse_host_tensors():
    from llmq_amd import kernels as K
    bf = torch.bfloat16
    qkv, out, lse = torch.zeros((1, 4, 4 * 64), dtype=bf), torch.zeros((1, 4, 128), dtype=bf), torch.zeros((1, 2, 4))
    with pytest.raises(ValueError, match="device tensor"):
        K.attention_forward(out, lse, qkv, None, 2, 1)
    with pytest.raises(ValueError, match="device tensor"):
        K.attention_backward(qkv, out, out, lse, qkv, torch.zeros(4096, dtype=torch.uint8), 2, 1)
    x, t, o = torch.zeros((2, 9)), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    with pytest.raises(ValueError, match="device tensor"):
        K.token_logprobs(o, o, o, None, None, x, t, None)
    with pytest.raises(ValueError, match="device tensor"):
        K.token_logprobs_backward(x, o, None, x, t, o, None, None)
    for shape, Nq, Nkv in (((4, 256), 2, 1), ((1, 4, 255), 2, 1), ((1, 4, 256), 3, 2), ((1, 4, 256), 0, 1), ((1, 4, 256), 2, 0)):
        with pytest.raises(ValueError):
            K.attention_forward(out, lse, torch.zeros(shape, dtype=bf), None, Nq, Nkv)
