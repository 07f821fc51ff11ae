"""Memory that attention and the token log probabilities write may not be memory that the same call reads or writes elsewhere: refused
on the host, without a GPU."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def capi():
    from llmq_amd import capi
    return capi


@pytest.fixture(scope="module")
def p():
    buf = (C.c_char * (1 << 20))()   # never read: every call below is refused or empty
    p.buf = buf
    return (C.addressof(buf) + 255) & ~255


def test_attention_refuses_first_keys_and_abs_max_inside_other_tensors(capi, p):
    B, T, Nq, Nkv, HD = 1, 8, 4, 2, 64
    k = 8192                                     # bytes of qkv and dqkv; out 4096, lse 128, first_key 32
    out, lse, qkv, first, am = p, p + k, p + 2 * k, p + 3 * k, p + 4 * k

    def forward(first=first, am=am):
        return capi.lib.llmq_attention_forward_bf16(out, lse, qkv, first, am, 0.125, B, T, Nq, Nkv, HD, None)

    for bad in (dict(first=out), dict(first=out + 4092), dict(first=lse), dict(first=lse + 124), dict(first=out - 28), dict(am=out), dict(am=out + 4092),
                dict(am=lse + 64), dict(am=qkv), dict(am=qkv + k - 4), dict(am=first), dict(am=first + 28)):
        assert forward(**bad) == capi.LLMQ_ERR_INVALID_ARGUMENT, bad
        assert b"memory of their own" in capi.lib.llmq_last_error(), bad
    need = capi.lib.llmq_attention_backward_scratch_bytes(B, T, Nq, Nkv, HD)
    dqkv, scratch = p + 10 * k, p + 12 * k

    def backward(first):
        return capi.lib.llmq_attention_backward_bf16(dqkv, p + 5 * k, p + 6 * k, p + 7 * k, p + 8 * k, first, scratch, need, 0.125, B, T, Nq, Nkv, HD,
                                                     None)

    for bad in (dqkv, dqkv + k - 4, dqkv - 28, scratch, scratch + need - 4, scratch - 28):
        assert backward(bad) == capi.LLMQ_ERR_INVALID_ARGUMENT, bad
        assert b"memory of their own" in capi.lib.llmq_last_error(), bad


def test_token_logprobs_backward_refuses_before_it_touches_abs_max(capi, p):
    """A grid that is too large is an error of the arguments, found before abs_max is reset (which needs a device)."""
    for ty, rows in (("bf16", p), ("f32", p)):
        f = getattr(capi.lib, "llmq_token_logprobs_backward_" + ty)
        rc = f(rows, p, None, rows, p, p, None, p + 4096, (1 << 24) - 1, 64, 1 << 20, None)
        assert rc == capi.LLMQ_ERR_INVALID_ARGUMENT, rc
        assert b"too large" in capi.lib.llmq_last_error()
