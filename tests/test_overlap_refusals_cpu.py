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


@pytest.mark.parametrize("ty,es", [("bf16", 2), ("f32", 4)])
def test_token_logprobs_refuse_shared_memory(capi, p, ty, es):
    N, V, P, k = 2, 10000, 10016, 3
    f, b = getattr(capi.lib, "llmq_token_logprobs_" + ty), getattr(capi.lib, "llmq_token_logprobs_backward_" + ty)
    need = capi.lib.llmq_token_logprobs_scratch_bytes(N, V, k)
    assert need > 0
    size = N * P * es
    x = p + 8192

    def forward(logp=p, ent=p + 256, lse=p + 512, top=p + 768, ids=p + 1024, targets=p + 1280, scratch=p + 2048, V=V, k=k):
        return f(logp, ent, lse, top, ids, x, targets, scratch, need, N, V, P, k, None)

    for name, start, n in (("logp", p, 4 * N), ("ent", p + 256, 4 * N), ("lse", p + 512, 4 * N), ("top", p + 768, 4 * N * k),
                           ("ids", p + 1024, 4 * N * k), ("targets", p + 1280, 4 * N), ("scratch", p + 2048, need)):
        own = {"logp": 4 * N, "ent": 4 * N, "lse": 4 * N, "top": 4 * N * k, "ids": 4 * N * k, "targets": 4 * N, "scratch": need}
        for other in own:
            if other == name or (name == "targets" and other == "targets"):
                continue
            for at in (start, start + n - 4, start - own[other] + 4):
                if other == "scratch":
                    at &= ~15
                if at < start + n and start < at + own[other]:
                    assert forward(**{other: at}) == capi.LLMQ_ERR_INVALID_ARGUMENT, (name, other, at - p)
                    assert b"memory of their own" in capi.lib.llmq_last_error(), (name, other)
        if name != "targets":
            for at in (x, (x + size - 4) & ~15 if name == "scratch" else x + size - 4):
                assert forward(**{name: at}) == capi.LLMQ_ERR_INVALID_ARGUMENT, (name, at - x)
                assert b"memory of their own" in capi.lib.llmq_last_error(), name

    d = p + 262144

    def backward(dlogits=d, dlogp=p, dent=p + 256, targets=p + 512, lse=p + 768, ent=p + 1024, am=p + 1280):
        return b(dlogits, dlogp, dent, x, targets, lse, ent, am, N, V, P, None)

    for name in ("dlogp", "dent", "targets", "lse", "ent", "am"):
        for base in (d, x) if name == "am" else (d,):
            for at in (base, base + size - 4) + ((base - 4 * N + 4,) if name != "am" else ()):
                assert backward(**{name: at}) == capi.LLMQ_ERR_INVALID_ARGUMENT, (name, at - base)
                assert b"memory of" in capi.lib.llmq_last_error() and b"own" in capi.lib.llmq_last_error(), name
    for at in (p, p + 4, p + 256, p + 512, p + 768, p + 1028):
        assert backward(am=at) == capi.LLMQ_ERR_INVALID_ARGUMENT, at - p
    for at in (p, p + 4):
        assert backward(dlogits=x, am=at) == capi.LLMQ_ERR_INVALID_ARGUMENT
