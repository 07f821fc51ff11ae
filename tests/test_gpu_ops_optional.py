"""GPU tests of the registered operators with their optional tensors left out, and of the gradient that overwrites its logits: the same
bits as the kernel layer's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_operators_without_their_optional_tensors():
    from llmq_amd import kernels as K, ops
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    x = rn(3, 5, 512)
    a, b = (torch.empty((3, 5, 256), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    K.swiglu_forward(a, x, None)
    torch.ops.llmq.swiglu_forward(b, x)
    assert torch.equal(a, b)
    ops.swiglu_forward(b.fill_(0), x, abs_max=None, stream=0)
    assert torch.equal(a, b)
    w, r = rn(512), torch.empty((3, 5), device="cuda")
    a, b = torch.empty_like(x), torch.empty_like(x)
    K.rmsnorm_forward(a, r, x, w, None, 1e-6)
    torch.ops.llmq.rmsnorm_forward(b, r, x, w)
    assert torch.equal(a, b)
    B, T, Nq, Nkv, HD = 2, 50, 4, 2, 64
    qkv = rn(B, T, (Nq + 2 * Nkv) * HD)
    o, p = (torch.empty((B, T, Nq * HD), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    l, m = (torch.empty((B, Nq, T), device="cuda") for _ in range(2))
    K.attention_forward(o, l, qkv, None, Nq, Nkv)
    version = p._version
    torch.ops.llmq.attention_forward(p, m, qkv, Nq=Nq, Nkv=Nkv)
    assert torch.equal(o, p) and torch.equal(l, m) and p._version > version


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_gradient_in_place_through_the_operator(dtype):
    from llmq_amd import kernels as K, ops  # noqa: F401
    x = torch.randn((6, 1003), device="cuda").to(dtype)
    t = torch.arange(6, device="cuda", dtype=torch.int32)
    logp, ent, lse = (torch.empty(6, device="cuda") for _ in range(3))
    torch.ops.llmq.token_logprobs(logp, ent, lse, None, None, x, t, None)
    ones, want = torch.ones(6, device="cuda"), torch.empty_like(x)
    K.token_logprobs_backward(want, ones, ones, x, t, lse, ent, None)
    torch.ops.llmq.token_logprobs_backward(x, ones, ones, x, t, lse, ent)
    assert torch.equal(x, want)
