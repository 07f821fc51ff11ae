"""A training step of the attention half of a transformer block, its head and the loss, composed from the library's entry points
with every GEMM input quantized to e4m3 from the abs-max its producer wrote:

    ln1 = rmsnorm_forward(x);  qkv = matmul(ln1, Wqkv);  rope_forward;  attention_forward;  y = matmul(att, Wo)
    r, ln2 = fused_residual_rmsnorm_forward(x, y);  logits = matmul(ln2, Wv);  token_logprobs
    loss = -mean(logp) - 0.01 mean(entropy), back through token_logprobs_backward, matmul, rmsnorm_backward, attention_backward,
    rope_backward and matmul to the weights and x.

(1) The abs-max each producer wrote equals abs_max() of its tensor.  (2) The attention and the loss inside the step agree with the
formulas in 64 bits on the tensors they were given.  (3) The step agrees with the same step in 64 bits without quantization within
twice a budget of relative errors that add in squares, e = 4.5 % for a product of two e4m3 operands:
    qkv e;  scores sqrt(2) e = 6.4 % of a unit deviation, so the probabilities 6.4 % and att sqrt(6.4^2 + 4.5^2) = 7.8 %;  y 9 %;
    the stream x + y below 9 %;  logits 10 %, of a deviation of 1, so logp 0.1;  dlogits: p moves by 10 % of itself, but its norm is
    sqrt(e / V) = 5 % of the target's 1: 0.5 %, and 0.4 % of rounding;  dln2 4.5 %;  dWv (ln2 9 %, product 4.5 %) 10 %;
    dr and dn2 (norm of a stream 9 % off) 10 %;  dWo 13.5 %;  datt 11 %;  ds (datt, values, probabilities) 13.6 %;  dqkv 14.5 %;
    dWqkv, dn1 and dx 15 %."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F8, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available()
    from llmq_amd import kernels
    return kernels


class Tensor:
    """A bf16 tensor with its abs-max, its e4m3 codes and their scale."""

    def __init__(self, K, *shape):
        self.K, self.value = K, torch.empty(shape, dtype=BF, device="cuda")
        self.quant, self.stats = torch.empty(shape, dtype=F8, device="cuda"), torch.zeros(2, device="cuda")

    abs_max = property(lambda s: s.stats[0:1])
    scale = property(lambda s: s.stats[1:2])

    def quantize(self):
        self.K.quantize_with_abs_max(self.quant, self.scale, self.value, self.abs_max)
        return self


def rel(got, ref):
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu().view(got.shape)
    return float((got - ref).norm() / ref.norm())


def test_attention_block_and_loss(K):
    B, T, C, Nq, Nkv, HD, V, eps = 2, 256, 512, 8, 2, 64, 1024, 1e-6
    BT, Q = B * T, (Nq + 2 * Nkv) * HD
    g = torch.Generator(device="cuda").manual_seed(21)
    rn = lambda std, *s: (std * torch.randn(s, device="cuda", generator=g)).to(BF)  # noqa: E731
    x = rn(1.0, B, T, C)
    n1, n2 = (1.0 + 0.1 * torch.randn(C, device="cuda", generator=g)).to(BF), (1.0 + 0.1 * torch.randn(C, device="cuda", generator=g)).to(BF)
    wqkv, wo, wv = rn(C ** -0.5, Q, C), rn(C ** -0.5, C, Nq * HD), rn(C ** -0.5, V, C)
    target = torch.randint(0, V, (B, T), device="cuda", generator=g, dtype=torch.int32)
    target[0, :7] = -100
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    first = torch.stack([(t // 100) * 100, t * 0]).contiguous()              # packed documents, one long one
    freqs = K.precompute_freqs_cis(HD, T, 10000.0).cuda()
    ws = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")

    def weight(w):
        q = Tensor(K, *w.shape)
        q.value.copy_(w)
        K.abs_max(q.abs_max, q.value)
        return q.quantize()

    Wqkv, Wo, Wv = weight(wqkv), weight(wo), weight(wv)

    def product(inp, w):
        n, k = w.quant.shape
        out = torch.empty((B, T, n), dtype=BF, device="cuda")
        K.matmul(out, w.quant, inp.quant, None, w.scale, inp.scale, n, BT, k, workspace=ws)
        return out

    def backward_product(dout, inp, w):
        """The gradients of `inp` and of the weight from the quantized gradient of the product."""
        n, k = w.quant.shape
        wt, it, gt = (torch.empty(s, dtype=F8, device="cuda") for s in ((k, n), (k, BT), (n, BT)))
        K.transpose(wt, w.quant)
        dinp = torch.empty((B, T, k), dtype=BF, device="cuda")
        K.matmul(dinp, wt, dout.quant, None, w.scale, dout.scale, k, BT, n, workspace=ws)
        K.transpose(it, inp.quant.view(BT, k))
        K.transpose(gt, dout.quant.view(BT, n))
        dw = torch.empty((n, k), device="cuda")
        K.matmul(dw, it, gt, None, inp.scale, dout.scale, k, n, BT, workspace=ws)
        return dinp, dw

    # forward
    ln1, rstd1 = Tensor(K, B, T, C), torch.empty((B, T), device="cuda")
    K.rmsnorm_forward(ln1.value, rstd1, x, n1, ln1.abs_max, eps)
    qkv = product(ln1.quantize(), Wqkv)
    K.rope_forward(qkv, qkv, freqs, None, Nq, Nkv)
    att, lse = Tensor(K, B, T, Nq * HD), torch.empty((B, Nq, T), device="cuda")
    K.attention_forward(att.value, lse, qkv, att.abs_max, Nq, Nkv, first)
    y = product(att.quantize(), Wo)
    r, ln2, rstd2 = torch.empty_like(x), Tensor(K, B, T, C), torch.empty((B, T), device="cuda")
    K.fused_residual_rmsnorm_forward(r, ln2.value, rstd2, x, y, n2, ln2.abs_max, eps)
    logits = product(ln2.quantize(), Wv)
    logp, ent, llse = (torch.empty((B, T), device="cuda") for _ in range(3))
    top, ids = torch.empty((B, T, 3), device="cuda"), torch.empty((B, T, 3), dtype=torch.int32, device="cuda")
    size = K.get_token_logprobs_scratch_size(BT, V, 3)
    K.token_logprobs(logp, ent, llse, top, ids, logits, target, torch.empty(max(size, 1), dtype=torch.uint8, device="cuda"))
    # backward
    dlogits = Tensor(K, B, T, V)
    K.token_logprobs_backward(dlogits.value, torch.full((B, T), -1.0 / BT, device="cuda"), torch.full((B, T), -0.01 / BT, device="cuda"), logits,
                              target, llse, ent, dlogits.abs_max)
    dln2, dwv = backward_product(dlogits.quantize(), ln2, Wv)
    scratch = torch.empty(K.get_rmsnorm_backward_scratch_size(C), device="cuda")
    dr, dn2 = Tensor(K, B, T, C), torch.zeros(C, dtype=BF, device="cuda")
    K.rmsnorm_backward(dr.value, dn2, scratch, torch.zeros_like(x), dln2, r, n2, rstd2, dr.abs_max)
    datt, dwo = backward_product(dr.quantize(), att, Wo)
    dqkv = Tensor(K, B, T, Q)
    buf = torch.empty(K.get_attention_backward_scratch_size(B, T, Nq, Nkv, HD), dtype=torch.uint8, device="cuda")
    K.attention_backward(dqkv.value, datt, att.value, lse, qkv, buf, Nq, Nkv, first)
    dqkv_attention = dqkv.value.clone()
    K.rope_backward(dqkv.value, dqkv.value, freqs, dqkv.abs_max, Nq, Nkv)
    dln1, dwqkv = backward_product(dqkv.quantize(), ln1, Wqkv)
    dx, dn1 = Tensor(K, B, T, C), torch.zeros(C, dtype=BF, device="cuda")
    K.rmsnorm_backward(dx.value, dn1, scratch, dr.value, dln1, x, n1, rstd1, dx.abs_max)

    # (1)
    ref = torch.zeros(1, device="cuda")
    for name, q in (("ln1", ln1), ("att", att), ("ln2", ln2), ("dlogits", dlogits), ("dr", dr), ("dqkv", dqkv), ("dx", dx)):
        K.abs_max(ref, q.value)
        assert q.abs_max.item() == ref.item(), name

    # (2)
    from test_gpu_attention import exact as attention
    from test_gpu_logprobs import es, exact as logprobs
    e = attention(qkv, datt, Nq, Nkv, first)
    assert ((att.value.double() - e["out"]).abs() <= e["bar_out"] + 1e-30).all()
    assert ((dqkv_attention.double() - e["grad"]).abs() <= e["bar_grad"] + 1e-30).all()
    elogp, eent, else_, xt, given, _, _ = logprobs(logits.view(BT, V), target.view(BT), V)
    bar = es(V) + 2.0 ** -23 * (else_.abs() + xt.abs())
    assert ((logp.view(BT) - elogp).abs() <= bar).all() and ((ent.view(BT) - eent).abs() <= 61 * es(V) + 2.0 ** -22 * (1 + eent)).all()
    assert torch.equal(ids.view(BT, 3), torch.sort(logits.view(BT, V).float(), dim=1, descending=True, stable=True)[1][:, :3].int())

    # (3)
    d64 = lambda z: z.detach().double().cpu()  # noqa: E731
    X, N1, N2, WQ, WO, WV = (d64(z).requires_grad_(True) for z in (x, n1, n2, wqkv, wo, wv))
    norm = lambda z, w: z * torch.rsqrt((z ** 2).mean(-1, keepdim=True) + eps) * w  # noqa: E731
    q = (norm(X, N1) @ WQ.t()).view(B, T, Nq + 2 * Nkv, HD)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, HD, 2, dtype=torch.float64) / HD)
    cs = torch.view_as_real(torch.polar(torch.ones_like(ang), ang))[:, None]
    a, b = q[:, :, :Nq + Nkv, :HD // 2], q[:, :, :Nq + Nkv, HD // 2:]
    q = torch.cat([torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1), q[:, :, Nq + Nkv:]], 2)
    kk, vv = (z.repeat_interleave(Nq // Nkv, 2) for z in (q[:, :, Nq:Nq + Nkv], q[:, :, Nq + Nkv:]))
    tt, f = torch.arange(T), first.long().cpu()
    mask = (tt[None, None, :] <= tt[None, :, None]) & (tt[None, None, :] >= f[:, :, None])
    s = torch.einsum("bthd,bkhd->bhtk", q[:, :, :Nq], kk) * HD ** -0.5
    p = torch.softmax(s.masked_fill(~mask[:, None], -math.inf), -1)
    A = torch.einsum("bhtk,bkhd->bthd", p, vv).reshape(B, T, Nq * HD)
    R = X + A @ WO.t()
    L = norm(R, N2) @ WV.t()
    lp = torch.log_softmax(L, -1)
    tok = target.long().cpu()
    picked = torch.where(tok >= 0, lp.gather(-1, tok.clamp_min(0)[..., None])[..., 0], torch.zeros((), dtype=torch.float64))
    loss = (-picked + 0.01 * (lp.exp() * lp).sum(-1)).sum() / BT
    loss.backward()
    errs = {"att": (rel(att.value, A), 0.156), "logits": (rel(logits, L), 0.20), "logp": ((logp.cpu() - picked).pow(2).mean().sqrt().item(), 0.2),
            "dwv": (rel(dwv, WV.grad), 0.20), "dn2": (rel(dn2, N2.grad), 0.20), "dwo": (rel(dwo, WO.grad), 0.27), "dwqkv": (rel(dwqkv, WQ.grad), 0.30),
            "dx": (rel(dx.value, X.grad), 0.30), "dn1": (rel(dn1, N1.grad), 0.30)}
    print({k: round(v[0], 4) for k, v in errs.items()})
    for k, (v, limit) in errs.items():
        assert v < limit, (k, v)
