"""The FP8-path kernels under the reference's Python signatures, registered as torch custom ops.

The reference exposes its kernels to Python as `torch.library.custom_op("llmq::<name>", mutates_args=...)`
wrappers over its compiled extension (src/binding/python/kernels.py:118-165, argument handling in
src/binding/kernel_binding.cpp:393-509).  This module registers the same operator names, argument
order, defaults and mutation declarations on top of the gfx950 C ABI, so code written against
`pyllmq.kernels` for this path runs unchanged after swapping the import:

    abs_max(scale, x, stream=0)
    quantize_with_abs_max(out, scale, x, abs_max, stream=0)
    quantize_and_transpose_with_abs_max(out, scale, x, abs_max, stream=0)
    transpose(dst, src, stream=0)
    matmul(c, a, b, bias, scale_a, scale_b, cublaslt_handle, workspace, mode, accumulate=False, stream=0)
    backward_bias(dbias, dout, scale_a, scale_b, dbias_buffer, stream=0)
    get_bias_backward_scratch_size(dtype, OC);  create_cublas_handle();  destroy_cublas_handle(handle)
    swiglu_forward(out, inp, abs_max=None, stream=0);  swiglu_forward_quant(out, scale, inp, abs_max, stream=0)
    swiglu_backward(dinp, dout, inp, abs_max=None, stream=0)
    rmsnorm_forward(out, rms, inp, weight, absmax=None, epsilon, stream=0)
    fused_residual_rmsnorm_forward(residual, normed, rrms, inp1, inp2, weight, absmax=None, epsilon, stream=0)
    rmsnorm_backward(dinp, dweight, scratch, dresidual, dout, inp, weight, rstd, absmax=None, stream=0)
    get_rmsnorm_backward_scratch_size(C)
    adamw_update(params, grads, m, v, learning_rate, beta1, beta2, t, eps, weight_decay, grad_scale, m_scales=None,
                 abs_max=None, seed=0, stream=0)
    rope_forward(out, inp, freqs_cis, absmax=None, Nq, Nkv, stream=0);  rope_backward(dinp, dout, freqs_cis, absmax=None, Nq, Nkv, stream=0)
    attention_forward(out, lse, inp, absmax=None, Nq, Nkv, first_key=None, softmax_scale=0, stream=0)
    attention_backward(dinp, dout, out, lse, inp, scratch, Nq, Nkv, first_key=None, softmax_scale=0, stream=0)
    get_attention_backward_scratch_size(B, T, Nq, Nkv, HD)
    token_logprobs(logp, entropy, lse, top_logp, top_ids, logits, targets, scratch, vocab=0, stream=0)
    token_logprobs_backward(dlogits, dlogp, dentropy, logits, targets, lse, entropy, absmax=None, vocab=0, stream=0)
    get_token_logprobs_scratch_size(N, V, k)

matmul is in the torch sense (c = op(a) @ op(b), mode: TT=0, TN=1, NT=2, NN=3).  FP8 operands are served in
mode NT (c[M,N] = a[M,K] @ b[N,K]^T, both K-contiguous: every shape with K % 16 == 0) and, for bf16 output on
whole 256-wide tiles, in the other three modes as well (a stored [K, M] and / or b stored [K, N]: the operand is
read in that storage, no transposed copy); other dtype combinations raise, as the reference does for what it does
not implement.
"""
import inspect

import torch

from . import kernels as _k

MODE_TT, MODE_TN, MODE_NT, MODE_NN = 0, 1, 2, 3

_library = torch.library.Library("llmq", "FRAGMENT")


def _register(name, mutates_args):
    """Registers a function that writes `mutates_args` and returns nothing as the operator llmq::name, with the schema its annotations
    and defaults give, and puts the operator in its place.

    Not torch.library.custom_op: its count of a written tensor's versions looks every one of `mutates_args` up among the arguments,
    but the dispatcher leaves out trailing ones that have their default value, and every call with an optional tensor left out, or
    given as None, ended in an IndexError."""
    def register(fn):
        schema = torch.library.infer_schema(fn, mutates_args=mutates_args)
        _library.define(name + schema, tags=(torch.Tag.pt2_compliant_tag,))
        names = list(inspect.signature(fn).parameters)
        written = [names.index(a) for a in mutates_args]

        def run(*args):
            fn(*args)
            for i in written:
                if i < len(args) and args[i] is not None and not args[i].is_inference():
                    torch.autograd.graph.increment_version(args[i])

        _library.impl(name, run, "CompositeExplicitAutograd")
        torch.library.register_fake("llmq::" + name, lambda *args: None, lib=_library)
        return getattr(torch.ops.llmq, name)
    return register


@_register("abs_max", ("scale",))
def abs_max(scale: torch.Tensor, x: torch.Tensor, stream: int = 0) -> None:
    _k.abs_max(scale, x, stream)


@_register("quantize_with_abs_max", ("out", "scale"))
def quantize_with_abs_max(out: torch.Tensor, scale: torch.Tensor, x: torch.Tensor, abs_max: torch.Tensor,
                          stream: int = 0) -> None:
    _k.quantize_with_abs_max(out, scale, x, abs_max, stream)


@_register("quantize_and_transpose_with_abs_max", ("out", "scale"))
def quantize_and_transpose_with_abs_max(out: torch.Tensor, scale: torch.Tensor, x: torch.Tensor,
                                        abs_max: torch.Tensor, stream: int = 0) -> None:
    _k.quantize_and_transpose_with_abs_max(out, scale, x, abs_max, stream)


@_register("transpose", ("dst",))
def transpose(dst: torch.Tensor, src: torch.Tensor, stream: int = 0) -> None:
    _k.transpose(dst, src, stream)


@_register("matmul", ("c", "workspace"))
def matmul(c: torch.Tensor, a: torch.Tensor, b: torch.Tensor, bias: torch.Tensor | None,
           scale_a: torch.Tensor | None, scale_b: torch.Tensor | None, cublaslt_handle: int,
           workspace: torch.Tensor, mode: int, accumulate: bool = False, stream: int = 0) -> None:
    if a.dim() != 2 or b.dim() != 2 or c.dim() != 2:
        raise ValueError("matmul: a, b and c must be 2-dimensional")
    if mode not in (MODE_NT, MODE_TT, MODE_TN, MODE_NN):
        raise ValueError("matmul: unknown mode %r (TT = 0, TN = 1, NT = 2, NN = 3)" % (mode,))
    m, k = a.shape if mode in (MODE_NT, MODE_NN) else (a.shape[1], a.shape[0])
    n, k2 = b.shape if mode in (MODE_NT, MODE_TT) else (b.shape[1], b.shape[0])
    if k != k2 or c.shape[0] != m or c.shape[1] != n:
        raise ValueError("matmul: shapes do not match: a %s, b %s, c %s" % (tuple(a.shape), tuple(b.shape), tuple(c.shape)))
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != n):
        raise ValueError("matmul: bias must have %d elements" % n)
    # torch vs column-major convention of the kernel layer: operands and their scales swap places
    # (src/binding/kernel_binding.cpp:403-431): c[m, n] = sum_k a[m, k] b[n, k]
    # a stored [K, M] (torch modes TN, TT) is the kernel layer's K-major second operand, b stored [K, N] (NN, TN) its
    # K-major first operand
    _k.matmul(c, b, a, bias, scale_b, scale_a, n, m, k, accumulate, stream, workspace,
              b_kmajor=mode in (MODE_TN, MODE_TT), a_kmajor=mode in (MODE_NN, MODE_TN))


@_register("backward_bias", ("dbias", "dbias_buffer"))
def backward_bias(dbias: torch.Tensor, dout: torch.Tensor, scale_a: torch.Tensor | None,
                  scale_b: torch.Tensor | None, dbias_buffer: torch.Tensor, stream: int = 0) -> None:
    _k.backward_bias(dbias, dout, scale_a, scale_b, dbias_buffer, stream)


@_register("swiglu_forward", ("out", "abs_max"))
def swiglu_forward(out: torch.Tensor, inp: torch.Tensor, abs_max: torch.Tensor | None = None, stream: int = 0) -> None:
    _k.swiglu_forward(out, inp, abs_max, stream)


@_register("swiglu_forward_quant", ("out", "scale"))
def swiglu_forward_quant(out: torch.Tensor, scale: torch.Tensor, inp: torch.Tensor, abs_max: torch.Tensor,
                         stream: int = 0) -> None:
    _k.swiglu_forward_quant(out, scale, inp, abs_max, stream)


@_register("swiglu_backward", ("dinp", "abs_max"))
def swiglu_backward(dinp: torch.Tensor, dout: torch.Tensor, inp: torch.Tensor, abs_max: torch.Tensor | None = None,
                    stream: int = 0) -> None:
    _k.swiglu_backward(dinp, dout, inp, abs_max, stream)


@_register("rmsnorm_forward", ("out", "rms", "absmax"))
def rmsnorm_forward(out: torch.Tensor, rms: torch.Tensor, inp: torch.Tensor, weight: torch.Tensor,
                    absmax: torch.Tensor | None = None, epsilon: float = 1e-6, stream: int = 0) -> None:
    _k.rmsnorm_forward(out, rms, inp, weight, absmax, epsilon, stream)


@_register("fused_residual_rmsnorm_forward", ("residual", "normed", "rrms", "absmax"))
def fused_residual_rmsnorm_forward(residual: torch.Tensor, normed: torch.Tensor, rrms: torch.Tensor, inp1: torch.Tensor,
                                   inp2: torch.Tensor, weight: torch.Tensor, absmax: torch.Tensor | None = None,
                                   epsilon: float = 1e-6, stream: int = 0) -> None:
    _k.fused_residual_rmsnorm_forward(residual, normed, rrms, inp1, inp2, weight, absmax, epsilon, stream)


@_register("rmsnorm_backward", ("dinp", "dweight", "scratch", "absmax"))
def rmsnorm_backward(dinp: torch.Tensor, dweight: torch.Tensor, scratch: torch.Tensor, dresidual: torch.Tensor,
                     dout: torch.Tensor, inp: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                     absmax: torch.Tensor | None = None, stream: int = 0) -> None:
    _k.rmsnorm_backward(dinp, dweight, scratch, dresidual, dout, inp, weight, rstd, absmax, stream)


@_register("rope_forward", ("out", "absmax"))
def rope_forward(out: torch.Tensor, inp: torch.Tensor, freqs_cis: torch.Tensor, absmax: torch.Tensor | None = None,
                 Nq: int = 0, Nkv: int = 0, stream: int = 0) -> None:
    _k.rope_forward(out, inp, freqs_cis, absmax, Nq, Nkv, stream)


@_register("rope_backward", ("dinp", "absmax"))
def rope_backward(dinp: torch.Tensor, dout: torch.Tensor, freqs_cis: torch.Tensor, absmax: torch.Tensor | None = None,
                  Nq: int = 0, Nkv: int = 0, stream: int = 0) -> None:
    _k.rope_backward(dinp, dout, freqs_cis, absmax, Nq, Nkv, stream)


@_register("adamw_update", ("params", "m", "v", "m_scales", "abs_max"))
def adamw_update(params: torch.Tensor, grads: torch.Tensor, m: torch.Tensor, v: torch.Tensor, learning_rate: float,
                 beta1: float, beta2: float, t: int, eps: float, weight_decay: float, grad_scale: torch.Tensor,
                 m_scales: torch.Tensor | None = None, abs_max: torch.Tensor | None = None, seed: int = 0,
                 stream: int = 0) -> None:
    _k.adamw_update(params, grads, m, v, learning_rate, beta1, beta2, t, eps, weight_decay, grad_scale, m_scales, abs_max,
                    seed, stream)


@_register("attention_forward", ("out", "lse", "absmax"))
def attention_forward(out: torch.Tensor, lse: torch.Tensor, inp: torch.Tensor, absmax: torch.Tensor | None = None, Nq: int = 0,
                      Nkv: int = 0, first_key: torch.Tensor | None = None, softmax_scale: float = 0.0, stream: int = 0) -> None:
    _k.attention_forward(out, lse, inp, absmax, Nq, Nkv, first_key, softmax_scale or None, stream)


@_register("attention_backward", ("dinp", "scratch"))
def attention_backward(dinp: torch.Tensor, dout: torch.Tensor, out: torch.Tensor, lse: torch.Tensor, inp: torch.Tensor,
                       scratch: torch.Tensor, Nq: int, Nkv: int, first_key: torch.Tensor | None = None,
                       softmax_scale: float = 0.0, stream: int = 0) -> None:
    _k.attention_backward(dinp, dout, out, lse, inp, scratch, Nq, Nkv, first_key, softmax_scale or None, stream)


def get_attention_backward_scratch_size(B: int, T: int, Nq: int, Nkv: int, HD: int):
    return _k.get_attention_backward_scratch_size(B, T, Nq, Nkv, HD)


@_register("token_logprobs", ("logp", "entropy", "lse", "top_logp", "top_ids", "scratch"))
def token_logprobs(logp: torch.Tensor, entropy: torch.Tensor | None, lse: torch.Tensor, top_logp: torch.Tensor | None,
                   top_ids: torch.Tensor | None, logits: torch.Tensor, targets: torch.Tensor, scratch: torch.Tensor | None,
                   vocab: int = 0, stream: int = 0) -> None:
    _k.token_logprobs(logp, entropy, lse, top_logp, top_ids, logits, targets, scratch, vocab or None, stream)


@_register("token_logprobs_backward", ("dlogits", "absmax"))
def token_logprobs_backward(dlogits: torch.Tensor, dlogp: torch.Tensor, dentropy: torch.Tensor | None, logits: torch.Tensor,
                            targets: torch.Tensor, lse: torch.Tensor, entropy: torch.Tensor | None,
                            absmax: torch.Tensor | None = None, vocab: int = 0, stream: int = 0) -> None:
    _k.token_logprobs_backward(dlogits, dlogp, dentropy, logits, targets, lse, entropy, absmax, vocab or None, stream)


def get_token_logprobs_scratch_size(N: int, V: int, k: int):
    return _k.get_token_logprobs_scratch_size(N, V, k)


def get_rmsnorm_backward_scratch_size(C: int):
    return _k.get_rmsnorm_backward_scratch_size(C)


def get_bias_backward_scratch_size(dtype: torch.dtype, OC: int):
    return _k.get_bias_backward_scratch_size(dtype, OC)


def create_cublas_handle() -> int:
    """The gfx950 kernels need no library handle; a placeholder keeps the reference's call pattern."""
    return 0


def destroy_cublas_handle(handle: int) -> None:
    return None
