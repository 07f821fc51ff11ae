"""The registered operators take the calls that their signatures allow: optional tensors left out, given as None or by name.  Without a
GPU every such call ends in the wrapper's refusal of host tensors, not in torch's dispatch."""
import pytest
import torch

from llmq_amd import ops

NAMES = ["abs_max", "quantize_with_abs_max", "quantize_and_transpose_with_abs_max", "transpose", "matmul", "backward_bias", "swiglu_forward",
         "swiglu_forward_quant", "swiglu_backward", "rmsnorm_forward", "fused_residual_rmsnorm_forward", "rmsnorm_backward", "rope_forward",
         "rope_backward", "adamw_update", "attention_forward", "attention_backward", "token_logprobs", "token_logprobs_backward"]


def arguments(schema):
    """Values for the arguments without a default: host tensors of shapes that no wrapper's first checks mind."""
    values = []
    for a in schema.arguments:
        if a.has_default_value():
            break
        kind = str(a.type)
        values.append(torch.zeros((1, 4, 4), dtype=torch.bfloat16) if kind == "Tensor" else None if kind == "Optional[Tensor]" else
                      1e-3 if kind == "float" else 1)
    return values


@pytest.mark.parametrize("name", NAMES)
def test_optional_arguments_may_be_left_out(name):
    op = getattr(torch.ops.llmq, name)
    schema = op.default._schema
    needed = arguments(schema)
    rest = schema.arguments[len(needed):]
    calls = [({}), {a.name: a.default_value for a in rest}] + [{a.name: a.default_value} for a in rest]
    for call in (op, getattr(ops, name)):
        for kw in calls:
            with pytest.raises(ValueError):
                call(*needed, **kw)
        for n in range(len(rest) + 1):
            with pytest.raises(ValueError):
                call(*needed, *(a.default_value for a in rest[:n]))


@pytest.mark.parametrize("name", NAMES)
def test_schemas_and_fake_tensors(name):
    schema = getattr(torch.ops.llmq, name).default._schema
    assert not schema.returns and schema.is_mutable
    written = {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    assert written and written <= {"scale", "out", "out_t", "dst", "c", "workspace", "dbias", "dbias_buffer", "abs_max", "absmax", "dinp", "rms", "residual",
                                   "normed", "rrms", "dweight", "scratch", "params", "m", "v", "m_scales", "lse", "logp", "entropy", "top_logp", "top_ids",
                                   "dlogits"}
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        assert getattr(torch.ops.llmq, name)(*arguments(schema)) is None


def test_written_tensors_count_as_changed():
    """Autograd sees that an operator has written a tensor that a graph still needs."""
    x = torch.ones(3, requires_grad=True)
    y = torch.zeros(3)
    loss = (x * y).sum()
    before = y._version

    @ops._register("version_probe", ("out",))
    def version_probe(out: torch.Tensor, missing: torch.Tensor | None = None) -> None:
        out.detach().fill_(2.0)

    torch.ops.llmq.version_probe(y)
    assert y._version > before and (y == 2).all()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    with torch.inference_mode():
        z = torch.zeros(2)
        torch.ops.llmq.version_probe(z)
        assert (z == 2).all()
