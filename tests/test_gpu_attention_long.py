"""GPU tests of attention on long rows, and of blocks of keys that are not split, against the formulas in 64 bits with the bars of
test_gpu_attention."""
import pytest
import torch

from test_gpu_attention import check, first_keys, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from llmq_amd import kernels
    return kernels


# (B, T, Nq, Nkv, HD), shares of the walk over the queries: 16, 8, 2, 5, 1, 2
@pytest.mark.parametrize("shape", [(1, 8191, 2, 1, 128), (1, 4500, 4, 2, 64), (5, 2100, 4, 4, 64), (8, 1029, 6, 3, 80), (24, 1300, 4, 4, 128),
                                   (24, 1100, 4, 2, 32)])
@pytest.mark.parametrize("kind", ["none", "window", "docs", "long docs", "pad"])
def test_long_rows_match_the_formulas(K, shape, kind):
    B, T, Nq, Nkv, HD = shape
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    first = (t // 900 * 900).expand(B, T).contiguous() if kind == "long docs" else first_keys(kind, B, T)
    qkv, dout = make(*shape, seed=23)
    check(K, qkv, dout, Nq, Nkv, first)


@pytest.mark.parametrize("shape", [(1, 5000, 3, 1, 64), (1, 3333, 2, 2, 128)])
def test_long_windows_with_large_scores(K, shape):
    B, T, Nq, Nkv, HD = shape
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    qkv, dout = make(*shape, seed=29, std=4.0)
    check(K, qkv, dout, Nq, Nkv, (t - 1500).expand(B, T).contiguous())
