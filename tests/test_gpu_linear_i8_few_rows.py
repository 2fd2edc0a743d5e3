"""The kernel of few rows of 8-bit layers where several workgroups share a row's k: ranges of whole units, the ragged end in the last one, the
sums joined by a second launch. Bounds as in the other tests of oz_linear_i8."""
import pytest
import torch

from tests.linear_i8_cases import RANGES, way
from tests.test_gpu_linear_i8 import forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", RANGES, ids=str)
@pytest.mark.parametrize("int8", [True, False], ids=["int8", "values"])
def test_ranges(dev, size, int8):
    assert way(*size)[0] == -1 and way(*size)[1] > 1
    print("linear_i8", size, int8, flush=True)
    forward(dev, *size, t="bf16" if size[0] % 2 else "f16", a="gelu", int8=int8)
    forward(dev, *size, y="f32", a="silu", bias=False, int8=int8, pad=5, inplace=True)


@pytest.mark.parametrize("M", [1, 2, 6])
def test_largest_sums_in_ranges(dev, M):
    """All bytes at int8's lowest: each range's sum and their join are exact."""
    N, K = 40, 32765
    assert way(M, N, K)[0] == -1 and way(M, N, K)[1] > 1
    X, W = (torch.full((n, 32768), -128, dtype=torch.int8, device="cuda:0")[:, :K] for n in (M, N))
    print("linear_i8 lowest", M, flush=True)
    forward(dev, M, N, K, y="f32", bias=False, residual=False, X=X, W=W)
