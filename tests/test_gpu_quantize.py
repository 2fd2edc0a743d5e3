"""oz_quantize_rows against the definition, bit by bit: NumPy's FP32 quotients, products and rounding to even are the same operations."""
import numpy as np
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, Ptr, generator, window

pytestmark = pytest.mark.gpu


def definition(x: np.ndarray):
    x = x.astype(np.float32)
    a = np.max(np.abs(x), axis=1)
    bad = ~np.isfinite(a)
    a = np.maximum(np.where(bad, np.float32(1), a), np.float32(127 * 2.0**-126))
    q = np.rint(np.where(bad[:, None], np.float32(0), x) * (np.float32(127) * (np.float32(1) / a))[:, None])
    scale = np.where(bad, np.float32(np.nan), a * (np.float32(1) / np.float32(127)))
    return q.astype(np.int8), scale.astype(np.float32)


def check(dev, X, K, ldx, ldq, shift=0):
    M = X.shape[0]
    base = torch.full((M * ldq + shift + 64,), 99, dtype=torch.int8, device="cuda:0")
    Q = base[shift : shift + M * ldq].view(M, ldq)[:, :K]
    scale = torch.full((M + 1,), 5.0, device="cuda:0")
    t = {v: k for k, v in DTYPE.items()}[X.dtype]
    torch.cuda.synchronize()
    dev.quantize_rows(ozd.quantize_desc(M, K, t, ldx=ldx, ldq=ldq), Ptr(X), Ptr(Q), Ptr(scale))
    dev.sync()
    with np.errstate(invalid="ignore"):
        q, s = definition(X.float().cpu().numpy())
    np.testing.assert_array_equal(Q.cpu().numpy(), q)
    np.testing.assert_array_equal(scale[:M].cpu().numpy(), s)
    assert float(scale[M]) == 5.0
    Q.fill_(99)
    assert bool((base == 99).all()), "bytes around Q"


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 511), (7, 512), (4, 513), (9, 1000), (24, 2048), (6, 2049), (300, 4096), (5, 4104), (3, 8192), (3, 8200),
         (2, 16384), (2, 16391), (2, 40000), (1, 131071), (5000, 40)]


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(dev, size, t):
    M, K = size
    print("quantize", size, t, flush=True)
    g = generator(M + K)
    x = (torch.randn((M, K), device="cuda:0", generator=g) * torch.exp(torch.randn((M, 1), device="cuda:0", generator=g))).to(DTYPE[t])
    check(dev, x, K, K, K)


@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 1), (1, 3), (0, 7)])
@pytest.mark.parametrize("K", [40, 1001, 20000])
def test_windows(dev, K, pad, shift):
    """NaN between X's rows, bytes between Q's that stay."""
    print("quantize window", K, pad, shift, flush=True)
    x, _ = window(torch.randn((6, K), device="cuda:0", generator=generator(1)).to(torch.float16), pad, shift)
    check(dev, x, K, K + pad, K + pad, shift)


@pytest.mark.parametrize("K", [3, 700, 20000])
def test_what_rows_may_hold(dev, K):
    """Zeros, one value alone, ties, the smallest and largest numbers, values that are not finite, each in a row of its own."""
    x = torch.randn((12, K), device="cuda:0", generator=generator(2))
    x[0] = 0
    x[1] = 0
    x[1, K - 1] = -3.5
    x[2] = torch.arange(K, device="cuda:0") % 127 + 0.5  # ties, with a scale that is a power of two times 1/127
    x[2, 0] = 127.0
    x[3] = 1e-45
    x[4] *= 1e-38
    x[5] *= 1e38
    x[5, 0] = 3.4028234e38
    x[6, K // 2] = float("inf")
    x[7, K - 1] = float("nan")
    x[8, 0] = -float("inf")
    x[9] = -0.0
    x[10] = -2.0
    check(dev, x, K, K, K)
    check(dev, x.to(torch.bfloat16), K, K, K)


def test_no_rows(dev):
    x = torch.zeros(1, device="cuda:0")
    dev.quantize_rows(ozd.quantize_desc(0, 16, "f32"), Ptr(None), Ptr(None), Ptr(None))
    dev.sync()
    assert float(x[0]) == 0
