"""oz_linear_grad with an activation and a dW in FP32, against the formula in 64 bits under bounds that a dZ in 16 bits misses.

Bounds: the slopes are off by at most 2^-20; dZ is the sum of two values of the operands' type, the second of what rounding to the
first leaves, so it is off by at most u^2 |dZ| (u: half the distance of neighbours) and the least values of FP16. Two sums of M
products each in FP32, and the roundings where they and what was there before meet."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, ROUND, U32, Ptr, act_grad, generator, window, within

pytestmark = pytest.mark.gpu


def gradient(dev, M, N, K, t, a, accumulate=False, pad=0, shift=0, size_of_dy=1.0):
    g = generator(M + N + K)
    normal = lambda rows, cols, s: window((s * torch.randn((rows, cols), device="cuda:0", generator=g)).to(DTYPE[t]), pad, shift)[0]  # noqa: E731
    dY, Z, X, W = normal(M, N, size_of_dy), normal(M, N, 1.5), normal(M, K, 1.0), normal(N, K, K**-0.5)
    before = torch.randn((N, K), device="cuda:0", generator=g)
    dW, around = window(before, pad, shift, fill=5.0)
    dX, dB = torch.zeros((M, K), dtype=DTYPE[t], device="cuda:0"), torch.zeros(N, device="cuda:0")
    d = ozd.linear_grad_desc(M, N, K, t, a, "f32", accumulate, lddy=N + pad, ldx=K + pad, ldw=K + pad, ldz=N + pad, lddw=K + pad)
    n = dev.linear_grad_workspace(d)
    work = torch.full((n + 256,), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear_grad(d, Ptr(dY), Ptr(X), Ptr(W), Ptr(Z), dX=Ptr(dX), dW=Ptr(dW), dbias=Ptr(dB), work=Ptr(work), work_bytes=n)
    dev.sync()
    assert bool((work[n:] == 0x7F).all())
    dz = dY.double() * act_grad(Z.double(), a)
    u, floor = ROUND[t]
    off = 2.0**-20 * dY.double().abs() + u * u * dz.abs() + floor
    x = X.double().abs()
    old = before.double() if accumulate else 0.0 * before.double()
    want = dz.T @ X.double() + old
    bound = (2 * M + 4) * U32 * (dz.abs().T @ x) + off.T @ x + 2 * U32 * (want.abs() + old.abs())
    within(dW, want, bound, "dW")
    dW.fill_(5.0)
    assert bool((around == 5.0).all())


@pytest.mark.parametrize("size", [(1, 33, 40), (40, 264, 136), (700, 320, 264), (1000, 257, 129), (300, 5, 64), (4100, 520, 516)], ids=str)
@pytest.mark.parametrize("t,a", [("bf16", "gelu"), ("f16", "silu"), ("f16", "gelu"), ("bf16", "silu")])
def test_bounds_of_32_bits(dev, size, t, a):
    for accumulate, pad, shift in ((False, 0, 0), (True, 8, 0), (False, 3, 1)):
        print("linear_grad f32", size, t, a, accumulate, pad, shift, flush=True)
        gradient(dev, *size, t, a, accumulate, pad, shift)


def test_small_gradients_in_fp16(dev):
    gradient(dev, 700, 320, 264, "f16", "gelu", size_of_dy=1e-2)


@pytest.mark.parametrize("a", ["gelu", "silu"])
def test_values_beyond_16_bits(dev, a):
    """A dZ that FP16 does not hold gives infinities in its row of dW, and no NaN."""
    M, N, K = 40, 72, 48
    dY = torch.full((M, N), 2.0, dtype=torch.float16, device="cuda:0")
    Z = torch.full((M, N), 2.0, dtype=torch.float16, device="cuda:0")
    dY[7, 3] = 65504.0  # the slope at 2 is above 1
    X = torch.ones((M, K), dtype=torch.float16, device="cuda:0")
    dW = torch.zeros((N, K), device="cuda:0")
    d = ozd.linear_grad_desc(M, N, K, "f16", a, "f32")
    n = dev.linear_grad_workspace(d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear_grad(d, Ptr(dY), Ptr(X), Ptr(None), Ptr(Z), dW=Ptr(dW), work=Ptr(work), work_bytes=n)
    dev.sync()
    assert not dW.isnan().any() and not dW[:3].isinf().any() and not dW[4:].isinf().any() and bool((dW[3] >= 65504).all())
