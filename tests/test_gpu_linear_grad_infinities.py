"""oz_linear_grad where dY or Z is infinite or not a number."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, Ptr, generator

pytestmark = pytest.mark.gpu


def gradients(dev, dY, Z, X, W, t, a, dw="f32"):
    (M, N), K = dY.shape, X.shape[1]
    out = {"dX": torch.zeros((M, K), dtype=DTYPE[t], device="cuda:0"), "dW": torch.zeros((N, K), dtype=DTYPE[dw], device="cuda:0"),
           "dbias": torch.zeros(N, dtype=DTYPE[dw], device="cuda:0")}
    d = ozd.linear_grad_desc(M, N, K, t, a, dw)
    n = dev.linear_grad_workspace(d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear_grad(d, Ptr(dY), Ptr(X), Ptr(W), Ptr(Z), work=Ptr(work), work_bytes=n, **{k: Ptr(v) for k, v in out.items()})
    dev.sync()
    return out


def inputs(M, N, K, t):
    g = generator(M + N)
    normal = lambda *s: torch.randn(s, device="cuda:0", generator=g).to(DTYPE[t])  # noqa: E731
    return normal(M, N), normal(M, N), normal(M, K), normal(N, K)


def same(a, b):
    return all(torch.equal(a[k], b[k]) for k in a)


def only_there(got, plain, m, n):
    """NaN in row m of dX, row n of dW and value n of dbias; everything else as without it."""
    for k, at in (("dX", m), ("dW", n), ("dbias", n)):
        others = torch.arange(len(got[k]), device="cuda:0") != at
        assert bool(got[k][at].isnan().all()), k
        assert torch.equal(got[k][others], plain[k][others]), k


SIZES = [(3, 5, 16), (40, 264, 136), (300, 72, 40)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_relu_leaves_out_what_it_masks(dev, size, t):
    """Where z <= 0 nothing of dY goes on, infinities and NaN included; a z that is not a number, which the forward pass hands on,
    is handed on."""
    print("linear_grad relu", size, t, flush=True)
    dY, Z, X, W = inputs(*size, t)
    Z[1, 2], Z[2, 3], Z[0, 1], Z[0, 4] = -1.0, 0.0, -0.0, -float("inf")
    masked = dY.clone()
    for k, (at, v) in enumerate((((1, 2), "inf"), ((2, 3), "-inf"), ((0, 1), "nan"), ((0, 4), "inf"))):
        dY[at], masked[at] = float(v), 0.25 * k
    want = gradients(dev, masked, Z, X, W, t, "relu")
    assert not any(bool(v.isnan().any()) for v in want.values())
    assert same(gradients(dev, dY, Z, X, W, t, "relu"), want)
    Z[2, 4] = float("nan")
    only_there(gradients(dev, masked, Z, X, W, t, "relu"), want, 2, 4)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("a", ["gelu", "silu"])
@pytest.mark.parametrize("t,dw", [("bf16", "bf16"), ("f16", "f32")])
def test_slopes_at_infinities(dev, size, a, t, dw):
    """A Z that left FP16's range is kept as infinite; its slope is the limit, 1 or 0, as of any large z."""
    print("linear_grad", a, size, t, flush=True)
    dY, Z, X, W = inputs(*size, t)
    Z[1, 2], Z[2, 3], Z[0, 1] = 300.0, -300.0, 300.0
    want = gradients(dev, dY, Z, X, W, t, a, dw)
    Z[1, 2], Z[2, 3], Z[0, 1] = float("inf"), -float("inf"), float("inf")
    assert same(gradients(dev, dY, Z, X, W, t, a, dw), want)
    Z[2, 4] = float("nan")
    only_there(gradients(dev, dY, Z, X, W, t, a, dw), want, 2, 4)
