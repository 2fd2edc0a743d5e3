"""8-bit layers and rows at the ends of their range: operands and outputs past 4 GiB, more rows than one row of a grid holds."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import Ptr, generator

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def integers(rows, K, seed):
    return torch.randint(-127, 128, (rows, K), device="cuda:0", dtype=torch.int8, generator=generator(seed))


def run(dev, X, W, M, N, K):
    xs = torch.rand(M, device="cuda:0", generator=generator(1)) + 0.5
    ws = (torch.rand(N, device="cuda:0", generator=generator(2)) + 0.5) * 1e-3
    Y = torch.zeros((M, N), device="cuda:0")
    d = ozd.linear_i8_desc(M, N, K, "bf16", "none", "f32", x_int8=True)
    n = dev.linear_i8_workspace(d)
    work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear_i8(d, Ptr(X), Ptr(W), Ptr(ws), Ptr(Y), x_scale=Ptr(xs), work=Ptr(work), work_bytes=n)
    dev.sync()
    return Y, xs, ws


# streamed, by the kernel of few rows, by tiles in ranges of k
@pytest.mark.parametrize("size", [(1, 2**18 + 9, 16384), (4, 2**17 + 5, 32768), (3, 40000, 131068)], ids=str)
def test_weights_past_4_gib(dev, size):
    M, N, K = size
    print("linear_i8", size, flush=True)
    X, W = integers(M, K, 3), integers(N, K, 4)
    Y, xs, ws = run(dev, X, W, M, N, K)
    for i in range(0, N, 8192):
        s = X.double() @ W[i : i + 8192].double().T  # exact: below 2^53
        want = s * xs.double()[:, None] * ws[i : i + 8192].double()
        assert bool(((Y[:, i : i + 8192].double() - want).abs() <= 4 * 2.0**-24 * want.abs()).all()), i


def test_outputs_past_4_gib(dev):
    M, N, K = 2**22 + 1, 600, 64
    print("linear_i8", M, N, K, flush=True)
    X, W = integers(M, K, 5), integers(N, K, 6)
    Y, xs, ws = run(dev, X, W, M, N, K)
    for i in range(0, M, 2**18):
        s = X[i : i + 2**18].float() @ W.float().T  # exact: below 2^24
        want = s.double() * xs[i : i + 2**18].double()[:, None] * ws.double()
        assert bool(((Y[i : i + 2**18].double() - want).abs() <= 4 * 2.0**-24 * want.abs()).all()), i


def test_many_rows_as_integers(dev):
    """2^27 rows and more of 16 values: the workgroups take two rows of the grid, Q ends past 2 GiB."""
    M, K = 2**27 + 100, 16
    print("quantize", M, K, flush=True)
    X = torch.empty((M, K), dtype=torch.bfloat16, device="cuda:0").normal_(generator=generator(7))
    Q, scale = torch.zeros((M, K), dtype=torch.int8, device="cuda:0"), torch.zeros(M, device="cuda:0")
    torch.cuda.synchronize()
    dev.quantize_rows(ozd.quantize_desc(M, K), Ptr(X), Ptr(Q), Ptr(scale))
    dev.sync()
    for i in range(0, M, 2**23):
        x = X[i : i + 2**23].float()
        a = x.abs().amax(1)
        got = Q[i : i + 2**23].float() * scale[i : i + 2**23, None]
        # half a step, and what rounding the scale, its reciprocal and the products adds to it
        assert bool(((got - x).abs() <= (a / 127 * 0.5)[:, None] * (1 + 1e-4)).all()), i
        assert bool((Q[i : i + 2**23].abs().amax(1) == 127).all())
