"""Grids of the products with an epilogue at the ends of their range: a launch takes fewer than 2^32 threads along x. The rule is
asked on the CPU, on 256 compute units; the GPU runs sizes whose workgroups go beyond one row of a grid."""
import ctypes

import pytest
import torch

from oztt_amd import device as ozd
from oztt_amd import hip
from tests.operator_cases import Ptr

# outputs of a tile and threads of its workgroup, by the rule's numbers
TILES = {0: (256, 256, 256), 1: (128, 128, 512), 2: (64, 64, 256), 3: (64, 32, 128), 4: (32, 32, 128)}
TOP = 2**31 - 1


@pytest.mark.parametrize("M", [2**24, 2**26 + 1, 2**28, 2**29 + 5, 2**30, TOP])
@pytest.mark.parametrize("N,K", [(1, 1), (16, 16), (33, 64), (64, 8), (129, 300), (256, 1)])
def test_the_rule_takes_tiles_that_a_launch_holds(M, N, K):
    ll = ctypes.c_longlong
    if 2 * (M * N + M * K + N * K) > 288 * 10**9:
        pytest.skip("more than the card's memory")
    for contiguous, nq, np, C in ((1, M, N, K), (0, M, K, N), (0, N, K, M)):
        s = ctypes.c_int()
        t = hip().oz_rule_linear_route(256, ll(nq), ll(np), ll(C), contiguous, 1, ctypes.byref(s))
        if t < 0:  # the kernels of few rows, whose grid goes by N
            assert contiguous and nq <= 32
            continue
        q, p, threads = TILES[t]
        assert -(-nq // q) * -(-np // p) * s.value * threads < 2**32, (t, s.value)


@pytest.fixture
def memory():
    """Up to 70 GB a test are given back."""
    yield
    torch.cuda.empty_cache()


def check(dev, M, K, X, W, Y, **kw):
    d = ozd.linear_desc(M, 1, K, **kw)
    n = dev.linear_workspace(d)
    work = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), work=Ptr(work), work_bytes=n)
    dev.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("M,shift", [(TOP, 0), (2**29 + 100, 1)])
def test_as_many_rows_as_there_may_be(dev, memory, M, shift):
    """All rows that an int counts; and more than 2^29 at an odd address, which the kernel that reads value by value takes."""
    print("linear", M, shift, flush=True)
    base = torch.empty(M + shift, dtype=torch.bfloat16, device="cuda:0")
    X, Y = base[shift:], torch.full((M,), 7.0, dtype=torch.bfloat16, device="cuda:0")
    step = 1 << 27
    part = lambda i: (torch.arange(i, min(i + step, M), device="cuda:0") % 97 - 48).bfloat16()  # noqa: E731
    for i in range(0, M, step):
        X[i : i + step] = part(i)
    check(dev, M, 1, X, torch.full((1,), 0.5, dtype=torch.bfloat16, device="cuda:0"), Y)
    assert all(torch.equal(Y[i : i + step], part(i) * 0.5) for i in range(0, M, step))


@pytest.mark.gpu
def test_an_operand_of_more_pieces_than_a_row_of_a_grid(dev, memory):
    """2^22 rows of 4097 values, which are laid out first: 2^23 workgroups and more."""
    M, K = 2**22, 4097
    print("linear", M, K, flush=True)
    X = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda:0")
    X[:, 0], X[:, K - 1] = 1.0, 2.0
    X[M - 1, 5] = 4.0
    W = torch.ones(K, dtype=torch.bfloat16, device="cuda:0")
    Y = torch.zeros(M, dtype=torch.bfloat16, device="cuda:0")
    check(dev, M, K, X, W, Y)
    assert bool((Y[:-1] == 3.0).all()) and float(Y[-1]) == 7.0
