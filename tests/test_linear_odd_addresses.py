"""Operands of oz_linear and oz_linear_grad at addresses that are no multiples of 4 bytes: the descriptor says so, the workspace has
room for their copies, and the call lays them out in it for the tiles instead of reading value by value."""
import ctypes

import pytest
import torch

from oztt_amd import device as ozd
from oztt_amd import hip
from tests.operator_cases import DTYPE, Ptr, generator, window


def ask(name, desc):
    return getattr(hip(), name)(None, ctypes.byref(desc))


@pytest.mark.parametrize("M,N,K", [(33, 64, 1000), (1000, 700, 1500), (300, 264, 520)])
def test_room(M, N, K):
    forward = lambda **o: ask("oz_linear_workspace", ozd.linear_desc(M, N, K, **o))  # noqa: E731
    least = forward()
    assert forward(odd=["X"]) >= least + 2 * M * K and forward(odd=["W"]) >= least + 2 * N * K
    assert forward(odd=["X", "W"]) >= least + 2 * (M + N) * K
    grad = lambda **o: ask("oz_linear_grad_workspace", ozd.linear_grad_desc(M, N, K, **o))  # noqa: E731
    assert grad(odd=["X"]) >= 2 * M * K and grad(odd=["W"]) >= 2 * N * K and grad(odd=["dY"]) >= grad() + 2 * M * N


def test_odd_leading_dimensions_have_room_already():
    for o in ((), ("X",), ("W", "X")):
        assert ask("oz_linear_workspace", ozd.linear_desc(100, 80, 64, ldx=65, ldw=67, odd=o)) == ask(
            "oz_linear_workspace", ozd.linear_desc(100, 80, 64, ldx=65, ldw=67))


def test_few_rows_need_none():
    """They are read in place; only the ranges' sums are kept."""
    assert ask("oz_linear_workspace", ozd.linear_desc(2, 64, 1000, odd=["X", "W"])) == 0


def test_refusals():
    for bits in (4, 8, -1):
        d = ozd.linear_desc(4, 8, 16)
        d.odd = bits
        assert ask("oz_linear_workspace", d) == -1
    g = ozd.linear_grad_desc(4, 8, 16)
    g.odd = 8
    assert ask("oz_linear_grad_workspace", g) == -1
    with pytest.raises(ValueError):
        ozd.linear_desc(4, 8, 16, odd=["Z"])


def laid_out(work, at, x):
    """Whether the copy of x stands at byte `at` of the workspace, rows of a multiple of 8 values, zeros behind."""
    rows, cols = x.shape
    ld = (cols + 7) // 8 * 8
    c = work[at : at + 2 * rows * ld].view(x.dtype).view(rows, ld)
    return torch.equal(c[:, :cols], x) and not c[:, cols:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [("X",), ("W",), ("X", "W")], ids=str)
@pytest.mark.parametrize("M,N,K", [(40, 264, 136), (33, 1000, 1502), (600, 704, 1504)])
def test_linear(dev, M, N, K, odd):
    """The same bits as from aligned operands (the same tiles), with a workspace of the size asked for."""
    print("linear odd", M, N, K, odd, flush=True)
    g = generator(M)
    x, w = (torch.randn(s, device="cuda:0", generator=g).bfloat16() for s in ((M, K), (N, K)))
    X, W = (window(v, 2, int(k in odd))[0] for k, v in (("X", x), ("W", w)))
    got = []
    for o in ((), odd):
        d = ozd.linear_desc(M, N, K, ldx=K + 2 if o else 0, ldw=K + 2 if o else 0, odd=o)
        n = dev.linear_workspace(d)
        work = torch.full((n + 256,), 0x7F, dtype=torch.uint8, device="cuda:0")
        Y = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear(d, Ptr(X if o else x), Ptr(W if o else w), Ptr(Y), work=Ptr(work), work_bytes=n)
        dev.sync()
        assert bool((work[n:] == 0x7F).all())
        got.append(Y)
    assert torch.equal(*got)
    tile = ozd.hip().oz_rule_linear_route(256, *(ctypes.c_longlong(v) for v in (M, N, K)), 1, 0, ctypes.byref(s := ctypes.c_int()))
    assert tile >= 0
    at = 0 if s.value == 1 else (4 * s.value * M * ((N + 7) // 8 * 8) + 255) // 256 * 256
    for k, v in (("X", x), ("W", w)):
        if k in odd:
            assert laid_out(work, at, v), k
            at += (2 * v.shape[0] * ((K + 7) // 8 * 8) + 255) // 256 * 256


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [("X",), ("W",), ("dY",), ("X", "W", "dY")], ids=str)
@pytest.mark.parametrize("a", ["none", "silu"])
@pytest.mark.parametrize("M,N,K", [(40, 264, 136), (600, 704, 1504)])
def test_linear_grad(dev, M, N, K, a, odd):
    print("linear_grad odd", M, N, K, a, odd, flush=True)
    g = generator(M)
    v = {k: torch.randn(s, device="cuda:0", generator=g).bfloat16() for k, s in (("dY", (M, N)), ("X", (M, K)), ("W", (N, K)), ("Z", (M, N)))}
    got = []
    for o in ((), odd):
        p = {k: Ptr(window(x, 2, int(k in o))[0]) for k, x in v.items()}
        d = ozd.linear_grad_desc(M, N, K, "bf16", a, "f32", lddy=N + 2, ldx=K + 2, ldw=K + 2, ldz=N + 2, odd=o)
        n = dev.linear_grad_workspace(d)
        work = torch.full((n + 256,), 0x7F, dtype=torch.uint8, device="cuda:0")
        out = {"dX": torch.zeros((M, K), dtype=DTYPE["bf16"], device="cuda:0"), "dW": torch.zeros((N, K), device="cuda:0"),
               "dbias": torch.zeros(N, device="cuda:0")}
        torch.cuda.synchronize()
        dev.linear_grad(d, p["dY"], p["X"], p["W"], p["Z"], work=Ptr(work), work_bytes=n, **{k: Ptr(t) for k, t in out.items()})
        dev.sync()
        assert bool((work[n:] == 0x7F).all())
        got.append(out)
    assert all(torch.equal(got[0][k], got[1][k]) for k in got[0])
    if "dY" in odd and a == "none":
        assert torch.equal(work[: 2 * M * N].view(torch.bfloat16).view(M, N), v["dY"])


@pytest.mark.gpu
def test_unsaid_addresses_are_taken_all_the_same(dev):
    """In the workspace that the leading dimensions ask for; of few rows, whose c would be cut into ranges with more, one range."""
    for M, N, K in ((40, 264, 136), (20, 40, 8192)):
        print("linear odd, unsaid", M, N, K, flush=True)
        x, w = (torch.randn(s, device="cuda:0", generator=generator(M)).bfloat16() for s in ((M, K), (N, K)))
        X, W = (window(v, 0, 1)[0] for v in (x, w))
        d = ozd.linear_desc(M, N, K, y_type="f32")
        n = dev.linear_workspace(d)
        work = torch.full((n + 256,), 0x7F, dtype=torch.uint8, device="cuda:0")
        Y = torch.zeros((M, N), device="cuda:0")
        torch.cuda.synchronize()
        dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), work=Ptr(work), work_bytes=n)
        dev.sync()
        assert bool((work[n:] == 0x7F).all())
        size = x.double().abs() @ w.double().abs().T
        assert bool(((Y.double() - x.double() @ w.double().T).abs() <= (K + 2) * 2.0**-24 * size).all())
