"""oz_linear and oz_linear_grad against the formulas in 64 bits.

Bounds: a sum of n products in FP32, in any order, is off by at most n 2^-24 times the sum of their sizes (every
product of two 16-bit values is exact in FP32); the activations' slopes are at most 1.13 and their evaluation is off by
at most 2^-21 |z|; every output is rounded once more, and so is dZ in front of the products."""
import numpy as np
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, ROUND, U32, Ptr, act, act_grad, generator, rounded, window, within

pytestmark = pytest.mark.gpu

# from one value to sizes on either side of every kernel's tiles
SIZES = [(1, 1, 1), (1, 700, 33), (1, 4096, 4096), (2, 16, 8), (7, 300, 2000), (16, 512, 512), (17, 130, 72), (24, 2048, 520),
         (33, 1000, 4104), (64, 64, 64), (65, 96, 1000), (100, 257, 1000), (129, 520, 64), (256, 256, 256), (300, 200, 2056),
         (257, 255, 129), (512, 1024, 96), (1000, 700, 1500), (1100, 1304, 40), (2048, 2304, 264)]


def operands(M, N, K, t, seed, pad, shift):
    g = generator(seed)
    x = torch.randn((M, K), device="cuda:0", generator=g).to(DTYPE[t])
    w = (torch.randn((N, K), device="cuda:0", generator=g) * K**-0.5).to(DTYPE[t])
    return window(x, pad, shift)[0], window(w, pad, shift)[0]


def forward(dev, M, N, K, t="bf16", a="none", y=None, bias=True, residual=True, keep=True, pad=0, shift=0, seed=1, inplace=False):
    y = y or t
    X, W = operands(M, N, K, t, seed, pad, shift)
    g = generator(seed + 100)
    B = torch.randn((1, N), device="cuda:0", generator=g).to(DTYPE[t]) if bias else None
    R = window(torch.randn((M, N), device="cuda:0", generator=g).to(DTYPE[y]), pad, shift)[0] if residual else None
    Y, around = window(torch.full((M, N), 7.0, device="cuda:0", dtype=DTYPE[y]), pad, shift, fill=5.0)
    if inplace:
        Y.copy_(R)
    r0 = R.double() if residual else None
    Z, zaround = window(torch.full((M, N), 7.0, device="cuda:0", dtype=DTYPE[t]), pad, shift, fill=5.0)
    d = ozd.linear_desc(M, N, K, t, a, y, ldx=K + pad, ldw=K + pad, ldy=N + pad, ldr=N + pad, ldz=N + pad)
    n = dev.linear_workspace(d)
    work = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), bias=Ptr(B), residual=Ptr(Y if inplace else R), Z=Ptr(Z if keep else None), work=Ptr(work), work_bytes=n)
    dev.sync()
    z = X.double() @ W.double().T
    size = X.double().abs() @ W.double().abs().T
    if bias:
        z, size = z + B.double(), size + B.double().abs()
    off = (K + 2) * U32 * size
    want = act(z, a)
    off_y = 1.13 * off + 2.0**-21 * z.abs()
    if residual:
        want = want + r0
        off_y = off_y + U32 * want.abs()
    within(Y, want, off_y + rounded(want.abs() + off_y, y), "Y")
    if keep:
        within(Z, z, off + rounded(z.abs() + off, t), "Z")
    # nothing around the outputs is touched
    for base, out in ((around, Y), (zaround, Z)):
        out.fill_(5.0)
        assert bool((base == 5.0).all())
    return X, W, Y


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_forward_sizes(dev, size, t):
    print("linear", size, t, flush=True)
    forward(dev, *size, t=t, a="gelu")


# the large tiles, in one range of c and in several, at sizes that fit none of them
LARGE = [(3498, 3506, 3502), (2050, 2043, 32766), (2052, 2310, 1000), (40, 6000, 4096), (5000, 516, 520)]


@pytest.mark.parametrize("size", LARGE, ids=str)
def test_forward_large(dev, size):
    print("linear", size, flush=True)
    forward(dev, *size, t="f16", a="silu")
    forward(dev, *size, t="bf16", a="none", y="f32", bias=False, keep=False, pad=6)


@pytest.mark.parametrize("size", [(3498, 3506, 3502), (4100, 520, 516), (5000, 1030, 2052), (130, 2052, 4100)], ids=str)
def test_gradient_large(dev, size):
    print("linear_grad", size, flush=True)
    gradients(dev, *size, t="bf16", a="gelu")
    gradients(dev, *size, t="f16", a="none", dw="f32", pad=2, accumulate=True)


@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 0), (0, 1), (16, 8), (3, 2)])
@pytest.mark.parametrize("size", [(1, 300, 512), (20, 304, 1000), (300, 264, 520), (520, 1030, 257)], ids=str)
def test_forward_windows(dev, size, pad, shift):
    """Rows apart by more than their length, and operands at addresses that are multiples of 2 bytes alone; NaN
    between the rows."""
    print("linear", size, pad, shift, flush=True)
    forward(dev, *size, pad=pad, shift=shift, a="silu")


@pytest.mark.parametrize("a", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("y", ["bf16", "f32"])
@pytest.mark.parametrize("M", [3, 200])
def test_forward_epilogues(dev, a, y, M):
    for bias, residual, keep in ((0, 0, 0), (1, 0, 1), (0, 1, 0), (1, 1, 1)):
        print("linear epilogue", M, a, y, bias, residual, keep, flush=True)
        forward(dev, M, 328, 136, a=a, y=y, bias=bias, residual=residual, keep=keep)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_residual_in_place(dev, M):
    forward(dev, M, 264, 128, inplace=True)
    forward(dev, M, 264, 128, y="f32", inplace=True)


@pytest.mark.parametrize("M", [2, 70, 520])
def test_infinities_stay_in_their_rows(dev, M):
    """One row of X with an infinity, one row of W with a NaN: every other output is what it is without them."""
    N, K = 272, 200
    X, W = operands(M, N, K, "bf16", 3, 0, 0)
    out = []
    for bad in (False, True):
        if bad:
            X[1, 7] = float("inf")
            W[5, 3] = float("nan")
        Y = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda:0")
        d = ozd.linear_desc(M, N, K, "bf16", "gelu")
        n = dev.linear_workspace(d)
        work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), work=Ptr(work), work_bytes=n)
        dev.sync()
        out.append(Y)
    rows = torch.tensor([m for m in range(M) if m != 1], device="cuda:0")
    cols = torch.tensor([c for c in range(N) if c != 5], device="cuda:0")
    assert torch.equal(out[0][rows][:, cols], out[1][rows][:, cols])
    assert bool(out[1][:, 5].isnan().all()) and bool((out[1][1, cols].isinf() | out[1][1, cols].isnan()).all())


def test_large_activations(dev):
    """Values whose square and cube overflow: the activations' limits, and no NaN."""
    z = torch.tensor([[-3e38, -1e20, -1e13, -200.0, -90.0, -20.0, -0.0, 0.0, 20.0, 90.0, 1e13, 3e38]], device="cuda:0").bfloat16()
    W = torch.eye(12, device="cuda:0").bfloat16()
    for a in ("relu", "gelu", "silu"):
        Y, dY = torch.zeros_like(z), torch.ones_like(z)
        dZ = torch.zeros_like(z)
        d, gd = ozd.linear_desc(1, 12, 12, "bf16", a), ozd.linear_grad_desc(1, 12, 12, "bf16", a)
        n, gn = dev.linear_workspace(d), dev.linear_grad_workspace(gd)
        work = torch.zeros(max(n, gn, 16), dtype=torch.uint8, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear(d, Ptr(z), Ptr(W), Ptr(Y), work=Ptr(work), work_bytes=n)
        dev.linear_grad(gd, Ptr(dY), Ptr(None), Ptr(W), Ptr(z), dX=Ptr(dZ), work=Ptr(work), work_bytes=gn)
        dev.sync()
        want = torch.where(z > 0, z, torch.zeros_like(z)).float()
        assert torch.allclose(Y.float(), want, rtol=2.0**-8, atol=1e-6), a
        assert torch.allclose(dZ.float(), (z > 0).float() + (0.5 if a != "relu" else 0) * (z == 0).float(), atol=1e-6), a


def gradients(dev, M, N, K, t="bf16", a="gelu", dw=None, pad=0, shift=0, accumulate=False, seed=5, want=("dX", "dW", "dbias")):
    dw = dw or t
    X, W = operands(M, N, K, t, seed, pad, shift)
    g = generator(seed + 100)
    dY = window(torch.randn((M, N), device="cuda:0", generator=g).to(DTYPE[t]), pad, shift)[0]
    Z = window((1.5 * torch.randn((M, N), device="cuda:0", generator=g)).to(DTYPE[t]), pad, shift)[0] if a != "none" else None
    before = torch.randn((N, K), device="cuda:0", generator=g).to(DTYPE[dw])
    bbefore = torch.randn((1, N), device="cuda:0", generator=g).to(DTYPE[dw])
    dX, xa = window(torch.full((M, K), 7.0, device="cuda:0", dtype=DTYPE[t]), pad, shift, fill=5.0)
    dW, wa = window(before, pad, shift, fill=5.0)
    dB, ba = window(bbefore, 0, shift, fill=5.0)
    d = ozd.linear_grad_desc(M, N, K, t, a, dw, accumulate, lddy=N + pad, ldx=K + pad, ldw=K + pad, ldz=N + pad, lddx=K + pad, lddw=K + pad)
    n = dev.linear_grad_workspace(d)
    work = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda:0")
    out = {"dX": dX, "dW": dW, "dbias": dB}
    torch.cuda.synchronize()
    dev.linear_grad(d, Ptr(dY), Ptr(X), Ptr(W), Ptr(Z), work=Ptr(work), work_bytes=n, **{k: Ptr(out[k]) for k in want})
    dev.sync()
    dz = dY.double() * (act_grad(Z.double(), a) if Z is not None else 1.0)
    # the slopes are off by at most 2^-20; dZ is rounded where it is not dY
    u, floor = ROUND[t] if Z is not None else (0.0, 0.0)
    off = (2.0**-20 * dY.double().abs() if Z is not None else torch.zeros_like(dz)) + u * dz.abs() + floor

    def product(p, dp, q, n):
        size = p.abs() @ q.abs()
        return p @ q, (n + 2) * U32 * size + dp @ q.abs()

    if "dX" in want:
        x, bx = product(dz, off, W.double(), N)
        within(dX, x, bx + rounded(x.abs() + bx, t), "dX")
    old, bold = (before.double(), bbefore.double()) if accumulate else (0.0, 0.0)
    if "dW" in want:
        w, bw = product(dz.T, off.T, X.double(), M)
        w, bw = w + old, bw + (U32 * (w.abs() + before.double().abs()) if accumulate else 0)
        within(dW, w, bw + rounded(w.abs() + bw, dw), "dW")
    if "dbias" in want:
        b = dz.sum(0, keepdim=True) + bold
        bb = ((M + 2) * U32 * dz.abs() + (2.0**-20 * dY.double().abs() if Z is not None else 0)).sum(0, keepdim=True) + U32 * (b.abs() + bbefore.double().abs())
        within(dB, b, bb + rounded(b.abs() + bb, dw), "dbias")
    for base, o in ((xa, dX), (wa, dW), (ba, dB)):
        o.fill_(5.0)
        assert bool((base == 5.0).all())


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_gradient_sizes(dev, size, t):
    print("linear_grad", size, t, flush=True)
    gradients(dev, *size, t=t)


@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 0), (0, 1), (16, 8), (3, 2)])
@pytest.mark.parametrize("size", [(1, 300, 512), (20, 304, 1000), (300, 264, 520), (520, 1030, 257)], ids=str)
def test_gradient_windows(dev, size, pad, shift):
    print("linear_grad", size, pad, shift, flush=True)
    gradients(dev, *size, pad=pad, shift=shift, a="silu")


@pytest.mark.parametrize("a", ["none", "relu", "silu"])
@pytest.mark.parametrize("dw", ["bf16", "f32"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_forms(dev, a, dw, accumulate):
    print("linear_grad", a, dw, accumulate, flush=True)
    for size in ((40, 264, 136), (700, 320, 264)):
        gradients(dev, *size, a=a, dw=dw, accumulate=accumulate)


@pytest.mark.parametrize("want", [("dX",), ("dW",), ("dbias",), ("dX", "dbias")], ids=str)
@pytest.mark.parametrize("a", ["none", "gelu"])
def test_single_gradients(dev, want, a):
    gradients(dev, 200, 136, 72, a=a, want=want)


def test_no_rows(dev):
    """M = 0: no outputs; the gradients of W and bias are sums of nothing."""
    W = torch.ones((8, 16), dtype=torch.bfloat16, device="cuda:0")
    dev.linear(ozd.linear_desc(0, 8, 16), Ptr(None), Ptr(W), Ptr(None))
    for accumulate, want in ((False, 0.0), (True, 3.0)):
        dW, dB = torch.full((8, 16), 3.0, device="cuda:0"), torch.full((8,), 3.0, device="cuda:0")
        d = ozd.linear_grad_desc(0, 8, 16, "bf16", "gelu", "f32", accumulate)
        n = dev.linear_grad_workspace(d)
        work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear_grad(d, Ptr(None), Ptr(None), Ptr(W), Ptr(None), dW=Ptr(dW), dbias=Ptr(dB), work=Ptr(work), work_bytes=n)
        dev.sync()
        assert bool((dW == want).all()) and bool((dB == want).all())


@pytest.mark.parametrize("a", ["gelu", "silu"])
def test_gradients_against_differences(dev, a):
    """dX, dW and dbias of sum(C Y) against central differences of the formula in 64 bits: their error is the step
    squared times a third derivative (below 1e-7 here), so the bound is that of dZ's and the outputs' rounding,
    2^-9 of the sum of the sizes of the terms each."""
    M, N, K = 40, 72, 48
    X, W = operands(M, N, K, "bf16", 9, 0, 0)
    g = generator(10)
    B = torch.randn(N, device="cuda:0", generator=g).bfloat16()
    C = torch.randn((M, N), device="cuda:0", generator=g).bfloat16()
    Z = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda:0")
    Y = torch.zeros_like(Z)
    out = {"dX": torch.zeros_like(X), "dW": torch.zeros_like(W), "dbias": torch.zeros_like(B)}
    d, gd = ozd.linear_desc(M, N, K, "bf16", a), ozd.linear_grad_desc(M, N, K, "bf16", a)
    n, gn = dev.linear_workspace(d), dev.linear_grad_workspace(gd)
    work = torch.zeros(max(n, gn, 16), dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), bias=Ptr(B), Z=Ptr(Z), work=Ptr(work), work_bytes=n)
    dev.linear_grad(gd, Ptr(C), Ptr(X), Ptr(W), Ptr(Z), work=Ptr(work), work_bytes=gn, **{k: Ptr(v) for k, v in out.items()})
    dev.sync()
    v = {"dX": X.double(), "dW": W.double(), "dbias": B.double()}
    loss = lambda: float((C.double() * act(v["dX"] @ v["dW"].T + v["dbias"], a)).sum())  # noqa: E731
    dz = (C.double() * act_grad(Z.double(), a)).abs()
    # Z itself is rounded, which moves the slopes by up to 2^-9 |z| times their own slope, at most 1.2
    dz = dz + 1.2 * (C.double() * Z.double()).abs()
    size = {"dX": dz @ W.double().abs(), "dW": dz.T @ X.double().abs(), "dbias": dz.sum(0)}
    h = 1e-4
    for k, x in v.items():
        flat = x.view(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 12)):
            at = float(flat[i])
            flat[i] = at + h
            up = loss()
            flat[i] = at - h
            diff = (up - loss()) / (2 * h)
            flat[i] = at
            assert abs(diff - float(out[k].view(-1)[i])) <= 3 * 2.0**-9 * float(size[k].view(-1)[i]) + 1e-6, (k, i)


def test_same_bits_again(dev):
    for M, N, K in ((1, 1000, 5000), (24, 520, 2048), (520, 264, 4096)):
        X, W = operands(M, N, K, "bf16", 2, 0, 0)
        dY = torch.randn((M, N), device="cuda:0").bfloat16()
        outs = []
        for _ in range(3):
            Y, dX, dW, dB = (torch.zeros(s, dtype=torch.bfloat16, device="cuda:0") for s in ((M, N), (M, K), (N, K), (N,)))
            d, gd = ozd.linear_desc(M, N, K), ozd.linear_grad_desc(M, N, K)
            n, gn = dev.linear_workspace(d), dev.linear_grad_workspace(gd)
            work = torch.zeros(max(n, gn, 16), dtype=torch.uint8, device="cuda:0")
            torch.cuda.synchronize()
            dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), work=Ptr(work), work_bytes=n)
            dev.linear_grad(gd, Ptr(dY), Ptr(X), Ptr(W), dX=Ptr(dX), dW=Ptr(dW), dbias=Ptr(dB), work=Ptr(work), work_bytes=gn)
            dev.sync()
            outs.append((Y, dX, dW, dB))
        for o in outs[1:]:
            assert all(torch.equal(p, q) for p, q in zip(o, outs[0]))


def test_refusals_name_what_is_wrong(dev):
    X = torch.zeros(4096, dtype=torch.bfloat16, device="cuda:0")
    p, odd = Ptr(X), Ptr(X.view(torch.uint8)[1:])
    good = ozd.linear_desc(4, 8, 16)
    for what, call in (
            ("null operand", lambda: dev.linear(good, Ptr(None), p, p)),
            ("null operand", lambda: dev.linear(good, p, p, Ptr(None))),
            ("addresses", lambda: dev.linear(good, odd, p, p)),
            ("leading dimension", lambda: dev.linear(ozd.linear_desc(4, 8, 16, ldx=15), p, p, p)),
            ("residual is Y", lambda: dev.linear(ozd.linear_desc(4, 8, 16, ldy=16), p, p, p, residual=p)),
            ("null operand", lambda: dev.linear_grad(ozd.linear_grad_desc(4, 8, 16, act="gelu"), p, p, p, dX=p)),
            ("null operand", lambda: dev.linear_grad(ozd.linear_grad_desc(4, 8, 16), p, None, p, dW=p)),
            ("workspace", lambda: dev.linear_grad(ozd.linear_grad_desc(4, 8, 16, act="gelu"), p, p, p, Z=p, dX=p))):
        with pytest.raises(RuntimeError, match=what):
            call()
    dev.sync()
    assert not X.any()
