"""oz_linear_i8 against the formula: sums of integers in 64 bits, the rest in binary64.

Bounds: the exact int32 sum is rounded to FP32 and multiplied twice (three roundings), the bias is added (one more); the activations' slopes
are at most 1.13 and their evaluation is off by at most 2^-21 |z|; the residual's addition and the output are rounded once each. X that
the call quantizes has the integers and scales of oz_quantize_rows, whose own tests hold them to the definition."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, U32, Ptr, act, generator, rounded, window, within

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 4), (1, 1, 1), (1, 700, 33), (1, 4096, 4096), (1, 515, 16384), (2, 16, 8), (2, 1000, 3000), (3, 64, 128), (7, 300, 2000), (16, 512, 512),
         (17, 130, 72), (24, 2048, 520), (33, 1000, 4104), (64, 64, 64), (65, 96, 1000), (100, 257, 1000), (129, 520, 64), (256, 256, 256), (300, 200, 2056),
         (257, 255, 129), (512, 1024, 96), (1000, 700, 1500), (1100, 1304, 40), (2048, 2304, 264)]
LARGE = [(3498, 3506, 3502), (2050, 2043, 32766), (2052, 2310, 1000), (40, 6000, 4096), (5000, 516, 520), (10, 24, 131071), (300, 260, 131071)]


def up4(n):
    return -(-n // 4) * 4


def integers(g, rows, K, pad, least=-127):
    """Bytes in rows that begin at multiples of 4; what is between them is 77."""
    x = torch.randint(least, 128, (rows, K), device="cuda:0", generator=g, dtype=torch.int8)
    return window(x, up4(K + pad) - K, fill=77)[0]


def whole_sum(X, W):
    """X W^T of integers, exactly: products in FP64, whose sums stay below 2^53."""
    return torch.matmul(X.double(), W.double().T)


def forward(dev, M, N, K, t="bf16", a="none", y=None, bias=True, residual=True, int8=True, pad=0, shift=0, seed=1, inplace=False, X=None, W=None):
    y = y or t
    g = generator(seed)
    W = integers(g, N, K, pad, -128) if W is None else W
    ws = torch.exp(torch.randn(N, device="cuda:0", generator=g)) * 0.01 * K**-0.5
    xs = None
    if int8:
        X = integers(g, M, K, pad, -128) if X is None else X
        xs = torch.exp(torch.randn(M, device="cuda:0", generator=g)) * 0.02
        q, s = X, xs
    else:
        x = torch.randn((M, K), device="cuda:0", generator=g) * torch.exp(torch.randn((M, 1), device="cuda:0", generator=g))
        X = window(x.to(DTYPE[t]), pad, shift)[0]
        q, s = torch.zeros((M, K), dtype=torch.int8, device="cuda:0"), torch.zeros(M, device="cuda:0")
        torch.cuda.synchronize()
        dev.quantize_rows(ozd.quantize_desc(M, K, t, ldx=X.stride(0)), Ptr(X), Ptr(q), Ptr(s))
        dev.sync()
    B = torch.randn((1, N), device="cuda:0", generator=g).to(DTYPE[t]) if bias else None
    R = window(torch.randn((M, N), device="cuda:0", generator=g).to(DTYPE[y]), pad, shift)[0] if residual else None
    Y, around = window(torch.full((M, N), 7.0, device="cuda:0", dtype=DTYPE[y]), pad, shift, fill=5.0)
    if inplace:
        Y.copy_(R)
    r0 = R.double() if residual else None
    d = ozd.linear_i8_desc(M, N, K, t, a, y, x_int8=int8, ldx=X.stride(0), ldw=W.stride(0), ldy=N + pad, ldr=N + pad)
    n = dev.linear_i8_workspace(d)
    work = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear_i8(d, Ptr(X), Ptr(W), Ptr(ws), Ptr(Y), x_scale=Ptr(xs), bias=Ptr(B), residual=Ptr(Y if inplace else R), work=Ptr(work), work_bytes=n)
    dev.sync()
    z = whole_sum(q, W) * s.double()[:, None] * ws.double()
    off = 3.01 * U32 * z.abs()
    if bias:
        z = z + B.double()
        off = off + U32 * (z.abs() + off)
    want, off_y = act(z, a), 1.13 * off + 2.0**-21 * z.abs()
    if residual:
        want = want + r0
        off_y = off_y + U32 * (want.abs() + off_y)
    got = Y.clone()
    within(got, want, off_y + rounded(want.abs() + off_y, y), "Y")
    Y.fill_(5.0)
    assert bool((around == 5.0).all()), "values around Y"
    return got


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("int8", [True, False], ids=["int8", "values"])
def test_sizes(dev, size, int8):
    print("linear_i8", size, int8, flush=True)
    forward(dev, *size, t="bf16" if size[0] % 2 else "f16", a="gelu", int8=int8)


@pytest.mark.parametrize("size", LARGE, ids=str)
def test_large(dev, size):
    print("linear_i8", size, flush=True)
    forward(dev, *size, t="f16", a="silu", int8=False)
    forward(dev, *size, t="bf16", y="f32", bias=False, pad=6)


@pytest.mark.parametrize("size", [(1, 40, 131071), (5, 40, 131071), (20, 40, 131071), (300, 40, 131071)], ids=str)
def test_largest_sums(dev, size):
    """All bytes -128 or 127: sums next to int32's largest, and W alone at its lowest."""
    M, N, K = size
    for x, w in ((-128, -128), (127, -128), (127, 127)):
        X = torch.full((M, up4(K)), x, dtype=torch.int8, device="cuda:0")[:, :K]
        W = torch.full((N, up4(K)), w, dtype=torch.int8, device="cuda:0")[:, :K]
        print("linear_i8", size, x, w, flush=True)
        forward(dev, M, N, K, y="f32", bias=False, residual=False, X=X, W=W)


@pytest.mark.parametrize("pad,shift", [(8, 0), (5, 0), (0, 1), (16, 8), (3, 2)])
@pytest.mark.parametrize("size", [(1, 300, 512), (2, 301, 511), (9, 302, 1000), (20, 304, 1000), (300, 264, 520), (520, 1030, 257)], ids=str)
def test_windows(dev, size, pad, shift):
    print("linear_i8", size, pad, shift, flush=True)
    forward(dev, *size, pad=pad, shift=shift, a="silu", int8=False)
    forward(dev, *size, pad=pad, shift=shift, y="f32")


@pytest.mark.parametrize("a", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("y", ["bf16", "f32"])
@pytest.mark.parametrize("M", [1, 2, 3, 30, 200])
def test_epilogues(dev, a, y, M):
    for bias, residual in ((0, 0), (1, 0), (0, 1), (1, 1)):
        print("linear_i8 epilogue", M, a, y, bias, residual, flush=True)
        forward(dev, M, 328, 136, a=a, y=y, bias=bias, residual=residual, int8=bool(bias))


@pytest.mark.parametrize("M", [1, 2, 8, 40, 300])
def test_residual_in_place(dev, M):
    forward(dev, M, 264, 128, inplace=True)
    forward(dev, M, 264, 128, y="f32", inplace=True, int8=False)


@pytest.mark.parametrize("M", [1, 2, 9, 70, 520])
def test_what_is_not_finite_stays_in_its_row(dev, M):
    """A row of X with an infinity has no scale: its outputs are NaN, all others as without it."""
    N, K = 272, 200
    g = generator(3)
    X = torch.randn((M, K), device="cuda:0", generator=g).to(torch.bfloat16)
    W, ws = integers(g, N, K, 0), torch.rand(N, device="cuda:0", generator=g) * 0.01
    out = []
    for bad in (False, True):
        if bad:
            X[M // 2, 7] = float("inf")
        Y = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda:0")
        d = ozd.linear_i8_desc(M, N, K, "bf16", "gelu")
        n = dev.linear_i8_workspace(d)
        work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear_i8(d, Ptr(X), Ptr(W), Ptr(ws), Ptr(Y), work=Ptr(work), work_bytes=n)
        dev.sync()
        out.append(Y)
    assert bool(torch.isnan(out[1][M // 2]).all())
    keep = [m for m in range(M) if m != M // 2]
    assert torch.equal(out[0][keep].view(torch.int16), out[1][keep].view(torch.int16))


@pytest.mark.parametrize("size", [(1, 512, 1024), (2, 512, 1024), (12, 512, 4096), (64, 256, 8192), (700, 512, 640)], ids=str)
def test_quantized_by_the_call_or_before(dev, size):
    """Both ways give the same bits."""
    M, N, K = size
    g = generator(5)
    X = torch.randn((M, K), device="cuda:0", generator=g).to(torch.bfloat16)
    W, ws = integers(g, N, K, 0), torch.rand(N, device="cuda:0", generator=g) * 0.01
    q, s = torch.zeros((M, K), dtype=torch.int8, device="cuda:0"), torch.zeros(M, device="cuda:0")
    torch.cuda.synchronize()
    dev.quantize_rows(ozd.quantize_desc(M, K), Ptr(X), Ptr(q), Ptr(s))
    out = []
    for int8 in (False, True):
        Y = torch.zeros((M, N), device="cuda:0")
        d = ozd.linear_i8_desc(M, N, K, "bf16", "silu", "f32", x_int8=int8)
        n = dev.linear_i8_workspace(d)
        work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear_i8(d, Ptr(q if int8 else X), Ptr(W), Ptr(ws), Ptr(Y), x_scale=Ptr(s) if int8 else None, work=Ptr(work), work_bytes=n)
        dev.sync()
        out.append(Y)
    assert torch.equal(out[0].view(torch.int32), out[1].view(torch.int32))


def test_refusals(dev):
    g = generator(1)
    W, ws, Y = integers(g, 8, 16, 0), torch.ones(8, device="cuda:0"), torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda:0")
    X = torch.zeros((4, 16), dtype=torch.bfloat16, device="cuda:0")
    d = ozd.linear_i8_desc(4, 8, 16)
    n = dev.linear_i8_workspace(d)
    work = torch.zeros(n + 16, dtype=torch.uint8, device="cuda:0")
    q = ozd.linear_i8_desc(4, 8, 16, x_int8=True)
    ok = dict(work=Ptr(work), work_bytes=n)
    for call, text in ((lambda: dev.linear_i8(d, Ptr(X), Ptr(W), Ptr(ws), Ptr(Y)), "workspace"),
                       (lambda: dev.linear_i8(d, Ptr(X), Ptr(W), Ptr(ws), Ptr(Y), work=Ptr(work[4:]), work_bytes=n), "workspace"),
                       (lambda: dev.linear_i8(d, Ptr(X), Ptr(W.view(-1)[2:]), Ptr(ws), Ptr(Y), **ok), "multiples of 4"),
                       (lambda: dev.linear_i8(q, Ptr(W.view(-1)[2:]), Ptr(W), Ptr(ws), Ptr(Y), x_scale=Ptr(ws), **ok), "multiples of 4"),
                       (lambda: dev.linear_i8(q, Ptr(W), Ptr(W), Ptr(ws), Ptr(Y), **ok), "null"),
                       (lambda: dev.linear_i8(d, Ptr(X), Ptr(W), Ptr(None), Ptr(Y), **ok), "null"),
                       (lambda: dev.linear_i8(ozd.linear_i8_desc(4, 8, 16, ldr=9), Ptr(X), Ptr(W), Ptr(ws), Ptr(Y), residual=Ptr(Y), **ok), "residual")):
        with pytest.raises(RuntimeError, match=text):
            call()
    dev.linear_i8(ozd.linear_i8_desc(0, 8, 16), Ptr(None), Ptr(W), Ptr(ws), Ptr(None))
    dev.sync()
