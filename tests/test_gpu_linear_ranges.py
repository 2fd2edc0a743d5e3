"""oz_linear, oz_linear_grad and oz_adamw_step past 32-bit offsets: leading dimensions of 2^22, the largest taken, operands past 4 GiB,
and one tensor of more than 2^32 values. Bounds as for small sizes."""
import ctypes

import numpy as np
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, U32, Ptr, generator, rounded, within
from tests.test_gpu_adamw import BLOCK, decode, encode, expected, same

pytestmark = pytest.mark.gpu

LD = 2**22


@pytest.fixture(autouse=True)
def memory():
    """Up to 100 GB a test are given back."""
    yield
    torch.cuda.empty_cache()


def wide(rows, cols, t, g, scale=1.0):
    """A matrix whose rows are 2^22 values apart, NaN between them."""
    base = torch.full((rows * LD,), float("nan"), dtype=DTYPE[t], device="cuda:0")
    w = base.view(rows, LD)[:, :cols]
    w.copy_((scale * torch.randn((rows, cols), device="cuda:0", generator=g)).to(DTYPE[t]))
    return w


def tile_of(M, N, K, contiguous=1):
    return ozd.hip().oz_rule_linear_route(256, *(ctypes.c_longlong(v) for v in (M, N, K)), contiguous, 1, None)


# streamed rows, few rows, and tiles of every size (the largest alone with wide rows of X and W)
@pytest.mark.parametrize("M,N,K,tile,outputs", [(1, 1100, 72, -1, True), (16, 1040, 520, -1, True), (520, 40, 136, None, True), (1040, 264, 72, None, True),
                                                (1030, 700, 1500, 2, False), (2048, 2048, 512, 1, False), (3300, 3900, 2048, 0, False)], ids=str)
def test_linear(dev, M, N, K, tile, outputs):
    print("linear ld", M, N, K, flush=True)
    assert tile is None or tile_of(M, N, K) == tile
    g = generator(M)
    X, W = wide(M, K, "bf16", g), wide(N, K, "bf16", g, K**-0.5)
    Y = wide(M, N, "f32", g) if outputs else torch.zeros((M, N), device="cuda:0")
    R = Y.double()
    d = ozd.linear_desc(M, N, K, "bf16", "none", "f32", ldx=LD, ldw=LD, ldy=LD if outputs else 0, ldr=LD if outputs else 0)
    n = dev.linear_workspace(d)
    work = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear(d, Ptr(X), Ptr(W), Ptr(Y), residual=Ptr(Y), work=Ptr(work), work_bytes=n)
    dev.sync()
    x, w = X.double(), W.double()
    want = x @ w.T + R
    within(Y, want, (K + 2) * U32 * (x.abs() @ w.abs().T) + 2 * U32 * want.abs(), "Y")


@pytest.mark.parametrize("M,N,K,tiles", [(520, 300, 200, None), (3500, 3500, 3500, (0,))], ids=str)
def test_linear_grad(dev, M, N, K, tiles):
    print("linear_grad ld", M, N, K, flush=True)
    g = generator(M)
    dY, X, W = wide(M, N, "f16", g), wide(M, K, "f16", g), wide(N, K, "f16", g)
    assert tiles is None or (tile_of(M, K, N, 0) in tiles and tile_of(N, K, M, 0) in tiles)
    dX, dW = torch.zeros((M, K), dtype=torch.float16, device="cuda:0"), torch.zeros((N, K), device="cuda:0")
    dB = torch.zeros(N, device="cuda:0")
    d = ozd.linear_grad_desc(M, N, K, "f16", "none", "f32", lddy=LD, ldx=LD, ldw=LD)
    n = dev.linear_grad_workspace(d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.linear_grad(d, Ptr(dY), Ptr(X), Ptr(W), dX=Ptr(dX), dW=Ptr(dW), dbias=Ptr(dB), work=Ptr(work), work_bytes=n)
    dev.sync()
    y, x, w = dY.double(), X.double(), W.double()
    for got, p, q, k, t in ((dX, y, w, N, "f16"), (dW, y.T, x, M, "f32")):
        want, bound = p @ q, (k + 2) * U32 * (p.abs() @ q.abs())
        within(got, want, bound + rounded(want.abs() + bound, t), t)
    within(dB, y.sum(0), (M + 2) * U32 * y.abs().sum(0), "dbias")


def test_adamw_of_more_than_2_32_values(dev):
    """One tensor with states in 8 bits; its last values, whose places in the hash went round 2^32, against the host's sequence, and
    blocks on either side of 2^31 and 2^32 values. The rest has zero gradients and stays zero."""
    n = 2**32 + 20000 - 7
    print("adamw", n, flush=True)
    zeros = lambda k, t: torch.zeros(k, dtype=t, device="cuda:0")  # noqa: E731
    t = {"param": zeros(n, torch.bfloat16), "grad": zeros(n, torch.bfloat16), "m": zeros(n, torch.uint8), "v": zeros(n, torch.uint8),
         "m_scale": zeros(-(-n // BLOCK), torch.uint8), "v_scale": zeros(-(-n // BLOCK), torch.uint8)}
    g = generator(1)
    spans = [(2**31 - 4096, 2**31 + 4096), (2**32 - 8192, n)]
    before = []
    for a, b in spans:
        k = b - a
        t["param"][a:b] = (0.05 * torch.randn(k, device="cuda:0", generator=g)).bfloat16()
        t["grad"][a:b] = torch.randn(k, device="cuda:0", generator=g).bfloat16()
        half = np.full(k, 0.5, dtype=np.float32)
        x = {"param": t["param"][a:b].float().cpu().numpy(), "grad": t["grad"][a:b].float().cpu().numpy(), "master": None, "decay": 0.1}
        for s, root in (("m", False), ("v", True)):
            v = (0.3 * torch.randn(k, device="cuda:0", generator=g)).abs().cpu().numpy()
            x[s], x[s + "_scale"] = encode(v, half, root)
            t[s][a:b] = torch.from_numpy(x[s]).cuda()
            t[s + "_scale"][a // BLOCK : a // BLOCK + len(x[s + "_scale"])] = torch.from_numpy(x[s + "_scale"]).cuda()
        before.append(x)
    o = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.99, "eps": 1e-8, "step": 3, "seed": 987654321, "grad_scale": 1.0}
    p = {k: v.data_ptr() for k, v in t.items()}
    plan = dev.adamw_plan([ozd.adamw_tensor(n, p["param"], p["grad"], p["m"], p["v"], 0, p["m_scale"], p["v_scale"], "bf16", "bf16", 0.1)], 8)
    torch.cuda.synchronize()
    dev.adamw_step(plan, o["lr"], o["beta1"], o["beta2"], o["eps"], o["step"], o["seed"])
    dev.sync()
    for (a, b), x in zip(spans, before):
        want = expected(x, o, 8, a // BLOCK)
        for s in ("m", "v"):
            same(t[s][a:b].cpu().numpy(), want[s], s)
            same(t[s + "_scale"][a // BLOCK : a // BLOCK + len(want[s + "_scale"])].cpu().numpy(), want[s + "_scale"], s + "_scale")
        assert torch.equal(t["param"][a:b].cpu(), torch.from_numpy(want["p"]).bfloat16())
        for k in ("param", "m", "v"):
            t[k][a:b] = 0
    assert not any(bool(t[k].any()) for k in ("param", "m", "v"))
    assert decode(t["m"][:64].cpu().numpy(), t["m_scale"][:1].cpu().numpy()).sum() == 0
