"""oz_orthogonalize against the iteration in 64 bits.

The bounds are what the header promises of the result before its last rounding, of its norm: 1e-5 with products of 22 bits, 2e-3 with
products of 11 (BF16 and more than 512 rows and columns). Where they come from: rounding to FP16 is off by at most 2^-11 of a value, 1.2e-4 in the mean
square; each of the five steps rounds A, B and X and multiplies what there was by at most 3.5, and by 0.7 to 1.8 where values are near 1. The same
steps with the same roundings in 64 bits, over Gaussian, power-law and low-rank matrices, were off by 1e-4 to 2e-3 and, with two parts,
by up to 8e-6. To that comes what rounding X itself to 22 bits leaves in directions where X has next to nothing: a step multiplies
them by a, and X's norm by a at most, so the rounding of each step arrives at the end as at most a^steps 2^-22 of |X0| = 1; the roundings of
different steps are independent and add up by their squares, a^steps 2^-22 sqrt(steps), 1.3e-4. (A matrix of 9 strong directions out of 128 and noise: 5.8e-5
of a result of norm 5.4.) Single values are held to 20 times the bound of the root mean square: a wrong tile, part or transposition is off by 1."""
import math

import pytest
import torch

from oztt_amd import device as ozd
from tests.newton_schulz_cases import BOTH, ONE
from tests.operator_cases import DTYPE, ROUND, Ptr, generator

pytestmark = pytest.mark.gpu

A, B, C = ozd.NEWTON_SCHULZ


def exact(G, steps=5, factors=(A, B, C), eps=1e-7):
    a, b, c = factors
    X = G.double()
    norm = X.square().sum((1, 2), keepdim=True).sqrt()
    X = torch.where(norm > 0, X / (norm + eps), torch.zeros_like(X))
    tall = X.shape[1] > X.shape[2]
    if tall:
        X = X.transpose(1, 2).contiguous()
    for _ in range(steps):
        S = torch.matmul(X, X.transpose(1, 2).contiguous())
        X = a * X + torch.matmul(b * S + c * torch.matmul(S, S), X)
    return X.transpose(1, 2) if tall else X


def bound_of(shape, t):
    return 2e-3 if t == "bf16" and min(shape[1:]) > 512 else 1e-5


def run(dev, G, t, inplace=False, ldo=0, **options):
    """G: count x rows x cols, possibly a window."""
    count, rows, cols = G.shape
    ldo = ldo or cols
    base = torch.full((count, rows, ldo), 5.0, dtype=DTYPE[t], device="cuda:0")
    O = G if inplace else base[:, :, :cols]
    d = ozd.orthogonalize_desc(rows, cols, count, t, ldg=G.stride(1), ldo=O.stride(1), stride_g=G.stride(0), stride_o=O.stride(0), **options)
    n = dev.orthogonalize_workspace(d)
    work = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.orthogonalize(d, Ptr(G), Ptr(O), Ptr(work), n)
    dev.sync()
    got = O.clone()
    if not inplace:
        O.fill_(5.0)
        assert bool((base == 5.0).all()), "values around O"
    return got


def rounding_of_x(steps=5, a=A):
    return max(a, 1.0) ** steps * 2.0**-22 * steps**0.5


def check(got, want, bound, t, x=rounding_of_x()):
    for i in range(len(want)):
        g, w = got[i].double(), want[i]
        norm = float(w.norm())
        bound_i, bound = bound, bound + x / norm
        rms = norm / math.sqrt(w.numel())
        half, floor = ROUND[t]
        off = float((g - w).norm())
        assert off <= bound * norm + half * norm + floor * math.sqrt(w.numel()), (i, off / norm)
        worst = float(((g - w).abs() - half * (1 + 20 * bound) * w.abs()).max())
        assert worst <= (20 * bound * (1 + half)) * max(rms, float(w.abs().max()) / 20) + floor, (i, worst / rms)
        bound = bound_i


def gaussian(count, rows, cols, t, seed=1):
    return torch.randn((count, rows, cols), device="cuda:0", generator=generator(seed)).to(DTYPE[t])


def low_rank(count, rows, cols, t, seed=1):
    g = generator(seed)
    k = 1 + min(rows, cols) // 16
    x = torch.matmul(torch.randn((count, rows, k), device="cuda:0", generator=g), torch.randn((count, k, cols), device="cuda:0", generator=g)) / k**0.5
    return (x + 0.01 * torch.randn((count, rows, cols), device="cuda:0", generator=g)).to(DTYPE[t])


SIZES = [(1, 1, 1), (3, 1, 5), (2, 5, 1), (1, 1, 1000), (1, 300, 2), (4, 3, 3), (2, 16, 64), (2, 64, 64), (1, 65, 64), (3, 63, 130), (1, 128, 512),
         (2, 512, 128), (1, 200, 200), (1, 129, 257), (1, 257, 129), (1, 16, 4100), (1, 2500, 40), (2, 500, 700), (1, 513, 515), (1, 700, 640), (1, 1030, 520)]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(dev, size, t):
    for make in (gaussian, low_rank):
        print("orthogonalize", size, t, make.__name__, flush=True)
        G = make(*size, t)
        check(run(dev, G, t), exact(G), bound_of(size, t), t)


LARGE = [(1, 1500, 2100), (1, 2100, 1500), (2, 1024, 1024), (1, 2048, 520), (1, 600, 8200), (1, 3500, 3500)]


@pytest.mark.parametrize("size", LARGE, ids=str)
def test_large(dev, size):
    for t in ("bf16", "f16"):
        print("orthogonalize", size, t, flush=True)
        G = low_rank(*size, t)
        check(run(dev, G, t), exact(G), bound_of(size, t), t)


@pytest.mark.parametrize("pad", [1, 8, 37])
@pytest.mark.parametrize("size", [(3, 70, 90), (2, 130, 65), (2, 520, 600)], ids=str)
def test_windows(dev, size, pad):
    print("orthogonalize window", size, pad, flush=True)
    count, rows, cols = size
    for t in ("f32", "bf16"):
        w = torch.full((count, rows + 3, cols + pad), float("nan"), dtype=DTYPE[t], device="cuda:0")
        G = w[:, 1 : rows + 1, pad // 2 : pad // 2 + cols]
        G.copy_(gaussian(count, rows, cols, t))
        check(run(dev, G, t, ldo=cols + pad), exact(G), bound_of(size, t), t)


@pytest.mark.parametrize("size", [(2, 100, 70), (1, 520, 530)], ids=str)
def test_in_place(dev, size):
    for t in ("f32", "bf16"):
        G = gaussian(*size, t)
        want = exact(G)
        check(run(dev, G, t, inplace=True), want, bound_of(size, t), t)


@pytest.mark.parametrize("size", [(40, 70), (600, 520)], ids=str)
def test_what_matrices_may_hold(dev, size):
    """Zeros, values near both ends of FP32, one value that is not finite, one that is not zero: each matrix by itself."""
    rows, cols = size
    G = gaussian(7, rows, cols, "f32")
    G[1] = 0
    G[2] *= 1e-38
    G[3] *= 5e37
    G[4, rows - 1, 0] = float("inf")
    G[5, 0, cols - 1] = float("nan")
    G[6] = 0
    G[6, rows // 2, cols // 2] = -2.0
    got = run(dev, G, "f32", eps=0.0)
    assert bool((got[1] == 0).all()) and bool(torch.isnan(got[4:6]).all())
    for i in (0, 2, 3, 6):
        check(got[i : i + 1], exact(G[i : i + 1], eps=0.0), 1e-5, "f32")


@pytest.mark.parametrize("size", [(1, 96, 160), (1, 640, 530)], ids=str)
def test_other_factors_and_steps(dev, size):
    """Factors that converge to 1 itself, and their result after many steps: rows that are orthogonal."""
    G = gaussian(*size, "f32", seed=4)
    for steps in (1, 2, 12):
        f = (15 / 8, -10 / 8, 3 / 8)
        got = run(dev, G, "f32", steps=steps, coefficients=f)
        check(got, exact(G, steps, f), 1e-5, "f32", rounding_of_x(steps, f[0]))


def test_the_norm_has_its_eps(dev):
    G = gaussian(1, 64, 80, "f32")
    check(run(dev, G, "f32", eps=50.0, steps=2), exact(G, 2, eps=50.0), 1e-5, "f32")


def test_the_same_bits_again(dev):
    for size, t in (((3, 200, 300), "f32"), ((1, 1100, 900), "bf16")):
        G = low_rank(*size, t)
        a, b = run(dev, G, t), run(dev, G, t)
        assert torch.equal(a, b)


def test_refusals(dev):
    G = gaussian(1, 8, 8, "f32")
    d = ozd.orthogonalize_desc(8, 8, 1, "f32")
    n = dev.orthogonalize_workspace(d)
    work = torch.zeros(n + 16, dtype=torch.uint8, device="cuda:0")
    for call, text in ((lambda: dev.orthogonalize(d, Ptr(G), Ptr(G), Ptr(work), n - 1), "workspace"), (lambda: dev.orthogonalize(d, Ptr(G), Ptr(G)), "workspace"),
                       (lambda: dev.orthogonalize(d, Ptr(None), Ptr(G), Ptr(work), n), "null"),
                       (lambda: dev.orthogonalize(ozd.orthogonalize_desc(8, 8, 1, "f32", ldo=9), Ptr(G), Ptr(G), Ptr(work), n), "other strides")):
        with pytest.raises(RuntimeError, match=text):
            call()
    dev.orthogonalize(ozd.orthogonalize_desc(8, 8, 0, "f32"), Ptr(None), Ptr(None))
    dev.sync()


@pytest.mark.parametrize("size", sorted(set(ONE.values())), ids=str)
def test_every_tile(dev, size):
    print("orthogonalize", size, "bf16", flush=True)
    G = low_rank(*size, "bf16")
    check(run(dev, G, "bf16"), exact(G), bound_of(size, "bf16"), "bf16")


@pytest.mark.parametrize("size", sorted(set(BOTH.values())), ids=str)
def test_every_tile_of_both_parts(dev, size):
    print("orthogonalize", size, "f32", flush=True)
    G = low_rank(*size, "f32")
    check(run(dev, G, "f32"), exact(G), bound_of(size, "f32"), "f32")


def test_offsets_past_32_bits(dev):
    """2^31 values and more in one matrix, wide and tall: one step, sampled, against A summed in 64 bits piece by piece."""
    short, long = 2100, 2**20
    for tall in (False, True):
        print("orthogonalize", "tall" if tall else "wide", short, long, flush=True)
        rows, cols = (long, short) if tall else (short, long)
        G = torch.empty((1, rows, cols), dtype=torch.bfloat16, device="cuda:0").normal_(generator=generator(7))
        got = run(dev, G, "bf16", steps=1, inplace=False)[0]
        S, squares = torch.zeros((short, short), dtype=torch.float64, device="cuda:0"), 0.0
        pieces = range(0, long, 2**17)
        part = lambda i, n=2**17: (G[0, i : i + n].double().T if tall else G[0][:, i : i + n].double())  # noqa: E731
        for i in pieces:
            x = part(i)
            squares += float(x.square().sum())
            S += x @ x.T
        norm = squares**0.5 + 1e-7
        S /= norm**2
        P = A * torch.eye(short, dtype=torch.float64, device="cuda:0") + B * S + C * (S @ S)
        for i in (0, 2**19 - 64, long - 128):
            want = P @ part(i, 128) / norm
            o = got[i : i + 128].T if tall else got[:, i : i + 128]
            check(o[None], want[None], 2e-3, "bf16", 0.0)
        del G, got
        torch.cuda.empty_cache()
