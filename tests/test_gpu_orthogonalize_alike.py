"""oz_orthogonalize of matrices whose values are alike, so that their roundings are and do not average: blocks of one value along the diagonal. Each
has one singular value, and the result is the matrix times a factor.

Products of 22 bits. A sum of n values alike takes 3 n / 32 additions (the matrix instructions', three products), each rounded to nearest, by up to 2^-24 of a sum
that is half of the last one on average: off by up to n 2^-28.4. With A's sum over the long side's n values and A^2's and B X's over the short side's m,
s' = s p(q), p = a + b q + c q^2, q = s^2, a step adds (|b q + 2 c q^2| n + (|c| q^2 + |b q + c q^2|) m) / |p| of that to the result's relative error and
multiplies what there was by |a + 3 b q + 5 c q^2| / |p|. From s = 1 on five steps with the usual factors come to 4.9 n + 33 m, that is
(0.3 n + 1.6 m) 2^-24; the bound taken is (n + 2 m) 2^-24 beside the 1e-5 of roundings that average. The second parts of A and B have to be there in
full for it: with values below FP16's normal ones the blocks are off by 3.5e-5 to 7.5e-5.

Products of 11 bits. To first order FP16's half step, 2^-11, comes in from X twice and from A in (b q + 2 c q^2) / p, and from X and B in (b q + c q^2) / p
(alike()); the header's 6.2e-2 is the largest sum of five steps over all numbers of blocks."""
import math

import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import generator
from tests.test_gpu_newton_schulz_bits import updates
from tests.test_gpu_orthogonalize import check, exact, gaussian, rounding_of_x, run

pytestmark = pytest.mark.gpu


def blocks(rows, cols, p, value=0.37, t="f32"):
    G = torch.zeros((1, rows * p, cols * p), device="cuda:0")
    for i in range(p):
        G[0, i * rows : (i + 1) * rows, i * cols : (i + 1) * cols] = value
    return G.to({"f32": torch.float32, "f16": torch.float16}[t])


def factor(G, rows, cols, p, steps=5, factors=ozd.NEWTON_SCHULZ, eps=1e-7):
    """The block's value in 64 bits."""
    a, b, c = factors
    v = float(G[0, 0, 0])
    s = v * math.sqrt(rows * cols) / (v * math.sqrt(rows * cols * p) + eps)
    for _ in range(steps):
        s = a * s + b * s**3 + c * s**5
    return s / math.sqrt(rows * cols)


def bound(rows, cols):
    return 1e-5 + 2.0**-24 * (max(rows, cols) + 2 * min(rows, cols))


def off(got, G, value):
    want = (G != 0).double() * value
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("size", [(128, 42, 4), (255, 168, 4), (255, 500, 2), (42, 128, 7), (11, 13, 40), (3, 200, 90), (333, 333, 3)], ids=str)
def test_blocks(dev, size):
    print("blocks", size, flush=True)
    G = blocks(*size)
    assert off(run(dev, G, "f32"), G, factor(G, *size)) <= bound(*size[:2])


@pytest.mark.parametrize("size", [(100, 140), (700, 1500), (1869, 1869), (1348, 2006), (2638, 5276), (64, 8191), (8191, 64), (1, 100003), (600, 100003)], ids=str)
def test_one_value(dev, size):
    print("one value", size, flush=True)
    G = blocks(*size, 1)
    assert off(run(dev, G, "f32"), G, factor(G, *size, 1)) <= bound(*size[:2])


@pytest.mark.parametrize("f,steps", [((1.5, 0.5, 0.0), 2), ((7.5, 0.25, 0.125), 1), ((1.0, 0.0, 0.0), 3), ((1.2, 0.0, 0.1), 2), ((1.25, 0.0, -0.25), 4)], ids=str)
def test_other_factors(dev, f, steps):
    """Singular values that grow to 7, as the factors allow; factors that leave parts out."""
    print("factors", f, steps, flush=True)
    for size in ((100, 140, 1), (33, 20, 3)):
        G = blocks(*size)
        assert off(run(dev, G, "f32", steps=steps, coefficients=f), G, factor(G, *size, steps, f)) <= bound(*size[:2])
    G = gaussian(1, 200, 260, "f32")
    check(run(dev, G, "f32", steps=steps, coefficients=f), exact(G, steps, f), 1e-5, "f32", rounding_of_x(steps, f[0]))


def alike(p, steps=5, factors=ozd.NEWTON_SCHULZ):
    """Bound of the relative error of p equal singular values in products of 11 bits."""
    a, b, c = factors
    s, e = p**-0.5, 0.0
    for _ in range(steps):
        q = s * s
        f = a + b * q + c * q * q
        e = abs((a + 3 * b * q + 5 * c * q * q) / f) * e + (3 * abs((b * q + 2 * c * q * q) / f) + 2 * abs((b * q + c * q * q) / f)) * 2.0**-11
        s *= f
    return e


def test_what_the_header_promises():
    assert max(alike(p) for p in range(1, 8193)) <= 6.2e-2


@pytest.mark.parametrize("size", [(2638, 5276, 1), (2717, 1418, 1), (1024, 1024, 1), (354, 325, 2), (677, 131, 4), (260, 270, 4), (43, 220, 13), (43, 55, 13), (24, 28, 30)], ids=str)
def test_blocks_in_11_bits(dev, size):
    print("blocks, 11 bits", size, flush=True)
    G = blocks(*size)[0]
    assert min(G.shape) > 512
    assert off(updates(dev, G, False), G, factor(G[None], *size)) <= 1.1 * alike(size[2]) + bound(*size[:2])
    assert off(updates(dev, G, True), G, factor(G[None], *size)) <= bound(*size[:2])


@pytest.mark.parametrize("equal,rest", [(1024, 0.0), (64, 0.0), (256, 0.01)], ids=str)
def test_equal_rows_in_11_bits(dev, equal, rest):
    """One strong direction; what the others hold adds the error of values that differ."""
    print("equal rows", equal, rest, flush=True)
    g = generator(2)
    G = rest * torch.randn((1024, 1400), device="cuda:0", generator=g)
    G[:equal] = torch.randn((1, 1400), device="cuda:0", generator=g)
    want = exact(G[None])[0]
    relative = lambda got: float((got - want).norm() / want.norm())  # noqa: E731
    assert relative(updates(dev, G, False)) <= 1.1 * alike(1) + (2e-3 if rest else 0.0) + bound(1024, 1400)
    assert relative(updates(dev, G, True)) <= bound(1024, 1400) + rounding_of_x() / float(want.norm())


def test_identity_and_noise_in_11_bits(dev):
    G = torch.eye(513, device="cuda:0") + 1e-3 * torch.randn((513, 513), device="cuda:0", generator=generator(3))
    want = exact(G[None])[0]
    assert float((updates(dev, G, False) - want).norm() / want.norm()) <= 1.1 * alike(513) + 2e-3


def test_bf16_matrix_of_one_value(dev):
    """Through oz_orthogonalize itself: its rounding to BF16 beside the bound, which `exact` takes to that of 22 bits."""
    G = torch.full((1, 2717, 1418), 0.37, device="cuda:0", dtype=torch.bfloat16)
    value = factor(G, 2717, 1418, 1)
    half = torch.finfo(torch.bfloat16).eps / 2
    assert off(run(dev, G, "bf16"), G, value) <= 1.1 * alike(1) + half
    assert off(run(dev, G, "bf16", exact=True), G, value) <= bound(2717, 1418) + half
