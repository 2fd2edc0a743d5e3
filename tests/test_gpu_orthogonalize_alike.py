"""oz_orthogonalize of matrices whose values are alike, so that their roundings are and do not average: blocks of one value along the diagonal. Each
has one singular value, and the result is the matrix times a factor.

Products of 22 bits. A sum of n values alike takes 3 n / 32 additions (the matrix instructions', three products), each rounded to nearest, by up to 2^-24 of a sum
that is half of the last one on average: off by up to n 2^-28.4. With A's sum over the long side's n values and A^2's and B X's over the short side's m,
s' = s p(q), p = a + b q + c q^2, q = s^2, a step adds (|b q + 2 c q^2| n + (|c| q^2 + |b q + c q^2|) m) / |p| of that to the result's relative error and
multiplies what there was by |a + 3 b q + 5 c q^2| / |p|. From s = 1 on five steps with the usual factors come to 4.9 n + 33 m, that is
(0.3 n + 1.6 m) 2^-24; the bound taken is (n + 2 m) 2^-24 beside the 1e-5 of roundings that average. The second parts of A and B have to be there in
full for it: with values below FP16's normal ones the blocks are off by 3.5e-5 to 7.5e-5."""
import math

import pytest
import torch

from oztt_amd import device as ozd
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
