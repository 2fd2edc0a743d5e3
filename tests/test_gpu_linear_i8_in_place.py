"""The residual is Y itself where a row's last pieces of 8 outputs overlap: each output adds it once, whatever the tile."""
import pytest

from tests.linear_i8_cases import way
from tests.test_gpu_linear_i8 import forward

pytestmark = pytest.mark.gpu

SIZES = [(40, 1030, 257), (24, 8187, 520), (300, 263, 520), (1000, 701, 1500), (2050, 2043, 4100), (3500, 3505, 4100), (40, 5999, 4096), (300, 261, 131071), (17, 9, 64), (33, 7, 100), (600, 1, 40)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_odd_rows(dev, size):
    print("linear_i8 in place", size, way(*size), flush=True)
    forward(dev, *size, inplace=True, a="relu", int8=False)
    forward(dev, *size, inplace=True, y="f32", pad=3)
    forward(dev, *size, t="f16", inplace=True, pad=5, shift=1, bias=False)


def test_every_way_is_there():
    assert {way(*s)[0] for s in SIZES} >= {0, 1, 2, 3, 4}
