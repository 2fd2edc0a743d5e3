"""The rule by which a product with an epilogue takes its kernel, tile and ranges of c (oz_linear.hip), on 256 compute units, at
sizes on either side of its lines; every choice was measured against the others at the size given. CPU only."""
import ctypes

import pytest

from oztt_amd.device import hip

FEW, T256, T128, T64, T64X32, T32 = -1, 0, 1, 2, 3, 4


def route(nq, np, C, contiguous=1, even=1):
    s = ctypes.c_int()
    ll = ctypes.c_longlong
    t = hip().oz_rule_linear_route(256, ll(nq), ll(np), ll(C), contiguous, even, ctypes.byref(s))
    return t, s.value


@pytest.mark.parametrize("size,want", [
    ((1, 8192, 8192), (FEW, 1)), ((2, 128, 8192), (FEW, 1)), ((3, 512, 8192), (FEW, 4)), ((16, 8192, 8192), (FEW, 1)),
    ((17, 8192, 8192), (T32, 1)), ((20, 8192, 8192), (T32, 1)), ((24, 8192, 2048), (T32, 1)), ((128, 2048, 2048), (T32, 1)),
    ((300, 300, 304), (T32, 1)), ((200, 4096, 1024), (T64, 1)), ((1000, 704, 1504), (T64, 1)), ((1024, 1024, 1024), (T64, 1)),
    ((256, 1024, 8192), (T64, 4)), ((512, 8192, 2048), (T128, 1)), ((2048, 2048, 512), (T128, 1)), ((2048, 2048, 2048), (T128, 1)),
    ((2048, 4096, 4096), (T128, 1)), ((4096, 4096, 1024), (T128, 1)), ((8192, 8192, 512), (T128, 1)), ((3500, 3500, 3500), (T256, 1)),
    ((4096, 4096, 4096), (T256, 1)), ((8192, 2048, 8192), (T256, 1)), ((8192, 8192, 2048), (T256, 1)),
], ids=str)
def test_forward(size, want):
    assert route(*size) == want


def test_odd_rows():
    """Operands whose rows begin at odd addresses: up to 32 rows by the kernel that reads them in place, more laid out first."""
    assert route(17, 1000, 999, even=0)[0] == FEW and route(32, 1000, 999, even=0)[0] == FEW
    assert route(33, 1000, 999, even=0)[0] != FEW
    # gradients' operands run along their own index: always tiles
    assert route(1, 1000, 999, contiguous=0)[0] != FEW


@pytest.mark.parametrize("size,tile", [((8192, 2048, 24), T128), ((512, 512, 8192), T64), ((1504, 704, 1000), T64), ((2048, 2048, 2048), T128),
                                       ((8192, 2048, 8192), T256), ((1024, 1024, 4096), T64)], ids=str)
def test_gradients(size, tile):
    t, splits = route(*size, contiguous=0)
    assert t == tile and (splits > 1) == (size == (512, 512, 8192))
