"""The tiles of the Newton-Schulz products at the sizes that the GPU tests take for them, and those of the routes of 8-bit layers."""
import ctypes

import pytest

from oztt_amd import hip
from tests.newton_schulz_cases import BOTH, ONE, tiles


@pytest.mark.parametrize("three", [0, 1])
def test_tiles(three):
    for (phase, tall, tile, rest), (count, rows, cols) in (BOTH if three else ONE).items():
        assert (rows > cols) == bool(tall)
        assert tiles(phase, count, rows, cols, three) == (tile, rest), (phase, count, rows, cols)


def test_every_size_has_a_tile():
    for three in (0, 1):
        for count, rows, cols in ((1, 1, 1), (100000, 16, 16), (1, 1, 2**20), (1, 2**20, 1), (1, 8192, 8192), (1, 90000, 90000)):
            for phase in range(3):
                for cus in (1, 64, 256, 304):
                    tile, rest = tiles(phase, count, rows, cols, three, cus)
                    assert tile in ((64, 128) if three else (64, 128, 256)) and rest in (0, 64, 128) and rest < tile


def test_linear_i8():
    def way(M, N, K):
        s = ctypes.c_int()
        return hip().oz_rule_linear_i8(256, M, N, K, ctypes.byref(s)), s.value

    assert way(1, 8192, 8192)[0] == way(2, 1, 16384)[0] == -2
    assert way(2, 64, 16385)[0] == way(3, 64, 128)[0] == way(16, 4096, 8192)[0] == way(4, 100000, 4096)[0] == -1
    assert way(5, 4097, 8192)[0] >= 0 and way(3, 64, 32769)[0] >= 0 and way(17, 64, 128)[0] >= 0
    assert way(8, 512, 8192)[1] > 1 and way(300, 260, 131071)[1] > 1
    assert {way(*s)[0] for s in ((8192, 8192, 8192), (2050, 2043, 32766), (1000, 700, 1500), (40, 6000, 4096), (24, 8192, 2048))} == {0, 1, 2, 3, 4}
