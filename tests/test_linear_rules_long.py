"""The rule of the linear layers where c is long and tiles are few, on 256 compute units: there its estimate is too short, and the
choice is up to a fifth slower than the fastest (operands from memory: 73 us where 128 x 128 tiles in 4 ranges take 64, 96 where 256
x 256 in 4 take 81, 144 where 256 x 256 in 2 take 129). CPU only."""
import ctypes

import pytest

from oztt_amd.device import hip


@pytest.mark.parametrize("size,want", [((256, 8192, 8192), (2, 1)), ((512, 8192, 8192), (1, 2)), ((1024, 8192, 8192), (1, 1))], ids=str)
def test_choice(size, want):
    s = ctypes.c_int()
    t = hip().oz_rule_linear_route(256, *(ctypes.c_longlong(v) for v in size), 1, 1, ctypes.byref(s))
    assert (t, s.value) == want
