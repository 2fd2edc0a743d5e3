"""Rows of 8-bit layers that take the kernel of few rows: how many ranges of k the rule cuts."""
import ctypes

import pytest

from oztt_amd import device as ozd
from oztt_amd import hip
from tests.linear_i8_cases import RANGES, way


@pytest.mark.parametrize("size", RANGES, ids=str)
def test_ranges(size):
    route, splits = way(*size)
    assert route == -1 and splits > 1


@pytest.mark.parametrize("N,K", [(64, 32768), (512, 16448), (16, 16385), (1000, 20000), (4096, 32000)])
def test_one_and_two_rows_have_the_ranges_of_three(N, K):
    """Beyond the length that is streamed; one range would leave 16 rows of W to a workgroup, 4 workgroups for 64."""
    assert way(1, N, K) == way(2, N, K) == way(3, N, K)


def test_workspace_holds_the_ranges():
    for M, N, K in RANGES:
        d = ozd.linear_i8_desc(M, N, K, x_int8=True, ldx=-(-K // 4) * 4, ldw=-(-K // 4) * 4)
        assert hip().oz_linear_i8_workspace(None, ctypes.byref(d)) >= 4 * way(M, N, K)[1] * M * N
