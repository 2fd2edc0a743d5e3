"""Sizes of 8-bit layers by their routes, for the tests of the rule and of the kernels."""
import ctypes

from oztt_amd import hip


def way(M, N, K):
    """-2 streamed, -1 the kernel of few rows, else the tile; and the ranges of k."""
    s = ctypes.c_int()
    return hip().oz_rule_linear_i8(256, M, N, K, ctypes.byref(s)), s.value


# the kernel of few rows with more than one range of k: whole units of 256 and ragged ones, one row to 16, few and many rows of W
RANGES = [(1, 64, 32768), (1, 512, 16448), (2, 300, 20001), (2, 17, 16387), (3, 64, 32767), (3, 1000, 8193), (7, 130, 5001), (12, 512, 4100), (16, 512, 8200),
          (16, 16, 4352), (5, 1, 30000), (4, 1000, 9999)]
