"""Sizes at which each tile of the Newton-Schulz products runs, alone and with a last round's own launch, of wide and of tall matrices."""
import ctypes

from oztt_amd import hip

GRAM, SQUARE, UPDATE = range(3)
# (phase, tall, tile, the rest's tile): count, rows, cols
ONE = {(GRAM, 1, 64, 0): (1, 600, 513), (GRAM, 1, 128, 0): (4, 1500, 1000), (GRAM, 1, 128, 64): (4, 2600, 2000), (GRAM, 1, 256, 0): (1, 5700, 5000),
       (GRAM, 1, 256, 64): (2, 4300, 4000), (GRAM, 1, 256, 128): (4, 4000, 3000), (GRAM, 0, 64, 0): (1, 513, 513), (GRAM, 0, 128, 0): (4, 1000, 1000),
       (GRAM, 0, 128, 64): (4, 2000, 2000), (GRAM, 0, 256, 0): (1, 5000, 5000), (GRAM, 0, 256, 64): (2, 4000, 4000), (GRAM, 0, 256, 128): (4, 3000, 3000),
       (SQUARE, 0, 256, 64): (2, 4000, 4000), (SQUARE, 0, 256, 128): (4, 3000, 3000), (SQUARE, 0, 128, 64): (4, 2000, 2000),
       (UPDATE, 1, 128, 0): (4, 1000, 513), (UPDATE, 1, 128, 64): (4, 4000, 513), (UPDATE, 1, 256, 0): (1, 4300, 3000), (UPDATE, 1, 256, 64): (1, 6000, 3000),
       (UPDATE, 1, 256, 128): (1, 5000, 4000), (UPDATE, 0, 128, 0): (4, 513, 1000), (UPDATE, 0, 128, 64): (4, 513, 4000), (UPDATE, 0, 256, 0): (1, 3000, 4300),
       (UPDATE, 0, 256, 64): (2, 3000, 3000), (UPDATE, 0, 256, 128): (1, 4300, 4300)}
BOTH = {(GRAM, 1, 64, 0): (1, 600, 513), (GRAM, 1, 128, 0): (4, 1500, 1000), (GRAM, 1, 128, 64): (4, 2000, 1500), (GRAM, 0, 64, 0): (1, 513, 513),
        (GRAM, 0, 128, 0): (4, 1000, 1000), (GRAM, 0, 128, 64): (4, 1500, 1500), (SQUARE, 0, 128, 64): (4, 1500, 1500), (UPDATE, 1, 128, 0): (4, 1000, 513),
        (UPDATE, 1, 128, 64): (4, 2000, 513), (UPDATE, 0, 128, 0): (4, 513, 1000), (UPDATE, 0, 128, 64): (4, 513, 2000)}


def tiles(phase, count, rows, cols, three, cus=256):
    rest = ctypes.c_int()
    t = hip().oz_rule_newton_schulz(cus, phase, rows, cols, count, three, ctypes.byref(rest))
    return t, rest.value
