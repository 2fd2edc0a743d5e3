"""The random bits of AdamW's 8-bit states from step to step. The hash of place xor seed gives an aligned group of 2^k places the
same set of numbers for all seeds below 2^k, each time dealt out anew: the group's mean rounding stays where it is. The seeds
of adamw_seed are spread over 32 bits, so that steps draw different sets. CPU only."""
import ctypes

import numpy as np
import pytest

from oztt_amd import device as ozd

N = 4096


def mix(x):
    """The header's hash, in whole numbers."""
    x = x.astype(np.uint64)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def drawn(seed):
    """The 16 bits of m and of v of an aligned group."""
    h = mix(np.arange(N, dtype=np.uint64) ^ np.uint64(seed))
    return h & np.uint64(0xFFFF), h >> np.uint64(16)


def test_seed_is_the_hash_of_the_step():
    for step in (1, 2, 3, 1000, 2**32 + 5, 2**40):
        want = int(mix(np.array([step & 0xFFFFFFFF], dtype=np.uint64) ^ mix(np.array([step >> 32], dtype=np.uint64)))[0])
        assert ozd.adamw_seed(step) == want
    assert len({ozd.adamw_seed(k) for k in range(1, 5001)}) == 5000


def test_steps_draw_different_sets():
    """The means of 200 steps are spread as means of N independent numbers are: by 2^16 / sqrt(12 N), within a third (the spread of 200
    values is known to 5%), and about the middle."""
    for k in (0, 1):
        means = np.array([drawn(ozd.adamw_seed(s))[k].mean() for s in range(1, 201)])
        assert len(set(means)) > 190
        spread = 2**16 / np.sqrt(12 * N)
        assert 2 / 3 * spread < means.std() < 4 / 3 * spread and abs(means.mean() - (2**15 - 0.5)) < 4 * spread / np.sqrt(200)
    # and why the step itself is no seed
    assert len({float(drawn(s)[0].mean()) for s in range(1, 201)}) == 1


@pytest.mark.parametrize("given", [None, 0, 5])
def test_a_step_without_a_seed_has_its_own(monkeypatch, given):
    real, seen = ozd.hip(), []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def oz_adamw_step(self, h, plan, options):
            seen.append(ctypes.cast(options, ctypes.POINTER(ozd.AdamwOptions)).contents.seed)
            return 0

    lib = Library()
    monkeypatch.setattr(ozd, "hip", lambda: lib)
    dev = object.__new__(ozd.Device)
    dev.h, dev.bufs = ctypes.c_void_p(), []
    for step in (1, 2, 7):
        dev.adamw_step(ozd.AdamwPlan(), 1e-3, step=step, **({} if given is None else {"seed": given}))
    assert seen == ([ozd.adamw_seed(s) for s in (1, 2, 7)] if given is None else [given] * 3)
