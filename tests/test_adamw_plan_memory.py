"""The size that Device.adamw_plan gives for the memory of a plan: what the buffer has, so that a list that has outgrown it is refused
before anything is copied. On the CPU the library's calls are recorded."""
import ctypes

import pytest

from oztt_amd import device as ozd


class Memory:
    ptr = ctypes.c_void_p(4096)


@pytest.fixture
def made(monkeypatch):
    """A device handle whose plans are not made: the sizes that came with them."""
    real, sizes = ozd.hip(), []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def oz_adamw_make_plan(self, h, tensors, count, bits, memory, size, plan):
            sizes.append(size.value)
            return 0

    lib = Library()
    monkeypatch.setattr(ozd, "hip", lambda: lib)
    dev = object.__new__(ozd.Device)
    dev.h, dev.bufs = ctypes.c_void_p(), []
    return dev, sizes


def tensors(n):
    return [ozd.adamw_tensor(100, 256, 256, 256, 256) for _ in range(n)]


def test_a_buffer_has_its_own_size(made):
    dev, sizes = made
    need = dev.adamw_plan_bytes(tensors(3))
    short, long = Memory(), Memory()
    short.nbytes, long.nbytes = dev.adamw_plan_bytes(tensors(2)), need + 512
    assert short.nbytes < need
    dev.adamw_plan(tensors(3), 32, short)
    dev.adamw_plan(tensors(3), 32, long)
    assert sizes == [short.nbytes, long.nbytes]


def test_memory_of_a_stated_size(made):
    """An address alone (another library's tensor) has the size that the caller states; without one it is taken to have room."""
    dev, sizes = made
    dev.adamw_plan(tensors(3), 8, Memory(), 64)
    dev.adamw_plan(tensors(3), 8, Memory())
    assert sizes == [64, dev.adamw_plan_bytes(tensors(3))]


def test_the_library_refuses_what_is_short():
    """No handle and no copy: the size is looked at first."""
    arr = (ozd.AdamwTensor * 3)(*tensors(3))
    need = ozd.hip().oz_adamw_plan_bytes(arr, 3)
    plan = ozd.AdamwPlan()
    for size in (0, need - 1):
        st = ozd.hip().oz_adamw_make_plan(None, arr, 3, 32, ctypes.c_void_p(4096), ctypes.c_size_t(size), ctypes.byref(plan))
        assert st == -1 and not plan.memory


@pytest.mark.gpu
def test_a_short_buffer_is_refused(dev):
    buf = dev.alloc(dev.adamw_plan_bytes(tensors(2)))
    with pytest.raises(RuntimeError, match="needed"):
        dev.adamw_plan(tensors(3), 32, buf)
    assert dev.adamw_plan(tensors(2), 32, buf).count == 2
