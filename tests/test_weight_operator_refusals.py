"""What the operators on weights (8-bit integers, orthogonalized updates) refuse, before any device is needed."""
import ctypes

import pytest

from oztt_amd import device as ozd
from oztt_amd import hip

ERR_ARG = -1
NONE = [None] * 10
SIZE = ctypes.c_size_t(0)


def changed(d, **fields):
    for k, v in fields.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("fields", [{"M": -1}, {"M": 2**31}, {"K": 0}, {"K": 2**22 + 1}, {"type": 3}, {"type": -1}, {"ldx": 15}, {"ldq": -1},
                                    {"ldq": 2**32 + 1}], ids=str)
def test_quantize(fields):
    assert hip().oz_quantize_rows(None, ctypes.byref(changed(ozd.quantize_desc(4, 16), **fields)), *NONE[:3]) == ERR_ARG


@pytest.mark.parametrize("fields", [{"M": -1}, {"N": 0}, {"K": 0}, {"N": 2**22 + 1}, {"K": 131072, "ldw": 131072}, {"type": 2}, {"y_type": 1}, {"act": 4},
                                    {"x_int8": 2}, {"ldx": 15}, {"ldw": 12}, {"ldw": 18}, {"ldy": 7}, {"ldr": 2**22 + 1}, {"x_int8": 1, "ldx": 17}], ids=str)
def test_linear_i8(fields):
    assert hip().oz_linear_i8_workspace(None, ctypes.byref(changed(ozd.linear_i8_desc(4, 8, 16), **fields))) == ERR_ARG


def test_linear_i8_rows_at_odd_places():
    """A row of 15 bytes is no multiple of 4, unless a leading dimension makes it one."""
    ask = lambda d: hip().oz_linear_i8_workspace(None, ctypes.byref(d))  # noqa: E731
    assert ask(ozd.linear_i8_desc(4, 8, 15)) == ERR_ARG
    assert ask(ozd.linear_i8_desc(4, 8, 15, ldw=16)) > 0
    assert ask(ozd.linear_i8_desc(4, 8, 15, x_int8=True, ldw=16)) == ERR_ARG
    assert ask(ozd.linear_i8_desc(4, 8, 15, x_int8=True, ldw=16, ldx=16)) >= 0
    assert ask(ozd.linear_i8_desc(0, 1, 4)) >= 0
    assert ask(ozd.linear_i8_desc(5, 3, 131071, ldw=131072)) >= 5 * 131072


@pytest.mark.parametrize("fields", [{"rows": 0}, {"cols": 0}, {"rows": 2**20 + 1}, {"rows": 2**20, "cols": 2**20}, {"count": -1}, {"type": 3}, {"steps": 0},
                                    {"steps": 101}, {"a": float("nan")}, {"b": float("inf")}, {"c": 1e39}, {"eps": -1.0}, {"eps": float("inf")}, {"ldg": 15},
                                    {"ldo": -1}, {"stride_g": 63}, {"stride_o": 63}], ids=str)
def test_orthogonalize(fields):
    assert hip().oz_orthogonalize_workspace(None, ctypes.byref(changed(ozd.orthogonalize_desc(4, 16, 2), **fields))) == ERR_ARG


def test_orthogonalize_sizes():
    ask = lambda d: hip().oz_orthogonalize_workspace(None, ctypes.byref(d))  # noqa: E731
    assert ask(ozd.orthogonalize_desc(4, 16, 0)) == 0
    assert ask(ozd.orthogonalize_desc(600, 700, 2)) >= 2 * 6 * 600 * 700
    assert ask(changed(ozd.orthogonalize_desc(4, 16, 1), stride_g=1)) > 0  # one matrix has no distance


def tensor(**fields):
    return changed(ozd.muon_tensor(4, 8, 256, 256, 256), **fields)


def make(tensors, memory=256, nbytes=1 << 20):
    plan = ozd.MuonPlan()
    arr = (ozd.MuonTensor * max(len(tensors), 1))(*tensors)
    return hip().oz_muon_make_plan(None, arr, len(tensors), ctypes.c_void_p(memory), ctypes.c_size_t(nbytes), ctypes.byref(plan))


@pytest.mark.parametrize("fields", [{"rows": -1}, {"cols": 2**20 + 1}, {"param_type": 3}, {"grad_type": -1}, {"master": 256}, {"param": None}, {"grad": None},
                                    {"m": None}, {"m": 258}, {"param": 255}, {"weight_decay": -1.0}, {"weight_decay": float("nan")}, {"lr_scale": -1.0},
                                    {"lr_scale": float("inf")}], ids=str)
def test_muon_plan(fields):
    assert make([tensor(), tensor(**fields)]) == ERR_ARG


def test_muon_plan_memory_and_sizes():
    assert make([tensor()], memory=None) == ERR_ARG
    assert make([tensor()], memory=264) == ERR_ARG
    assert make([tensor()], nbytes=16) == ERR_ARG
    assert make([tensor(rows=4 + k) for k in range(ozd.MUON_SHAPES + 1)]) == ERR_ARG
    assert hip().oz_muon_plan_bytes(None, -1) == ERR_ARG and hip().oz_muon_plan_bytes(None, 1) == ERR_ARG
    assert hip().oz_muon_make_plan(None, None, 0, None, SIZE, None) == ERR_ARG


def plan(**fields):
    p = ozd.MuonPlan()
    p.memory, p.count, p.shapes = 256, 3, 1
    p.shape[0] = ozd.MuonShape(4, 8, 3, 0)
    return changed(p, **fields)


@pytest.mark.parametrize("fields", [{"memory": None}, {"shapes": 17}, {"shapes": -1}, {"count": 2}, {"shapes": 2}], ids=str)
def test_muon_bad_plans(fields):
    assert hip().oz_muon_workspace(None, ctypes.byref(plan(**fields))) == ERR_ARG


@pytest.mark.parametrize("o", [(-1.0, 0.9, 1, 5), (float("nan"), 0.9, 1, 5), (0.1, 1.0, 1, 5), (0.1, -0.1, 1, 5), (0.1, 0.9, 2, 5), (0.1, 0.9, 1, 0)], ids=str)
def test_muon_options(o):
    opt = ozd.MuonOptions(*o, *ozd.NEWTON_SCHULZ, 1e-7, None)
    n = hip().oz_muon_workspace(None, ctypes.byref(plan()))
    assert n > 0
    assert hip().oz_muon_step(None, ctypes.byref(plan()), ctypes.byref(opt), ctypes.c_void_p(256), ctypes.c_size_t(n)) == ERR_ARG


def test_muon_workspace_is_checked():
    opt = ozd.MuonOptions(0.1, 0.9, 1, 5, *ozd.NEWTON_SCHULZ, 1e-7, None)
    n = hip().oz_muon_workspace(None, ctypes.byref(plan()))
    for at, size in ((None, n), (256, n - 1), (264, n)):
        assert hip().oz_muon_step(None, ctypes.byref(plan()), ctypes.byref(opt), ctypes.c_void_p(at), ctypes.c_size_t(size)) == ERR_ARG


def test_no_device_and_no_operands():
    q, l, o = ozd.quantize_desc(4, 16), ozd.linear_i8_desc(4, 8, 16), ozd.orthogonalize_desc(4, 8)
    assert hip().oz_quantize_rows(None, ctypes.byref(q), *NONE[:3]) == ERR_ARG
    assert hip().oz_quantize_rows(None, None, *NONE[:3]) == ERR_ARG
    assert hip().oz_linear_i8(None, ctypes.byref(l), *NONE[:8], SIZE) == ERR_ARG
    assert hip().oz_linear_i8(None, None, *NONE[:8], SIZE) == ERR_ARG
    assert hip().oz_orthogonalize(None, ctypes.byref(o), *NONE[:3], SIZE) == ERR_ARG
    assert hip().oz_muon_step(None, None, None, None, SIZE) == ERR_ARG


def test_names():
    for call in (lambda: ozd.quantize_desc(1, 1, "int8"), lambda: ozd.linear_i8_desc(1, 1, 1, act="tanh"), lambda: ozd.orthogonalize_desc(1, 1, type="x"),
                 lambda: ozd.muon_tensor(1, 1, 0, 0, 0, param_type="x")):
        with pytest.raises(ValueError):
            call()
