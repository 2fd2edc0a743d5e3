"""What the operators around a product refuse, before any device is needed: the sizes of workspaces are asked for without a
handle, and an invalid description gives a negative status."""
import ctypes

import pytest

from oztt_amd import device as ozd
from oztt_amd import hip

ERR_ARG = -1


def ask(name, desc):
    return getattr(hip(), name)(None, ctypes.byref(desc))


def changed(make, **fields):
    d = make
    for k, v in fields.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("fields", [{"M": -1}, {"N": 0}, {"K": 0}, {"N": 2**22 + 1}, {"type": 2}, {"type": -1}, {"y_type": 1}, {"act": 4},
                                    {"act": -1}, {"ldx": 15}, {"ldw": -1}, {"ldy": 7}, {"ldr": 2**22 + 1}, {"ldz": 3}], ids=str)
def test_linear(fields):
    assert ask("oz_linear_workspace", changed(ozd.linear_desc(4, 8, 16), **fields)) == ERR_ARG


@pytest.mark.parametrize("fields", [{"M": -1}, {"N": 0}, {"K": 2**22 + 1}, {"type": 2}, {"dw_type": 1}, {"act": 9}, {"accumulate": 2},
                                    {"lddy": 7}, {"ldx": 15}, {"ldw": 15}, {"ldz": 7}, {"lddx": 15}, {"lddw": 15}], ids=str)
def test_linear_grad(fields):
    assert ask("oz_linear_grad_workspace", changed(ozd.linear_grad_desc(4, 8, 16), **fields)) == ERR_ARG


@pytest.mark.parametrize("fields", [{"T": -1}, {"T": 2**31}, {"vocab": 0}, {"vocab": 2**31}, {"D": 0}, {"D": 2**22 + 1}, {"type": 3},
                                    {"grad_type": 1}, {"id_bits": 16}, {"accumulate": -1}, {"ldt": 15}, {"ldo": 15}], ids=str)
def test_embedding(fields):
    assert ask("oz_embedding_grad_workspace", changed(ozd.embedding_desc(4, 8, 16), **fields)) == ERR_ARG


def test_valid_descriptions():
    assert ask("oz_linear_workspace", ozd.linear_desc(0, 1, 1)) >= 0
    assert ask("oz_linear_grad_workspace", ozd.linear_grad_desc(7, 5, 3, "f16", "gelu", "f32", True)) >= 7 * 5 * 2
    assert ask("oz_embedding_grad_workspace", ozd.embedding_desc(0, 1, 1)) == 0
    assert ask("oz_embedding_grad_workspace", ozd.embedding_desc(1000, 50, 64)) >= 4 * 4 * 1000


def test_no_device_and_no_operands():
    """Without a handle every call ends with a status."""
    d, g, e = ozd.linear_desc(4, 8, 16), ozd.linear_grad_desc(4, 8, 16), ozd.embedding_desc(4, 8, 16)
    n = [None] * 10
    assert hip().oz_linear(None, ctypes.byref(d), *n[:7], ctypes.c_size_t(0)) == ERR_ARG
    assert hip().oz_linear_grad(None, ctypes.byref(g), *n[:8], ctypes.c_size_t(0)) == ERR_ARG
    assert hip().oz_embedding(None, ctypes.byref(e), *n[:4]) == ERR_ARG
    assert hip().oz_embedding_grad(None, ctypes.byref(e), *n[:5], ctypes.c_size_t(0)) == ERR_ARG
    assert hip().oz_linear(None, None, *n[:7], ctypes.c_size_t(0)) == ERR_ARG
    assert hip().oz_adamw_step(None, None, None) == ERR_ARG


def test_adamw_plan():
    assert hip().oz_adamw_plan_bytes((ozd.AdamwTensor * 1)(ozd.adamw_tensor(100, 0, 0, 0, 0)), 1) > 0
    assert hip().oz_adamw_plan_bytes((ozd.AdamwTensor * 1)(ozd.adamw_tensor(-1, 0, 0, 0, 0)), 1) == ERR_ARG
    assert hip().oz_adamw_plan_bytes(None, 1) == ERR_ARG and hip().oz_adamw_plan_bytes(None, -1) == ERR_ARG


def test_names():
    for call in (lambda: ozd.linear_desc(1, 1, 1, "int8"), lambda: ozd.linear_desc(1, 1, 1, act="tanh"), lambda: ozd.embedding_desc(1, 1, 1, grad_type="x")):
        with pytest.raises(ValueError):
            call()
