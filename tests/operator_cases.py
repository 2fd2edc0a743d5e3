"""Helpers of the tests of the operators around a product: tensors in GPU memory as the device layer's buffers, windows
of wider matrices, and the formulas in 64 bits."""
import ctypes
import math

import numpy as np
import torch

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half the distance of neighbours, relative to the lower one (eps / 2), and at the smallest values of FP16
ROUND = {t: (torch.finfo(d).eps / 2, 2.0**-25 if t == "f16" else 0.0) for t, d in DTYPE.items()}
U32 = 2.0**-24


class Ptr:
    """A tensor (kept alive), or none, as a buffer."""

    def __init__(self, t):
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr() if t is not None else None)


def generator(seed):
    return torch.Generator(device="cuda:0").manual_seed(seed)


def window(x, pad=0, shift=0, fill=float("nan")):
    """x as a window of a matrix `pad` columns wider that begins `shift` values behind an aligned address; what lies
    around it is `fill`."""
    rows, cols = x.shape
    base = torch.full((rows * (cols + pad) + shift + 64,), fill, dtype=x.dtype, device=x.device)
    w = base[shift : shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    w.copy_(x)
    return w, base


def act(z, a):
    if a == "relu":
        return z.clamp(min=0)
    if a == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    return z * torch.sigmoid(z) if a == "silu" else z


def act_grad(z, a):
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(act(z, a).sum(), z)[0]


def within(got, want, bound, what):
    """Every value of got within `bound` of want (64 bits), with the largest excess named."""
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, d - bound, torch.zeros_like(d)).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {d.numel()} values off; at {np.unravel_index(i, d.shape)} "
                             f"{float(got.flatten()[i])} for {float(want.flatten()[i])}, bound {float(bound.flatten()[i])}")


def rounded(want, name):
    rel, floor = ROUND[name]
    return rel * want.abs() + floor
