"""A layer's life: trained by Muon from its gradients, its weights quantized by channel, then answering batches and single tokens in 8-bit
integers. Each stage is held to its formula in 64 bits on what the stage before has left."""
import numpy as np
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import Ptr, generator, rounded, within
from tests.test_gpu_orthogonalize import exact, rounding_of_x

pytestmark = pytest.mark.gpu

TOKENS, IN, OUT = 300, 200, 136
LR, MOMENTUM = 0.02, 0.9


def test_trained_quantized_and_asked(dev):
    g = generator(11)
    X = torch.randn((TOKENS, IN), device="cuda:0", generator=g).bfloat16()
    T = torch.randn((TOKENS, OUT), device="cuda:0", generator=g).bfloat16()
    W = (torch.randn((OUT, IN), device="cuda:0", generator=g) * IN**-0.5)
    P = W.bfloat16()
    dW, m = torch.zeros((OUT, IN), device="cuda:0"), torch.zeros((OUT, IN), device="cuda:0")
    Y = torch.zeros((TOKENS, OUT), dtype=torch.bfloat16, device="cuda:0")
    a = lambda t: t.data_ptr()  # noqa: E731
    plan = dev.muon_plan([ozd.muon_tensor(OUT, IN, a(P), a(dW), a(m), a(W), "bf16", "f32", 0.01)])
    d, e = ozd.linear_desc(TOKENS, OUT, IN), ozd.linear_grad_desc(TOKENS, OUT, IN, "bf16", "none", "f32")
    sizes = [dev.linear_workspace(d), dev.linear_grad_workspace(e), dev.muon_workspace(plan)]
    work = torch.zeros(max(sizes), dtype=torch.uint8, device="cuda:0")
    for k in range(5):
        torch.cuda.synchronize()
        dev.linear(d, Ptr(X), Ptr(P), Ptr(Y), work=Ptr(work), work_bytes=sizes[0])
        dev.sync()
        dY = (Y.float() - T.float()).bfloat16()
        w0, m0 = W.clone(), m.clone()
        torch.cuda.synchronize()
        dev.linear_grad(e, Ptr(dY), Ptr(X), Ptr(P), dW=Ptr(dW), work=Ptr(work), work_bytes=sizes[1])
        dev.muon_step(plan, LR, MOMENTUM, work=Ptr(work), work_bytes=sizes[2])
        dev.sync()
        size = dY.double().abs().T @ X.double().abs()
        within(dW, dY.double().T @ X.double(), (TOKENS + 2) * 2.0**-24 * size, "dW")
        f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda:0")  # noqa: E731
        assert torch.equal(m, f(MOMENTUM) * m0 + f(1 - MOMENTUM) * dW)
        o = exact((f(MOMENTUM) * m + f(1 - MOMENTUM) * dW)[None])[0]
        rate = LR * 0.2 * max(OUT, IN) ** 0.5
        off = 20 * (1e-5 + rounding_of_x() / float(o.norm())) * float(o.square().mean().sqrt()) * rate + 4 * 2.0**-24 * (w0.double().abs() + rate * o.abs())
        within(W, w0.double() * (1 - LR * 0.01) - rate * o, off, "W")
        assert torch.equal(P, W.bfloat16())
    Wq, ws = torch.zeros((OUT, IN), dtype=torch.int8, device="cuda:0"), torch.zeros(OUT, device="cuda:0")
    torch.cuda.synchronize()
    dev.quantize_rows(ozd.quantize_desc(OUT, IN, "f32"), Ptr(W), Ptr(Wq), Ptr(ws))
    dev.sync()
    dw = (Wq.double() * ws.double()[:, None] - W.double()).abs()
    assert bool((dw <= ws.double()[:, None] * 0.5 * (1 + 1e-4)).all())
    for first, tokens in ((0, TOKENS), (7, 1), (100, 2), (3, 11)):
        x = X[first : first + tokens]
        y = torch.zeros((tokens, OUT), dtype=torch.bfloat16, device="cuda:0")
        q = ozd.linear_i8_desc(tokens, OUT, IN)
        n = dev.linear_i8_workspace(q)
        w = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda:0")
        torch.cuda.synchronize()
        dev.linear_i8(q, Ptr(x), Ptr(Wq), Ptr(ws), Ptr(y), work=Ptr(w), work_bytes=n)
        dev.sync()
        want = x.double() @ W.double().T
        # each x is off by half a step of its token's scale, each w by half a step of its channel's
        step = x.double().abs().amax(1, keepdim=True) / 127 * 0.5 * (1 + 1e-4)
        half = ws.double() * 0.5 * (1 + 1e-4)
        off = step * W.double().abs().sum(1) + x.double().abs().sum(1, keepdim=True) * half + IN * step * half
        within(y, want, off + rounded(want.abs() + off, "bf16"), f"{tokens} tokens")
    assert np.isfinite(y.float().cpu().numpy()).all()
