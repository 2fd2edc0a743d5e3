"""A small next-token network, trained on the device layer's operators from the lookup to the optimizer's step, and
then asked token by token.

    x = embedding(t);  h = gelu(x W1^T + b1);  y = h W2^T + b2 + x;  logits = y W3^T

Weights, activations and gradients stay in GPU memory in BF16, the optimizer keeps FP32 copies of the weights and its states
in 8 bits. Only the logits come to the host, for the loss. Run from the repository's root: python examples/train_tokens.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from oztt_amd import device as ozd  # noqa: E402

VOCAB, WIDTH, HIDDEN, TOKENS = 96, 128, 512, 1024


def to_bf16(x: np.ndarray) -> np.ndarray:
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


class Weight:
    """A weight in BF16, its FP32 copy, its gradient in FP32 and its states in 8 bits."""

    def __init__(self, dev, x: np.ndarray, decay: float):
        n, blocks = x.size, -(-x.size // ozd.ADAMW_BLOCK)
        self.param, self.master = dev.upload(to_bf16(x)), dev.upload(x.astype(np.float32))
        self.grad = dev.upload(np.zeros(n, np.float32))
        self.m, self.v = dev.upload(np.zeros(n, np.uint8)), dev.upload(np.zeros(n, np.uint8))
        self.m_scale, self.v_scale = dev.upload(np.zeros(blocks, np.uint8)), dev.upload(np.zeros(blocks, np.uint8))
        a = lambda b: b.ptr.value  # noqa: E731
        self.tensor = ozd.adamw_tensor(n, a(self.param), a(self.grad), a(self.m), a(self.v), a(self.master), a(self.m_scale),
                                       a(self.v_scale), "bf16", "f32", decay)


class Network:
    def __init__(self, dev, seed: int = 0):
        rng = np.random.default_rng(seed)
        normal = lambda *shape: (rng.standard_normal(shape) * shape[-1] ** -0.5).astype(np.float32)  # noqa: E731
        self.dev = dev
        self.w = {"E": Weight(dev, rng.standard_normal((VOCAB, WIDTH)), 0.0), "W1": Weight(dev, normal(HIDDEN, WIDTH), 0.01),
                  "b1": Weight(dev, np.zeros(HIDDEN), 0.0), "W2": Weight(dev, normal(WIDTH, HIDDEN), 0.01),
                  "b2": Weight(dev, np.zeros(WIDTH), 0.0), "W3": Weight(dev, normal(VOCAB, WIDTH), 0.01)}
        self.plan = dev.adamw_plan([w.tensor for w in self.w.values()], 8)
        self.buffers = {}

    def room(self, name: str, nbytes: int):
        if name not in self.buffers or self.buffers[name].nbytes < nbytes:
            self.buffers[name] = self.dev.alloc(nbytes)
        return self.buffers[name]

    def linear(self, x, name, bias, out, T, N, K, act="none", y_type=None, residual=None, Z=None):
        d = ozd.linear_desc(T, N, K, "bf16", act, y_type)
        n = self.dev.linear_workspace(d)
        y = self.room(out, T * N * (4 if y_type == "f32" else 2))
        self.dev.linear(d, x, self.w[name].param, y, bias=self.w[bias].param if bias else None, residual=residual, Z=Z,
                        work=self.room("work", n) if n else None, work_bytes=n)
        return y

    def logits(self, ids: np.ndarray) -> np.ndarray:
        """FP32 logits of each token's successor; the activations stay for gradients()."""
        T = len(ids)
        self.ids = self.dev.upload(ids.astype(np.int32))
        x = self.room("x", T * WIDTH * 2)
        self.dev.embedding(ozd.embedding_desc(T, VOCAB, WIDTH, "bf16", 32), self.w["E"].param, self.ids, x)
        h = self.linear(x, "W1", "b1", "h", T, HIDDEN, WIDTH, "gelu", Z=self.room("z", T * HIDDEN * 2))
        y = self.linear(h, "W2", "b2", "y", T, WIDTH, HIDDEN, residual=x)
        out = self.linear(y, "W3", None, "logits", T, VOCAB, WIDTH, y_type="f32")
        got = self.dev.download(out, np.float32, T * VOCAB).reshape(T, VOCAB)
        self.ids.free()
        return got

    def linear_grad(self, dy, x, name, bias, T, N, K, act="none", Z=None, out=None):
        d = ozd.linear_grad_desc(T, N, K, "bf16", act, "f32")
        n = self.dev.linear_grad_workspace(d)
        dx = self.room(out, T * K * 2)
        self.dev.linear_grad(d, dy, x, self.w[name].param, Z, dX=dx, dW=self.w[name].grad, dbias=self.w[bias].grad if bias else None,
                             work=self.room("work", n), work_bytes=n)
        return dx

    def gradients(self, ids: np.ndarray, dlogits: np.ndarray):
        T, b = len(ids), self.buffers
        dl, tokens = self.dev.upload(to_bf16(dlogits)), self.dev.upload(ids.astype(np.int32))
        dy = self.linear_grad(dl, b["y"], "W3", None, T, VOCAB, WIDTH, out="dy")
        dh = self.linear_grad(dy, b["h"], "W2", "b2", T, WIDTH, HIDDEN, out="dh")
        dx = self.linear_grad(dh, b["x"], "W1", "b1", T, HIDDEN, WIDTH, "gelu", b["z"], out="dx")
        # x goes two ways, through the layers and past them: its rows' gradients are added one after the other
        for k, d in enumerate((dx, dy)):
            e = ozd.embedding_desc(T, VOCAB, WIDTH, "bf16", 32, grad_type="f32", accumulate=bool(k))
            n = self.dev.embedding_grad_workspace(e)
            self.dev.embedding_grad(e, d, tokens, self.w["E"].grad, None, self.room("work", n), n)
        self.dev.sync()
        dl.free()
        tokens.free()

    def step(self, ids: np.ndarray, targets: np.ndarray, number: int, lr: float) -> float:
        z = self.logits(ids).astype(np.float64)
        z -= z.max(1, keepdims=True)
        p = np.exp(z)
        p /= p.sum(1, keepdims=True)
        rows = np.arange(len(ids))
        loss = float(-np.log(p[rows, targets]).mean())
        p[rows, targets] -= 1
        self.gradients(ids, p / len(ids))
        self.dev.adamw_step(self.plan, lr, 0.9, 0.95, 1e-8, number)
        return loss


def successor(t: np.ndarray) -> np.ndarray:
    """The language: every word has one successor."""
    return (t * 37 + 11) % VOCAB


def main(steps: int = 60) -> tuple[list[float], float]:
    """Losses of the steps, and the share of words whose successor the trained network names, asked one by one."""
    rng = np.random.default_rng(1)
    with ozd.Device(0) as dev:
        net = Network(dev)
        losses = []
        for k in range(1, steps + 1):
            ids = rng.integers(0, VOCAB, TOKENS)
            losses.append(net.step(ids, successor(ids), k, 1e-3))
            if k == 1 or k % 10 == 0:
                print(f"step {k}: loss {losses[-1]:.4f}", flush=True)
        words = np.arange(VOCAB)
        right = np.mean([int(net.logits(np.array([t])).argmax()) == successor(t) for t in words])
    print(f"successors named right: {right:.3f}", flush=True)
    return losses, float(right)


if __name__ == "__main__":
    main()
