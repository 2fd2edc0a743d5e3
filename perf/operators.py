"""The operators around the matrix product that a program needs to train a network and to answer with it:

  "linear"       Y = act(X W^T + bias) + residual, the product with its epilogue
  "linear_grad"  its gradients: dX, dW and dbias from dY and the kept values Z in front of the activation
  "embedding"    rows of a table by token, scaled
  "embedding_grad"  the table's gradient: the rows of dY summed by token
  "adamw"        one AdamW step over many tensors, the two states of each value in 32 bits or in 8

In the plain form an operator is the formula in elementary operations, in 32 bits. Otherwise it is the call
that a program makes of the device layer (oztt_amd.device) on tensors that it keeps in GPU memory.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one token through a square layer of an answering program: the weights are read once, nothing else counts
        {"name": "linear_token", "kind": "linear", "M": 1, "N": 8192, "K": 8192, "type": "bf16", "act": "none", "y": "bf16", "bias": False, "residual": True, "keep": False, "pad": 0},
        # a batch of answers being written, one token each, through a widening layer; FP16
        {"name": "linear_batch", "kind": "linear", "M": 24, "N": 8192, "K": 2048, "type": "f16", "act": "silu", "y": "f16", "bias": True, "residual": False, "keep": False, "pad": 0},
        # sizes that fit no tile and operands that are windows of wider matrices, the activation's input kept for training
        {"name": "linear_ragged", "kind": "linear", "M": 1000, "N": 700, "K": 1500, "type": "bf16", "act": "gelu", "y": "bf16", "bias": True, "residual": True, "keep": True, "pad": 12},
        # a long batch through a square layer, everything in the epilogue: the largest product
        {"name": "linear_8192", "kind": "linear", "M": 8192, "N": 8192, "K": 8192, "type": "bf16", "act": "gelu", "y": "bf16", "bias": True, "residual": True, "keep": True, "pad": 0},
        # gradients of a small layer whose sizes fit no tile
        {"name": "linear_grad_ragged", "kind": "linear_grad", "M": 1000, "N": 700, "K": 1500, "type": "f16", "act": "silu", "dw": "f16", "pad": 0},
        # gradients of a widening layer over a training batch of 8192 tokens
        {"name": "linear_grad_8192", "kind": "linear_grad", "M": 8192, "N": 8192, "K": 2048, "type": "bf16", "act": "gelu", "dw": "bf16", "pad": 0},
        # the tokens of a training batch looked up in a large table
        {"name": "embedding_8192", "kind": "embedding", "T": 8192, "vocab": 65536, "D": 4096, "type": "bf16", "ids": 64},
        # the gradient of a small table from a short text, a few words of it very frequent
        {"name": "embedding_grad_512", "kind": "embedding_grad", "T": 512, "vocab": 5000, "D": 500, "type": "bf16", "dw": "f32", "ids": 64},
        # the gradient of a large table from a training batch: most rows are zero, some are sums of a thousand
        {"name": "embedding_grad_32768", "kind": "embedding_grad", "T": 32768, "vocab": 65536, "D": 2048, "type": "bf16", "dw": "f32", "ids": 32},
        # a small network's tensors, from single biases to matrices: nothing but latency
        {"name": "adamw_small", "kind": "adamw", "count": 24, "total": 200000, "param": "f32", "master": False, "grad": "f32", "bits": 32},
        # the matrices and biases of some large layers, BF16 with 32-bit copies, states in 32 bits
        {"name": "adamw_32bit", "kind": "adamw", "count": 60, "total": 100000000, "param": "bf16", "master": True, "grad": "bf16", "bits": 32},
        # the same with states in 8 bits
        {"name": "adamw_8bit", "kind": "adamw", "count": 60, "total": 100000000, "param": "bf16", "master": True, "grad": "bf16", "bits": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "linear_grad", "linear_grad", "embedding", "embedding_grad", "adamw", "adamw"])
    c = {"kind": kind}
    if kind in ("linear", "linear_grad"):
        while True:
            M, N, K = _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 16, 8192)
            if M * N * K <= 2.0**36:
                break
        if rng.random() < 0.5:  # widths as networks have them
            N, K = -(-N // 64) * 64, -(-K // 64) * 64
        c.update(M=M, N=N, K=K, type=rng.choice(["bf16", "bf16", "f16"]), act=rng.choice(["none", "relu", "gelu", "silu"]), pad=rng.choice([0, 0, 0, 8, 5]))
        if kind == "linear":
            c.update(y=rng.choice([c["type"], c["type"], "f32"]), bias=rng.random() < 0.7, residual=rng.random() < 0.5, keep=rng.random() < 0.5)
        else:
            # With an activation the products take dZ rounded to the operands' type, so a 32-bit dW holds no more
            # than that; without one dZ is dY itself.
            c.update(dw=rng.choice([c["type"], "f32"]) if c["act"] == "none" else c["type"])
    elif kind in ("embedding", "embedding_grad"):
        while True:
            T, vocab, D = _log(rng, 1, 32768), _log(rng, 50, 131072), _log(rng, 16, 8192)
            if T * D <= 2**26 and vocab * D <= 2**28:
                break
        c.update(T=T, vocab=vocab, D=-(-D // 64) * 64 if rng.random() < 0.6 else D, type=rng.choice(["bf16", "f16"]), ids=rng.choice([32, 64]))
        if kind == "embedding_grad":
            c["dw"] = rng.choice([c["type"], "f32"])
    else:
        count = _log(rng, 1, 300)
        param = rng.choice(["f32", "bf16", "f16"])
        c.update(count=count, total=max(count, _log(rng, 1000, 100000000)), param=param, master=param != "f32" and rng.random() < 0.7, grad=rng.choice([param, "f32"]), bits=rng.choice([8, 32]))
    return c


# ---- inputs -----------------------------------------------------------------------------------------

SCALE = 0.125  # of the embedding
LR, BETA1, BETA2, EPS, STEP = 1e-3, 0.9, 0.95, 1e-8, 7
BLOCK = 64     # values of a state in 8 bits that share a scale


def _generator(seed):
    return torch.Generator(device="cuda:0").manual_seed((int(seed) * 2654435761 + 12345) % (1 << 62))


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda:0", generator=g) * scale).to(dtype)


def _window(x, pad):
    """x as a window of a matrix `pad` columns wider, whose other columns hold what nobody may use."""
    if not pad:
        return x
    w = torch.full((x.shape[0], x.shape[1] + pad), float("nan"), dtype=x.dtype, device=x.device)
    w[:, : x.shape[1]] = x
    return w[:, : x.shape[1]]


def _rows(rows, cols, dtype, pad):
    """An output of the same kind."""
    return torch.zeros((rows, cols + pad), dtype=dtype, device="cuda:0")[:, :cols]


def _linear_inputs(case, seed):
    M, N, K, t, pad = case["M"], case["N"], case["K"], DTYPES[case["type"]], case["pad"]
    g = _generator(seed)
    # activations whose channels differ in size, weights that keep the variance
    size = torch.exp(0.5 * torch.randn(K, device="cuda:0", generator=g))
    s = {"X": _window((torch.randn((M, K), device="cuda:0", generator=g) * size).to(t), pad), "W": _window(_normal(g, (N, K), t, K**-0.5), pad)}
    if case["kind"] == "linear":
        s["bias"] = _normal(g, (N,), t, 0.2) if case["bias"] else None
        s["residual"] = _window(_normal(g, (M, N), DTYPES[case["y"]]), pad) if case["residual"] else None
    else:
        s["dY"] = _window(_normal(g, (M, N), t, 0.05), pad)
        s["Z"] = _window(_normal(g, (M, N), t, 1.5), pad) if case["act"] != "none" else None
    return s


def _ids(case, g):
    """Tokens by Zipf's law, the frequent ones anywhere in the vocabulary."""
    V = case["vocab"]
    u = torch.rand(case["T"], dtype=torch.float64, device="cuda:0", generator=g)
    rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp(0, V - 1)
    return torch.randperm(V, device="cuda:0", generator=g)[rank].to(torch.int32 if case["ids"] == 32 else torch.int64)


def _embedding_inputs(case, seed):
    g = _generator(seed)
    t = DTYPES[case["type"]]
    s = {"ids": _ids(case, g)}
    if case["kind"] == "embedding":
        s["table"] = _normal(g, (case["vocab"], case["D"]), t)
    else:
        s["dY"] = _normal(g, (case["T"], case["D"]), t, 0.05)
    return s


def _sizes(case):
    """Sizes of `count` tensors, `total` values together: every third a bias, the others matrices of growing size."""
    weight = [1e-3 if i % 3 == 2 else 1.0 + i for i in range(case["count"])]
    return [max(1, int(case["total"] * w / sum(weight))) for w in weight]


def _adamw_inputs(case, seed):
    """The tensors are parts of one buffer a kind, each at a multiple of BLOCK values; zeros between them."""
    g = _generator(seed)
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    first = np.concatenate([[0], np.cumsum(blocks)])
    nb = int(first[-1])
    left = torch.full((nb,), BLOCK, dtype=torch.int64, device="cuda:0")
    left[torch.from_numpy(first[1:] - 1).cuda()] = torch.tensor([n - BLOCK * (b - 1) for n, b in zip(sizes, blocks)], device="cuda:0")
    valid = torch.arange(BLOCK, device="cuda:0") < left[:, None]
    # sizes that differ from block to block; a tenth of the blocks have never had a gradient (rows of tokens not seen)
    size = torch.exp(torch.randn((nb, 1), device="cuda:0", generator=g)) * 1e-3 * (torch.rand((nb, 1), device="cuda:0", generator=g) > 0.1)
    normal = lambda: torch.randn((nb, BLOCK), device="cuda:0", generator=g)  # noqa: E731
    s = {"sizes": sizes, "first": first}
    p = normal() * 0.02 * valid
    s["param"] = p.to(DTYPES[case["param"]])
    s["master"] = p if case["master"] else None
    s["grad"] = (normal() * size * valid).to(DTYPES[case["grad"]])
    m, r = normal() * size * 0.3 * valid, (torch.abs(normal()) * 0.5 + 0.5) * size * valid
    # biases (every third tensor) have no weight decay
    decay = torch.tensor([0.0 if i % 3 == 2 else 0.1 for i in range(len(sizes))], device="cuda:0")
    s["decay"] = decay.repeat_interleave(torch.tensor(blocks, device="cuda:0"))
    s["seed"] = int(seed) * 40503 % (1 << 32)
    if case["bits"] == 32:
        s["m"], s["v"] = m, r * r
    else:
        half = torch.full((nb, BLOCK), 0.5, device="cuda:0")
        s["m"], s["m_scale"] = _to_8bit(m, half, False)
        s["v"], s["v_scale"] = _to_8bit(r, half, True)
    return s


_DEV = None


def _device():
    """The program's device handle: one stream, as one thread of a program has."""
    global _DEV
    if _DEV is None:
        from oztt_amd import device as ozd

        _DEV = ozd.Device(0)
    return _DEV


class _Ptr:
    """A tensor, or none, as the device layer's buffer."""

    def __init__(self, t):
        self.t, self.ptr = t, ctypes.c_void_p(t.data_ptr() if t is not None else None)


def _bytes(n):
    return _Ptr(torch.empty(max(int(n), 256), dtype=torch.uint8, device="cuda:0"))


def prepare(case, seed):
    kind, pad = case["kind"], case.get("pad", 0)
    s = {"case": case}
    if kind in ("linear", "linear_grad"):
        s.update(_linear_inputs(case, seed))
        M, N, K, t = case["M"], case["N"], case["K"], DTYPES[case["type"]]
        if kind == "linear":
            s["Y"] = _rows(M, N, DTYPES[case["y"]], pad)
            s["keepZ"] = _rows(M, N, t, pad) if case["keep"] else None
        else:
            s["dX"], s["dW"] = _rows(M, K, t, pad), _rows(N, K, DTYPES[case["dw"]], pad)
            s["dbias"] = torch.zeros(N, dtype=DTYPES[case["dw"]], device="cuda:0")
    elif kind in ("embedding", "embedding_grad"):
        s.update(_embedding_inputs(case, seed))
        rows, dtype = (case["T"], DTYPES[case["type"]]) if kind == "embedding" else (case["vocab"], DTYPES[case["dw"]])
        s["out"] = torch.zeros((rows, case["D"]), dtype=dtype, device="cuda:0")
        s["flags"] = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    else:
        s.update(_adamw_inputs(case, seed))
    if own:
        _prepare_call(s)
    return s


def _prepare_call(s):
    """What a program keeps beside its tensors: descriptors, workspaces and the optimizer's plan."""
    from oztt_amd import device as ozd

    case, dev = s["case"], _device()
    kind = case["kind"]
    s["ptr"] = {k: _Ptr(x) for k, x in s.items() if isinstance(x, torch.Tensor) or x is None}
    if kind == "linear":
        N = case["N"] + case["pad"]
        K = case["K"] + case["pad"]
        s["desc"] = ozd.linear_desc(case["M"], case["N"], case["K"], case["type"], case["act"], case["y"], ldx=K, ldw=K, ldy=N, ldr=N, ldz=N)
        s["work_bytes"] = dev.linear_workspace(s["desc"])
    elif kind == "linear_grad":
        N = case["N"] + case["pad"]
        K = case["K"] + case["pad"]
        s["desc"] = ozd.linear_grad_desc(case["M"], case["N"], case["K"], case["type"], case["act"], case["dw"], lddy=N, ldx=K, ldw=K, ldz=N, lddx=K, lddw=K)
        s["work_bytes"] = dev.linear_grad_workspace(s["desc"])
    elif kind in ("embedding", "embedding_grad"):
        s["desc"] = ozd.embedding_desc(case["T"], case["vocab"], case["D"], case["type"], id_bits=case["ids"], scale=SCALE, grad_type=case.get("dw"))
        s["work_bytes"] = dev.embedding_grad_workspace(s["desc"]) if kind == "embedding_grad" else 0
    else:
        part = lambda k, i: s[k].data_ptr() + int(s["first"][i]) * BLOCK * s[k].element_size()  # noqa: E731
        scale = lambda k, i: s[k].data_ptr() + int(s["first"][i])  # noqa: E731
        tensors = []
        for i, n in enumerate(s["sizes"]):
            tensors.append(ozd.adamw_tensor(
                n, part("param", i), part("grad", i), part("m", i), part("v", i), master=part("master", i) if case["master"] else 0,
                m_scale=scale("m_scale", i) if case["bits"] == 8 else 0, v_scale=scale("v_scale", i) if case["bits"] == 8 else 0,
                param_type=case["param"], grad_type=case["grad"], weight_decay=0.0 if i % 3 == 2 else 0.1))
        s["plan"] = dev.adamw_plan(tensors, case["bits"], _bytes(dev.adamw_plan_bytes(tensors)))
        return
    s["work"] = _bytes(s["work_bytes"])


# ---- one pass -----------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        p, dev = s["ptr"], _device()
        if kind == "linear":
            dev.linear(s["desc"], p["X"], p["W"], p["Y"], bias=p["bias"], residual=p["residual"], Z=p["keepZ"], work=s["work"], work_bytes=s["work_bytes"])
        elif kind == "linear_grad":
            dev.linear_grad(s["desc"], p["dY"], p["X"], p["W"], p["Z"], dX=p["dX"], dW=p["dW"], dbias=p["dbias"], work=s["work"], work_bytes=s["work_bytes"])
        elif kind == "embedding":
            dev.embedding(s["desc"], p["table"], p["ids"], p["out"], p["flags"])
        elif kind == "embedding_grad":
            dev.embedding_grad(s["desc"], p["dY"], p["ids"], p["out"], p["flags"], s["work"], s["work_bytes"])
        else:
            dev.adamw_step(s["plan"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, step=STEP, seed=s["seed"])
    else:
        {"linear": _plain_linear, "linear_grad": _plain_linear_grad, "embedding": _plain_embedding, "embedding_grad": _plain_embedding_grad, "adamw": _plain_adamw}[kind](s)
    return _outputs(s)


def _outputs(s):
    kind = s["case"]["kind"]
    if kind == "linear":
        return {"Y": s["Y"], "Z": s["keepZ"]}
    if kind == "linear_grad":
        return {"dX": s["dX"], "dW": s["dW"], "dbias": s["dbias"]}
    if kind in ("embedding", "embedding_grad"):
        return {"out": s["out"], "flags": s["flags"]}
    o = {"param": s["param"], "master": s["master"]}
    if s["case"]["bits"] == 32:
        return {**o, "m": s["m"], "v": s["v"]}
    # the values that the bytes stand for, and the powers of two that they are times
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return {**o, "m": s["m"].view(e4m3), "m_scale": s["m_scale"].view(e8m0), "v_root": s["v"].view(e4m3), "v_scale": s["v_scale"].view(e8m0)}


_GELU0, _GELU1 = 0.7978845608028654, 0.044715


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(_GELU0 * (z + _GELU1 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_act_grad(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        t = torch.tanh(_GELU0 * (z + _GELU1 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _GELU0 * (1 + 3 * _GELU1 * z * z)
    p = 1 / (1 + torch.exp(-z))
    return p * (1 + z * (1 - p))


def _plain_linear(s):
    z = s["X"].float() @ s["W"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if s["keepZ"] is not None:
        s["keepZ"].copy_(z)
    y = _plain_act(z, s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    s["Y"].copy_(y)


def _plain_linear_grad(s):
    dz = s["dY"].float()
    if s["Z"] is not None:
        dz = dz * _plain_act_grad(s["Z"].float(), s["case"]["act"])
    s["dX"].copy_(dz @ s["W"].float())
    s["dW"].copy_(dz.t() @ s["X"].float())
    s["dbias"].copy_(dz.sum(0))


def _plain_embedding(s):
    s["out"].copy_(s["table"][s["ids"].long()].float() * SCALE)


def _plain_embedding_grad(s):
    d = torch.zeros(s["out"].shape, dtype=torch.float32, device="cuda:0")
    d.index_put_((s["ids"].long(),), s["dY"].float(), accumulate=True)
    s["out"].copy_(d * SCALE)


def _power(e):
    """2^e for whole e from -127 to 127, in 32 bits."""
    return torch.where(e < -126, torch.full_like(e, 0x00400000), (e + 127) << 23).view(torch.float32)


def _exponent(x):
    return (x.view(torch.int32) >> 23) - 127  # of x >= 0


def _to_8bit(x, u, root):
    """e4m3 bytes of x / 2^e and the bytes e + 127, one for each block of values, 2^e the least power of two
    (from 2^-127 on) with which all of the block are at most 448; x / 2^e is rounded to a neighbour of it, up with
    the probability of its distance from the lower one (u: a number of [0, 1) for each). A root is never rounded to 0."""
    a = torch.where(torch.isfinite(x), torch.abs(x), torch.zeros_like(x))
    top = a.amax(1)
    e = (_exponent(top) - 8 + ((top.view(torch.int32) & 0x7FFFFF) > 0x600000).int()).clamp(min=-127)
    y = a * _power(-e)[:, None]
    ey = _exponent(y).clamp(min=-6)
    code = 8 * (ey + 6) + torch.floor(y * _power(3 - ey) + u).int()
    if root:
        code = torch.where(a > 0, code.clamp(min=1), code)
    code = torch.where(torch.isfinite(x), code, torch.full_like(code, 127)) | (x < 0).int() << 7
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def _mix(x):
    """32 bits spread over each other: two rounds of a shift and a product, and a shift."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _plain_adamw(s):
    g = s["grad"].float()
    p = s["master"] if s["master"] is not None else s["param"].float()
    f = lambda x: float(np.float32(x))  # noqa: E731  (the step's constants, rounded once)
    if s["case"]["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = s["m"].view(torch.float8_e4m3fn).float() * _power(s["m_scale"].int() - 127)[:, None]
        r = s["v"].view(torch.float8_e4m3fn).float() * _power(s["v_scale"].int() - 127)[:, None]
        v = r * r
    m = f(BETA1) * m + f(1 - BETA1) * g
    v = f(BETA2) * v + (f(1 - BETA2) * g) * g
    r = torch.sqrt(v)
    update = (m / (r * f(1 / math.sqrt(1 - BETA2**STEP)) + f(EPS))) * f(LR / (1 - BETA1**STEP))
    p = p * (1 - f(LR) * s["decay"])[:, None] - update
    if s["master"] is not None:
        s["master"].copy_(p)
    s["param"].copy_(p)
    if s["case"]["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return
    # 32 random bits for each value, by its place among all blocks: 16 for each state
    h = _mix(torch.arange(m.numel(), device=m.device).view(m.shape) ^ s["seed"])
    for k, x, bits in (("m", m, h & 0xFFFF), ("v", r, h >> 16)):
        code, scale = _to_8bit(x, (bits.float() + 0.5) * 2.0**-16, k == "v")
        s[k].copy_(code)
        s[k + "_scale"].copy_(scale)


# ---- what a pass cannot do without, and its result in 64 bits ----------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("linear", "linear_grad"):
        M, N, K, e = case["M"], case["N"], case["K"], SIZES[case["type"]]
        if kind == "linear":
            ey = SIZES[case["y"]]
            return {"bytes": e * (M * K + N * K + case["keep"] * M * N + case["bias"] * N) + ey * M * N * (1 + case["residual"]), "flops": 2 * M * N * K}
        ew = SIZES[case["dw"]]
        return {"bytes": e * (2 * M * K + N * K + M * N * (1 + (case["act"] != "none"))) + ew * (N * K + N), "flops": 4 * M * N * K}
    if kind in ("embedding", "embedding_grad"):
        T, D, e = case["T"], case["D"], SIZES[case["type"]]
        if kind == "embedding":
            # a repeated token's row is read once: by Zipf's law nearly half of the tokens are new ones
            return {"bytes": e * D * (T + min(T, case["vocab"]) // 2) + case["ids"] // 8 * T, "flops": T * D}
        return {"bytes": e * T * D + SIZES[case["dw"]] * case["vocab"] * D + case["ids"] // 8 * T, "flops": T * D}
    n = sum(_sizes(case))
    state = 4 * n * 4 if case["bits"] == 32 else 4 * n + 4 * n // BLOCK
    param = 8 * n + SIZES[case["param"]] * n if case["master"] else 2 * SIZES[case["param"]] * n
    return {"bytes": param + SIZES[case["grad"]] * n + state, "flops": 15 * n}


def _exact_act(z, act):
    if act == "gelu":
        return z * torch.sigmoid(2 * _GELU0 * (z + _GELU1 * z**3))
    return {"none": lambda x: x, "relu": lambda x: x.clamp(min=0), "silu": lambda x: x * torch.sigmoid(x)}[act](z)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("linear", "linear_grad"):
        s = {k: x.double() if x is not None else None for k, x in _linear_inputs(case, seed).items()}
        if kind == "linear":
            z = torch.matmul(s["X"], s["W"].T)
            if case["bias"]:
                z += s["bias"]
            y = _exact_act(z, case["act"])
            return {"Y": y + s["residual"] if case["residual"] else y, "Z": z if case["keep"] else None}
        d = s["dY"]
        if s["Z"] is not None:
            z = s["Z"].requires_grad_()
            d = torch.autograd.grad(_exact_act(z, case["act"]), z, d)[0]
        return {"dX": torch.matmul(d, s["W"]), "dW": torch.matmul(d.T, s["X"]), "dbias": d.sum(0)}
    if kind == "embedding":
        s = _embedding_inputs(case, seed)
        return {"out": torch.index_select(s["table"], 0, s["ids"]).double() * SCALE, "flags": None}
    if kind == "embedding_grad":
        s = _embedding_inputs(case, seed)
        d = torch.zeros((case["vocab"], case["D"]), dtype=torch.float64, device="cuda:0")
        return {"out": d.index_add_(0, s["ids"], s["dY"].double() * SCALE), "flags": None}
    return _exact_adamw(case, _adamw_inputs(case, seed))


def _exact_adamw(case, s):
    eight = case["bits"] == 8
    if eight:
        two = lambda k: torch.pow(2.0, s[k].double() - 127)[:, None]  # noqa: E731
        m, v = (s[k].view(torch.float8_e4m3fn).double() * two(k + "_scale") for k in "mv")
        v = v.square()
    else:
        m, v = s["m"].double(), s["v"].double()
    g, p = s["grad"].double(), (s["master"] if case["master"] else s["param"]).double()
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g.square() - v)
    mean, var = m / (1 - BETA1**STEP), v / (1 - BETA2**STEP)
    p = p - LR * (mean / (var.sqrt() + EPS) + s["decay"].double()[:, None] * p)
    o = {"param": p, "master": p if case["master"] else None}
    if not eight:
        return {**o, "m": m, "v": v}
    i = torch.arange(p.numel(), device=p.device).view(p.shape)
    h = _mix(i ^ s["seed"])
    del i
    for k, name, x, bits in (("m", "m", m, h % 65536), ("v", "v_root", v.sqrt(), h // 65536)):
        top = x.abs().amax(1, keepdim=True)
        # the least power of two with top / 2^e <= 448, not under 2^-127
        f, e = torch.frexp(top / 448)
        e = torch.where(top > 0, e - (f == 0.5).int(), torch.full_like(e, -127)).clamp(min=-127).double()
        y = x.abs() / torch.pow(2.0, e)
        step = torch.pow(2.0, (torch.frexp(y)[1].double() - 1).clamp(min=-6) - 3)
        q = torch.floor(y / step + (bits.double() + 0.5) / 65536) * step
        if k == "v":
            q = torch.where(y > 0, q.clamp(min=2.0**-9), q)
        o[name], o[k + "_scale"] = torch.where(x < 0, -q, q), torch.pow(2.0, e[:, 0])
    return o
