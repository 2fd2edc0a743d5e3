"""What a program does to the weights of linear layers beside the product itself:

  "quantize"       rows as 8-bit integers with a scale each: activations by token, weights by channel
  "linear_i8"      Y = act(X W^T + bias) + residual with 8-bit integers, products of the scales of a token and a channel
  "orthogonalize"  the Newton-Schulz iteration, which moves all singular values of a matrix near 1
  "muon"           Muon's step over many matrices: momentum, orthogonalized, added to the weights

In the plain form an operator is the formula in elementary operations, in 32 bits. Otherwise it is the call
that a program makes of the device layer (oztt_amd.device) on tensors that it keeps in GPU memory.
"""
import ctypes
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the tokens of a batch of answers on their way into a layer: nothing but latency
        {"name": "quantize_24x2048", "kind": "quantize", "M": 24, "K": 2048, "type": "bf16", "pad": 0},
        # a layer's weights, once, or the tokens of a long prompt: the largest
        {"name": "quantize_8192", "kind": "quantize", "M": 8192, "K": 8192, "type": "bf16", "pad": 0},
        # one token through a square layer of an answering program: half the bytes of 16-bit weights
        {"name": "linear_i8_token", "kind": "linear_i8", "M": 1, "N": 8192, "K": 8192, "type": "bf16", "act": "none", "y": "bf16", "bias": False, "residual": True, "int8": False, "pad": 0},
        # a batch of answers being written, one token each, through a widening layer; FP16
        {"name": "linear_i8_batch", "kind": "linear_i8", "M": 24, "N": 8192, "K": 2048, "type": "f16", "act": "silu", "y": "f16", "bias": True, "residual": False, "int8": False, "pad": 0},
        # sizes that fit no tile, operands that are windows of wider matrices, tokens that are 8-bit integers already
        {"name": "linear_i8_ragged", "kind": "linear_i8", "M": 1000, "N": 700, "K": 1500, "type": "bf16", "act": "gelu", "y": "f32", "bias": True, "residual": True, "int8": True, "pad": 12},
        # a long prompt through a square layer, everything in the epilogue: the largest product
        {"name": "linear_i8_8192", "kind": "linear_i8", "M": 8192, "N": 8192, "K": 8192, "type": "bf16", "act": "gelu", "y": "bf16", "bias": True, "residual": True, "int8": False, "pad": 0},
        # the update of a small network's widening layer: a chain of short products
        {"name": "orthogonalize_small", "kind": "orthogonalize", "count": 1, "rows": 512, "cols": 128, "type": "bf16", "pad": 0},
        # sizes that fit no tile, several matrices in one call, windows of wider ones
        {"name": "orthogonalize_ragged", "kind": "orthogonalize", "count": 3, "rows": 700, "cols": 1500, "type": "f16", "pad": 12},
        # the update of a large square layer
        {"name": "orthogonalize_8192", "kind": "orthogonalize", "count": 1, "rows": 8192, "cols": 8192, "type": "bf16", "pad": 0},
        # all layers of a small network: a widening and a narrowing one in each of some blocks, FP32
        {"name": "muon_small", "kind": "muon", "blocks": 12, "width": 128, "hidden": 512, "param": "f32", "master": False, "grad": "f32", "nesterov": True},
        # the same of a network whose sizes fit no tile
        {"name": "muon_ragged", "kind": "muon", "blocks": 5, "width": 500, "hidden": 1500, "param": "f16", "master": True, "grad": "f32", "nesterov": False},
        # some blocks of a large network, BF16 with 32-bit copies
        {"name": "muon_large", "kind": "muon", "blocks": 4, "width": 2048, "hidden": 8192, "param": "bf16", "master": True, "grad": "bf16", "nesterov": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear_i8", "linear_i8", "linear_i8", "orthogonalize", "orthogonalize", "muon", "muon"])
    c = {"kind": kind}
    if kind == "quantize":
        while True:
            M, K = _log(rng, 1, 65536), _log(rng, 16, 32768)
            if M * K <= 2**26:
                break
        c.update(M=M, K=-(-K // 64) * 64 if rng.random() < 0.5 else K, type=rng.choice(["bf16", "f16", "f32"]), pad=rng.choice([0, 0, 8, 5]))
    elif kind == "linear_i8":
        while True:
            M, N, K = _log(rng, 1, 8192), _log(rng, 16, 8192), _log(rng, 16, 16384)
            if M * N * K <= 2.0**37:
                break
        if rng.random() < 0.5:  # widths as networks have them
            N, K = -(-N // 64) * 64, -(-K // 64) * 64
        t = rng.choice(["bf16", "bf16", "f16"])
        c.update(M=M, N=N, K=K, type=t, act=rng.choice(["none", "relu", "gelu", "silu"]), y=rng.choice([t, t, "f32"]), bias=rng.random() < 0.6, residual=rng.random() < 0.4, int8=rng.random() < 0.4, pad=rng.choice([0, 0, 0, 8, 5]))
    elif kind == "orthogonalize":
        while True:
            count, rows, cols = rng.choice([1, 1, 1, 2, 5]), _log(rng, 16, 8192), _log(rng, 16, 8192)
            if count * _products(rows, cols) <= _products(8192, 8192) / 4:
                break
        c.update(count=count, rows=rows, cols=cols, type=rng.choice(["bf16", "bf16", "f16"]), pad=rng.choice([0, 0, 0, 8, 5]))
        if rng.random() < 0.5:
            c.update(rows=-(-rows // 64) * 64, cols=-(-cols // 64) * 64)
    else:
        while True:
            blocks, width, hidden = _log(rng, 1, 30), _log(rng, 16, 4096), _log(rng, 16, 8192)
            if blocks * (_products(width, width) + 2 * _products(width, hidden)) <= _products(8192, 8192) / 2:
                break
        if rng.random() < 0.5:
            width, hidden = -(-width // 64) * 64, -(-hidden // 64) * 64
        param = rng.choice(["f32", "bf16", "f16"])
        c.update(blocks=blocks, width=width, hidden=hidden, param=param, master=param != "f32" and rng.random() < 0.7, grad=rng.choice([param, "f32"]), nesterov=rng.random() < 0.7)
    return c


# ---- inputs -----------------------------------------------------------------------------------------

STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7  # of the Newton-Schulz iteration
LR, MOMENTUM, DECAY = 1e-4, 0.95, 0.1
LEAST = 127.0 * 2.0**-126  # of a row's largest value, so that its scale is a normal number


def _generator(seed):
    return torch.Generator(device="cuda:0").manual_seed((int(seed) * 2654435761 + 54321) % (1 << 62))


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda:0", generator=g) * scale).to(dtype)


def _window(x, pad):
    """x as a window of matrices `pad` columns wider, whose other columns hold what nobody may use."""
    if not pad:
        return x
    w = torch.full((*x.shape[:-1], x.shape[-1] + pad), float("nan") if x.is_floating_point() else 77, dtype=x.dtype, device=x.device)
    w[..., : x.shape[-1]] = x
    return w[..., : x.shape[-1]]


def _rows(shape, dtype, pad):
    """An output of the same kind."""
    return torch.zeros((*shape[:-1], shape[-1] + pad), dtype=dtype, device="cuda:0")[..., : shape[-1]]


def _activations(g, M, K):
    """Values whose channels differ in size, a few of them much larger than the others."""
    size = torch.exp(0.5 * torch.randn(K, device="cuda:0", generator=g)) * (1 + 9 * (torch.rand(K, device="cuda:0", generator=g) > 0.99))
    return torch.randn((M, K), device="cuda:0", generator=g) * size


def _row_pad(K, pad):
    """Columns behind K of an 8-bit matrix, whose rows begin at multiples of 4 bytes."""
    return -(-(K + pad) // 4) * 4 - K


def _gradient(g, count, rows, cols):
    """Gradients of layers: some strong directions, noise, columns that differ in size."""
    k = 16
    x = torch.matmul(torch.randn((count, rows, k), device="cuda:0", generator=g), torch.randn((count, k, cols), device="cuda:0", generator=g)) * (0.25 * 1e-3)
    x += torch.randn((count, rows, cols), device="cuda:0", generator=g) * 3e-4
    return x * torch.exp(0.5 * torch.randn((count, 1, cols), device="cuda:0", generator=g))


def _shapes(case):
    """A network's layers by shape: a square one, a widening and a narrowing one in each block."""
    w, h, n = case["width"], case["hidden"], case["blocks"]
    return [(n, w, w), (n, h, w), (n, w, h)]


def _inputs(case, seed):
    g, kind, pad = _generator(seed), case["kind"], case.get("pad", 0)
    if kind == "quantize":
        return {"X": _window(_activations(g, case["M"], case["K"]).to(DTYPES[case["type"]]), pad)}
    if kind == "linear_i8":
        M, N, K, t = case["M"], case["N"], case["K"], DTYPES[case["type"]]
        s = {"X": _activations(g, M, K).to(t), "x_scale": None}
        if case["int8"]:
            q, s["x_scale"] = _quantized(s["X"])
            s["X"] = _window(q, _row_pad(K, pad))
        else:
            s["X"] = _window(s["X"], pad)
        q, s["w_scale"] = _quantized(_normal(g, (N, K), scale=K**-0.5))
        s["W"] = _window(q, _row_pad(K, pad))
        s["bias"] = _normal(g, (N,), t, 0.2) if case["bias"] else None
        s["residual"] = _window(_normal(g, (M, N), DTYPES[case["y"]]), pad) if case["residual"] else None
        return s
    if kind == "orthogonalize":
        return {"G": _window(_gradient(g, case["count"], case["rows"], case["cols"]).to(DTYPES[case["type"]]), pad)}
    s = {}
    for i, shape in enumerate(_shapes(case)):
        p = _normal(g, shape, scale=0.02)
        s["param", i], s["master", i] = p.to(DTYPES[case["param"]]), p if case["master"] else None
        s["grad", i] = _gradient(g, *shape).to(DTYPES[case["grad"]])
        s["m", i] = _gradient(g, *shape) * 0.5
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
    s = {"case": case, **_inputs(case, seed)}
    if kind == "quantize":
        s["Q"] = _rows((case["M"], case["K"]), torch.int8, _row_pad(case["K"], pad))
        s["scale"] = torch.zeros(case["M"], dtype=torch.float32, device="cuda:0")
    elif kind == "linear_i8":
        s["Y"] = _rows((case["M"], case["N"]), DTYPES[case["y"]], pad)
    elif kind == "orthogonalize":
        s["O"] = _rows((case["count"], case["rows"], case["cols"]), DTYPES[case["type"]], pad)
    if own:
        _prepare_call(s)
    return s


def _prepare_call(s):
    """What a program keeps beside its tensors: descriptors, workspaces and the optimizer's plan."""
    from oztt_amd import device as ozd

    case, dev = s["case"], _device()
    kind = case["kind"]
    s["ptr"] = {k: _Ptr(x) for k, x in s.items() if isinstance(x, torch.Tensor) or x is None}
    s["work_bytes"] = 0
    if kind == "quantize":
        s["desc"] = ozd.quantize_desc(case["M"], case["K"], case["type"], ldx=s["X"].stride(0), ldq=s["Q"].stride(0))
    elif kind == "linear_i8":
        r = s["residual"].stride(0) if case["residual"] else 0
        s["desc"] = ozd.linear_i8_desc(case["M"], case["N"], case["K"], case["type"], case["act"], case["y"], x_int8=case["int8"],
                                       ldx=s["X"].stride(0), ldw=s["W"].stride(0), ldy=s["Y"].stride(0), ldr=r)
        s["work_bytes"] = dev.linear_i8_workspace(s["desc"])
    elif kind == "orthogonalize":
        s["desc"] = ozd.orthogonalize_desc(case["rows"], case["cols"], case["count"], case["type"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS,
                                           ldg=s["G"].stride(1), ldo=s["O"].stride(1), stride_g=s["G"].stride(0), stride_o=s["O"].stride(0))
        s["work_bytes"] = dev.orthogonalize_workspace(s["desc"])
    else:
        at = lambda k, i, j: s[k, i][j].data_ptr() if s[k, i] is not None else 0  # noqa: E731
        tensors = [ozd.muon_tensor(rows, cols, at("param", i, j), at("grad", i, j), at("m", i, j), master=at("master", i, j), param_type=case["param"],
                                   grad_type=case["grad"], weight_decay=DECAY, lr_scale=_lr_scale(rows, cols))
                   for i, (count, rows, cols) in enumerate(_shapes(case)) for j in range(count)]
        s["plan"] = dev.muon_plan(tensors, _bytes(dev.muon_plan_bytes(tensors)))
        s["work_bytes"] = dev.muon_workspace(s["plan"])
    s["work"] = _bytes(s["work_bytes"])


# ---- one pass -----------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        p, dev = s["ptr"], _device()
        if kind == "quantize":
            dev.quantize_rows(s["desc"], p["X"], p["Q"], p["scale"])
        elif kind == "linear_i8":
            dev.linear_i8(s["desc"], p["X"], p["W"], p["w_scale"], p["Y"], x_scale=p["x_scale"], bias=p["bias"], residual=p["residual"], work=s["work"], work_bytes=s["work_bytes"])
        elif kind == "orthogonalize":
            dev.orthogonalize(s["desc"], p["G"], p["O"], s["work"], s["work_bytes"])
        else:
            dev.muon_step(s["plan"], lr=LR, momentum=MOMENTUM, nesterov=s["case"]["nesterov"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, work=s["work"], work_bytes=s["work_bytes"])
    else:
        {"quantize": _plain_quantize, "linear_i8": _plain_linear_i8, "orthogonalize": _plain_orthogonalize, "muon": _plain_muon}[kind](s)
    return _outputs(s)


def _outputs(s):
    kind = s["case"]["kind"]
    if kind == "quantize":
        return {"Q": s["Q"], "scale": s["scale"]}
    if kind == "linear_i8":
        return {"Y": s["Y"]}
    if kind == "orthogonalize":
        return {"O": s["O"]}
    return {k: [s[k, i] for i in range(3)] for k in ("param", "master", "m")}


def _quantized(x):
    """8-bit integers and a scale for each row: all in 32 bits, ties to even; a row with a value that is not finite has no scale."""
    x = x.float()
    a = x.abs().amax(1)
    a = torch.where(torch.isfinite(a), a.clamp(min=LEAST), torch.full_like(a, float("nan")))
    q = torch.nan_to_num(torch.round(x * (127 / a)[:, None]))
    return q.to(torch.int8), a / 127


def _plain_quantize(s):
    q, scale = _quantized(s["X"])
    s["Q"].copy_(q)
    s["scale"].copy_(scale)


_GELU0, _GELU1 = 0.7978845608028654, 0.044715


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(_GELU0 * (z + _GELU1 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_linear_i8(s):
    q, scale = (s["X"], s["x_scale"]) if s["case"]["int8"] else _quantized(s["X"])
    y = torch.matmul(q.float(), s["W"].float().t()) * scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _plain_act(y, s["case"]["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    s["Y"].copy_(y)


def _plain_newton_schulz(x):
    """Of a batch of matrices in 32 bits. The products are those of the shorter side."""
    a, b, c = COEFFICIENTS
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        g = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x.transpose(1, 2) if tall else x


def _plain_orthogonalize(s):
    s["O"].copy_(_plain_newton_schulz(s["G"].float()))


def _lr_scale(rows, cols):
    """Makes an orthogonal update's values as large as 0.2, what AdamW's are."""
    return 0.2 * math.sqrt(max(rows, cols))


def _plain_muon(s):
    for i, (_, rows, cols) in enumerate(_shapes(s["case"])):
        g = s["grad", i].float()
        m = MOMENTUM * s["m", i] + (1 - MOMENTUM) * g
        o = _plain_newton_schulz(MOMENTUM * m + (1 - MOMENTUM) * g if s["case"]["nesterov"] else m)
        p = s["master", i] if s["master", i] is not None else s["param", i].float()
        p = p * (1 - LR * DECAY) - o * (LR * _lr_scale(rows, cols))
        if s["master", i] is not None:
            s["master", i].copy_(p)
        s["param", i].copy_(p)
        s["m", i].copy_(m)


# ---- what a pass cannot do without, and its result in 64 bits ----------------------------------------


def _products(rows, cols):
    """Operations of an orthogonalization: both products of a matrix with its transpose are symmetric, half of their values do."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3 * m * m * n + m * m * m)


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        return {"bytes": (SIZES[case["type"]] + 1) * case["M"] * case["K"] + 4 * case["M"], "flops": 3 * case["M"] * case["K"]}
    if kind == "linear_i8":
        M, N, K, e, ey = case["M"], case["N"], case["K"], SIZES[case["type"]], SIZES[case["y"]]
        x = M * K + 4 * M if case["int8"] else e * M * K
        return {"bytes": x + N * K + 4 * N + case["bias"] * e * N + ey * M * N * (1 + case["residual"]), "flops": 2 * M * N * K}
    if kind == "orthogonalize":
        n = case["count"] * case["rows"] * case["cols"]
        return {"bytes": 2 * SIZES[case["type"]] * n, "flops": case["count"] * _products(case["rows"], case["cols"])}
    n = sum(c * rows * cols for c, rows, cols in _shapes(case))
    param = 8 * n + SIZES[case["param"]] * n if case["master"] else 2 * SIZES[case["param"]] * n
    return {"bytes": param + SIZES[case["grad"]] * n + 8 * n, "flops": sum(c * _products(rows, cols) for c, rows, cols in _shapes(case))}


def _exact_quantized(x):
    """The definition rounds the reciprocal of a scale and its products with the values to 32 bits."""
    x = x.double()
    top = torch.maximum(x.amax(1), -x.amin(1)).clamp(min=LEAST)
    q = (x * (127 / top).float().double()[:, None]).float().double()
    floor = torch.floor(q)
    up = (q - floor > 0.5) | ((q - floor == 0.5) & (torch.remainder(floor, 2) == 1))
    return floor + up, (top / 127).float().double()


def _exact_act(z, act):
    if act == "gelu":
        return z * torch.sigmoid(2 * _GELU0 * (z + _GELU1 * z**3))
    return {"none": lambda x: x, "relu": lambda x: x.clamp(min=0), "silu": lambda x: x * torch.sigmoid(x)}[act](z)


def _exact_orthogonal(u):
    a, b, c = COEFFICIENTS
    u = u / (torch.linalg.vector_norm(u) + EPS)
    eye = torch.eye(min(u.shape), dtype=torch.float64, device=u.device)
    for _ in range(STEPS):
        s = u.mT @ u if u.shape[0] > u.shape[1] else u @ u.mT
        p = a * eye + s @ (b * eye + c * s)
        u = u @ p if u.shape[0] > u.shape[1] else p @ u
    return u


def exact(case, seed):
    kind, s = case["kind"], _inputs(case, seed)
    if kind == "quantize":
        q, scale = _exact_quantized(s["X"])
        return {"Q": q.to(torch.int8), "scale": scale}
    if kind == "linear_i8":
        x, sx = (s["X"].double(), s["x_scale"].double()) if case["int8"] else _exact_quantized(s["X"])
        y = torch.matmul(x * sx[:, None], (s["W"].double() * s["w_scale"].double()[:, None]).T)
        if case["bias"]:
            y += s["bias"].double()
        y = _exact_act(y, case["act"])
        return {"Y": y + s["residual"].double() if case["residual"] else y}
    if kind == "orthogonalize":
        return {"O": torch.stack([_exact_orthogonal(x.double()) for x in s["G"]])}
    out = {"param": [], "master": [], "m": []}
    for i, (count, rows, cols) in enumerate(_shapes(case)):
        g, m = s["grad", i].double(), s["m", i].double()
        m = m + (1 - MOMENTUM) * (g - m)
        u = m + (1 - MOMENTUM) * (g - m) if case["nesterov"] else m
        o = torch.stack([_exact_orthogonal(x) for x in u])
        p = (s["master", i] if case["master"] else s["param", i]).double()
        p = p - LR * (DECAY * p + _lr_scale(rows, cols) * o)
        out["param"].append(p)
        out["master"].append(p if case["master"] else None)
        out["m"].append(m)
    return out
