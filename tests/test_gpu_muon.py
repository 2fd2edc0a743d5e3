"""oz_muon_step: momenta bit by bit with the header's FP32 operations, weights against the iteration in 64 bits (bounds as in the tests of
oz_orthogonalize, times what the step multiplies the result by)."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, ROUND, U32, Ptr, generator
from tests.test_gpu_orthogonalize import exact, rounding_of_x

pytestmark = pytest.mark.gpu


class Matrix:
    def __init__(self, rows, cols, param="f32", master=False, grad="f32", decay=0.1, scale=None, seed=1):
        g = generator(seed + 1000 * rows + cols)
        normal = lambda s: torch.randn((rows, cols), device="cuda:0", generator=g) * s  # noqa: E731
        self.rows, self.cols, self.type, self.decay = rows, cols, param, decay
        p = normal(0.05)
        self.param, self.master = p.to(DTYPE[param]), p.clone() if master else None
        self.grad, self.grad_type, self.m = normal(1e-2).to(DTYPE[grad]), grad, normal(1e-2)
        a = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
        self.tensor = ozd.muon_tensor(rows, cols, a(self.param), a(self.grad), a(self.m), a(self.master), param, grad, decay, scale)
        self.scale = self.tensor.lr_scale

    def step(self, lr, momentum, nesterov, gs=1.0, **options):
        """What the step makes of it: m' and the bounds of p'."""
        f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda:0")  # noqa: E731
        g = self.grad.float() * f(gs)
        m = f(momentum) * self.m + f(1 - momentum) * g
        u = f(momentum) * m + f(1 - momentum) * g if nesterov else m
        o = exact(u[None], **options)[0]
        p = (self.master if self.master is not None else self.param).double()
        want = p * (1 - float(f(lr)) * float(f(self.decay))) - o * float(f(lr)) * self.scale
        bound = (2e-3 if min(self.rows, self.cols) > 512 else 1e-5) + rounding_of_x() / max(float(o.norm()), 1e-30)
        peak = max(float(o.square().mean().sqrt()), float(o.abs().max()) / 20)
        off = 20 * bound * peak * lr * self.scale + 4 * U32 * (p.abs() + o.abs() * lr * self.scale)
        norm = bound * float(o.norm()) * lr * self.scale + 4 * U32 * float(p.norm())
        return m, want, off, norm

    def check(self, wanted):
        m, want, off, norm = wanted
        assert torch.equal(self.m, m), (self.rows, self.cols)
        got = self.master if self.master is not None else self.param
        half, floor = ROUND["f32" if self.master is not None else self.type]
        d = (got.double() - want).abs()
        assert bool((d <= off + half * (want.abs() + off) + floor).all()), (self.rows, self.cols, float(d.max()))
        assert float((got.double() - want).norm()) <= norm + half * float(want.norm()) + floor * want.numel() ** 0.5
        if self.master is not None:
            assert torch.equal(self.param, self.master.to(self.param.dtype))


def step(dev, matrices, lr=0.02, momentum=0.9, nesterov=True, grad_scale=None, plan=None, **options):
    plan = plan or dev.muon_plan([x.tensor for x in matrices])
    n = dev.muon_workspace(plan)
    work = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda:0")
    wanted = [x.step(lr, momentum, nesterov, 1.0 if grad_scale is None else float(grad_scale[0]), **options) for x in matrices if x.rows * x.cols]
    torch.cuda.synchronize()
    dev.muon_step(plan, lr, momentum, nesterov, grad_scale=Ptr(grad_scale) if grad_scale is not None else None, work=Ptr(work), work_bytes=n, **options)
    dev.sync()
    for x, w in zip([x for x in matrices if x.rows * x.cols], wanted):
        x.check(w)
    return plan


TYPES = [("f32", False, "f32"), ("f32", False, "bf16"), ("bf16", True, "bf16"), ("bf16", False, "f32"), ("f16", True, "f32"), ("f16", False, "f16")]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("nesterov", [True, False])
def test_types(dev, types, nesterov):
    print("muon", types, nesterov, flush=True)
    step(dev, [Matrix(70, 90, *types), Matrix(129, 33, *types), Matrix(1, 7, *types), Matrix(520, 530, *types)], nesterov=nesterov)


def test_many_sizes_together(dev):
    """Sizes mixed, wide, tall and square, several of one size, empty ones, types of their own; three steps with one plan."""
    sizes = [(64, 64), (128, 512), (512, 128), (3, 1000), (128, 512), (0, 5), (700, 650), (1, 1), (128, 512), (64, 64), (600, 1030), (5, 0), (1030, 600)]
    ms = [Matrix(r, c, *TYPES[i % len(TYPES)], seed=i) for i, (r, c) in enumerate(sizes)]
    plan = None
    for k in range(3):
        print("muon step", k, flush=True)
        plan = step(dev, ms, nesterov=bool(k % 2), plan=plan)


@pytest.mark.parametrize("size", [(2048, 1024), (1000, 3001), (2500, 2500)], ids=str)
def test_large(dev, size):
    print("muon", size, flush=True)
    step(dev, [Matrix(*size, "bf16", True, "bf16"), Matrix(*size, "f32", False, "f32", seed=2)])


def updates(dev, G):
    """The orthogonalized matrix in 32 bits: the negative of what a step makes of weights of zeros."""
    x = Matrix(*G.shape, decay=0.0, scale=1.0)
    x.param.zero_()
    x.grad.copy_(G)
    plan = dev.muon_plan([x.tensor])
    n = dev.muon_workspace(plan)
    work = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.muon_step(plan, 1.0, 0.0, True, work=Ptr(work), work_bytes=n)
    dev.sync()
    return -x.param.double()


@pytest.mark.parametrize("size", [(545, 4482), (4482, 545), (1030, 1030), (2100, 1500)], ids=str)
def test_updates_of_32_bit_weights(dev, size):
    """With B's diagonal in FP32 products of 11 bits leave Gaussian matrices of 513 to 1500 rows off by 4e-4 to 8.5e-4 (the same roundings in 64
    bits), with all of B in 11 bits by 1.3e-3 to 1.8e-3."""
    print("updates", size, flush=True)
    G = torch.randn(size, device="cuda:0", generator=generator(3))
    want = exact(G[None], eps=1e-7)[0]
    assert float((updates(dev, G) - want).norm() / want.norm()) <= 1.2e-3


def off_alike(n, a, b, c, steps=5):
    """Bound of the relative error for the identity of n rows, to first order: X = s I and s' = s p(s^2), p(q) = a + b q + c q^2. FP16 rounds h (twice
    in A) and A by half a step, 2^-11, alike for all values; B is its diagonal, in FP32."""
    s, e = n**-0.5, 0.0
    for _ in range(steps):
        q = s * s
        p = a + b * q + c * q * q
        e = abs((a + 3 * b * q + 5 * c * q * q) / p) * e + abs((b * q + 2 * c * q * q) / p) * 3 * 2.0**-11
        s *= p
    return e


@pytest.mark.parametrize("n", [513, 600, 1024, 2048, 4096])
def test_identity(dev, n):
    """All singular values, and all roundings, alike."""
    print("identity", n, flush=True)
    eye = torch.eye(n, device="cuda:0")
    got, want = updates(dev, eye), exact(eye[None], eps=1e-7)[0]
    assert torch.equal(got, torch.diag(torch.diagonal(got)))
    bound = off_alike(n, *ozd.NEWTON_SCHULZ)
    assert bound <= 1.12e-2 and float((got - want).norm() / want.norm()) <= 1.1 * bound + 1e-5


def test_grad_scale_decay_and_rate(dev):
    scale = torch.tensor([0.25], device="cuda:0")
    step(dev, [Matrix(80, 60, decay=0.0, scale=3.0), Matrix(60, 80, decay=0.5, scale=0.0)], lr=0.5, grad_scale=scale, steps=3, eps=1e-3)
    step(dev, [Matrix(80, 60)], lr=0.0, momentum=0.0)


def test_first_step_and_no_gradient(dev):
    """Momenta of zeros; a gradient of zeros as well leaves the decay alone."""
    a, b = Matrix(100, 50), Matrix(100, 50, seed=2)
    a.m.zero_()
    b.m.zero_()
    b.grad.zero_()
    step(dev, [a, b])


def test_a_gradient_that_is_not_finite_stays_in_its_matrix(dev):
    a, b, c = Matrix(90, 70), Matrix(90, 70, seed=2), Matrix(600, 520, seed=3)
    b.grad[3, 4] = float("inf")
    plan = dev.muon_plan([x.tensor for x in (a, b, c)])
    n = dev.muon_workspace(plan)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda:0")
    wa, wc = a.step(0.02, 0.9, True), c.step(0.02, 0.9, True)
    torch.cuda.synchronize()
    dev.muon_step(plan, 0.02, 0.9, work=Ptr(work), work_bytes=n)
    dev.sync()
    a.check(wa)
    c.check(wc)
    assert bool(torch.isnan(b.param).all())


def test_empty_plan(dev):
    plan = dev.muon_plan([])
    assert dev.muon_workspace(plan) == 0
    dev.muon_step(plan, 0.1)
    dev.sync()


def test_plan_memory_from_python(dev):
    """A buffer that is too small is refused before anything is copied."""
    ms = [Matrix(20, 30), Matrix(30, 20)]
    small = dev.alloc(32)
    with pytest.raises(RuntimeError, match="needed"):
        dev.muon_plan([x.tensor for x in ms], small)
    small.free()


def test_rounds_cut_across_sizes(dev):
    """So many tiles of several sizes that a last round's own launch takes up two of them."""
    sizes = [(2048, 2048)] * 3 + [(1024, 4096)] * 2 + [(3000, 1024)] * 2 + [(700, 600)] * 5
    step(dev, [Matrix(r, c, "bf16", True, "bf16", seed=i) for i, (r, c) in enumerate(sizes)])
    sizes = [(500, 1500)] * 6 + [(1500, 400)] * 7 + [(512, 512)] * 9
    step(dev, [Matrix(r, c, "f32", False, "f32", seed=i) for i, (r, c) in enumerate(sizes)], nesterov=False)


def test_two_handles_at_once(dev):
    """Two handles step two lists, each in its own workspace, with nothing between the calls."""
    other = ozd.Device(0)
    try:
        lists = [[Matrix(600, 700, seed=1), Matrix(90, 300, seed=2)], [Matrix(700, 600, seed=3), Matrix(128, 128, seed=4)]]
        wanted = [[x.step(0.02, 0.9, True) for x in l] for l in lists]
        plans = [d.muon_plan([x.tensor for x in l]) for d, l in zip((dev, other), lists)]
        sizes = [d.muon_workspace(p) for d, p in zip((dev, other), plans)]
        works = [torch.zeros(n, dtype=torch.uint8, device="cuda:0") for n in sizes]
        torch.cuda.synchronize()
        for d, p, w, n in zip((dev, other), plans, works, sizes):
            d.muon_step(p, 0.02, 0.9, work=Ptr(w), work_bytes=n)
        dev.sync()
        other.sync()
        for l, ws in zip(lists, wanted):
            for x, w in zip(l, ws):
                x.check(w)
    finally:
        other.close()
