"""The bits of the Newton-Schulz products as callers choose them: matrices and weights in FP32 have 22 without asking, large BF16 ones where `exact`
asks for them. Bounds as in the tests of oz_orthogonalize."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import Ptr
from tests.test_gpu_muon import Matrix, off_alike
from tests.test_gpu_orthogonalize import check, exact, gaussian, low_rank, rounding_of_x, run

pytestmark = pytest.mark.gpu


def updates(dev, G, plan_exact=None, master=False):
    """The orthogonalized matrix in 32 bits: the negative of what a step makes of weights of zeros."""
    x = Matrix(*G.shape, "bf16" if master else "f32", master, decay=0.0, scale=1.0)
    (x.master if master else x.param).zero_()
    x.grad.copy_(G)
    plan = dev.muon_plan([x.tensor], exact=plan_exact)
    n = dev.muon_workspace(plan)
    work = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.muon_step(plan, 1.0, 0.0, True, work=Ptr(work), work_bytes=n)
    dev.sync()
    return -(x.master if master else x.param).double()


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


SIZES = [(545, 4482), (4482, 545), (1030, 1030), (2100, 1500)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_32_bit_weights(dev, size):
    print("32-bit weights", size, flush=True)
    G = gaussian(1, *size, "f32")[0]
    want = exact(G[None])[0]
    assert off(updates(dev, G), want) <= 1e-5 + rounding_of_x() / float(want.norm())


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_what_a_plan_asks_for(dev, size):
    """Masters of 16-bit weights and FP32 weights alike: 11 bits or 22."""
    print("plans", size, flush=True)
    G = gaussian(1, *size, "f32")[0]
    want = exact(G[None])[0]
    for master in (False, True):
        assert off(updates(dev, G, True, master), want) <= 1e-5 + rounding_of_x() / float(want.norm())
        assert 1e-4 <= off(updates(dev, G, False, master), want) <= 1.2e-3
    assert torch.equal(updates(dev, G, None, True), updates(dev, G, False, True)) and torch.equal(updates(dev, G), updates(dev, G, True))


@pytest.mark.parametrize("n", [513, 600, 1024, 2048, 4096])
def test_identity_in_11_bits(dev, n):
    """All singular values, and all roundings, alike; B is its diagonal, which is kept in FP32."""
    print("identity", n, flush=True)
    eye = torch.eye(n, device="cuda:0")
    got, want = updates(dev, eye, False), exact(eye[None])[0]
    assert torch.equal(got, torch.diag(torch.diagonal(got)))
    assert off(got, want) <= 1.1 * off_alike(n, *ozd.NEWTON_SCHULZ) + 1e-5


@pytest.mark.parametrize("size", [(1, 513, 515), (2, 1030, 700), (1, 2048, 2048)], ids=str)
def test_exact_bf16_matrices(dev, size):
    for make in (gaussian, low_rank):
        print("orthogonalize exact", size, make.__name__, flush=True)
        G = make(*size, "bf16")
        check(run(dev, G, "bf16", exact=True), exact(G), 1e-5, "bf16")


def test_sizes_of_a_plan_by_themselves(dev):
    """FP32 weights of one size beside 16-bit ones of another, and of the same: a size with an FP32 weight has 22 bits."""
    ms = [Matrix(600, 700, "bf16", True, "bf16", seed=1), Matrix(700, 600, "f32", seed=2), Matrix(700, 600, "bf16", True, "bf16", seed=3), Matrix(90, 70, "f32", seed=4)]
    plan = dev.muon_plan([x.tensor for x in ms])
    assert [(plan.shape[k].rows, plan.exact >> k & 1) for k in range(plan.shapes)] == [(600, 0), (700, 1), (90, 1)]
    n = dev.muon_workspace(plan)
    work = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda:0")
    wanted = [x.step(0.02, 0.9, True) for x in ms]
    torch.cuda.synchronize()
    dev.muon_step(plan, 0.02, 0.9, work=Ptr(work), work_bytes=n)
    dev.sync()
    for x, w in zip(ms, wanted):
        x.check(w)
