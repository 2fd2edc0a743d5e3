"""oz_embedding and oz_embedding_grad against the formulas in 64 bits.

Bounds: the lookup is one product, rounded once. A sum of n values in FP32, in any order, is off by at most n 2^-24
times the sum of their sizes; the scale and the output are one rounding each."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, U32, Ptr, generator, rounded, window, within

pytestmark = pytest.mark.gpu


def tokens(kind, T, vocab, bits, seed):
    g = generator(seed)
    if kind == "same":
        t = torch.full((T,), vocab // 2, device="cuda:0")
    elif kind == "frequent":  # a word in three is the same, the others rare
        t = torch.randint(0, vocab, (T,), device="cuda:0", generator=g)
        t[torch.rand(T, device="cuda:0", generator=g) < 0.3] = vocab // 3
    elif kind == "sorted":
        t = torch.arange(T, device="cuda:0") % vocab
    else:
        t = torch.randint(0, vocab, (T,), device="cuda:0", generator=g)
    return t.to(torch.int32 if bits == 32 else torch.int64)


@pytest.mark.parametrize("T,vocab,D", [(0, 5, 8), (1, 1, 1), (3, 10, 7), (5, 100, 512), (100, 50, 520), (1000, 3, 1030), (33, 2000, 4096)])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [32, 64])
def test_lookup(dev, T, vocab, D, t, bits):
    for pad, shift in ((0, 0), (8, 0), (3, 1)):
        print("embedding", T, vocab, D, t, bits, pad, shift, flush=True)
        table = window(torch.randn((vocab, D), device="cuda:0", generator=generator(1)).to(DTYPE[t]), pad, shift)[0]
        ids = tokens("random", T, vocab, bits, 2)
        out, around = window(torch.full((T, D), 7.0, device="cuda:0", dtype=DTYPE[t]), pad, shift, fill=5.0)
        flags = torch.zeros(1, dtype=torch.int32, device="cuda:0")
        torch.cuda.synchronize()
        dev.embedding(ozd.embedding_desc(T, vocab, D, t, bits, scale=0.3, ldt=D + pad, ldo=D + pad), Ptr(table), Ptr(ids), Ptr(out), Ptr(flags))
        dev.sync()
        assert torch.equal(out, (table[ids.long()].float() * torch.tensor(0.3)).to(DTYPE[t]))
        out.fill_(5.0)
        assert bool((around == 5.0).all()) and not int(flags)


@pytest.mark.parametrize("D", [9, 16, 22, 33, 64, 100, 129, 200, 256, 257, 511, 513])
def test_lookup_widths(dev, D):
    """Several rows a wave, one, and a second wave for a few values; tokens outside the vocabulary among them."""
    T, vocab = 301, 70
    for t in ("bf16", "f32"):
        print("embedding", D, t, flush=True)
        table = torch.randn((vocab, D), device="cuda:0", generator=generator(1)).to(DTYPE[t])
        ids = tokens("random", T, vocab, 32, 3)
        ids[::7] = vocab
        out, flags = torch.full((T, D), 7.0, device="cuda:0", dtype=DTYPE[t]), torch.zeros(1, dtype=torch.int32, device="cuda:0")
        torch.cuda.synchronize()
        dev.embedding(ozd.embedding_desc(T, vocab, D, t, 32, scale=0.3), Ptr(table), Ptr(ids), Ptr(out), Ptr(flags))
        dev.sync()
        want = (table[ids.long().clamp(max=vocab - 1)].float() * torch.tensor(0.3)).to(DTYPE[t])
        want[::7] = 0
        assert torch.equal(out, want) and int(flags) == 1


@pytest.mark.parametrize("bits", [32, 64])
def test_tokens_outside_the_vocabulary(dev, bits):
    """They give rows of zeros and no gradient, set the flag, and leave the others alone; infinities of the table do
    not reach their rows."""
    vocab, D = 40, 72
    table = torch.full((vocab, D), float("inf"), device="cuda:0")
    table[3] = 2.0
    bad = [-1, vocab, 2**31 - 1, -2**31] + ([2**40 + 3, -2**62] if bits == 64 else [])
    ids = torch.tensor([3] + bad + [3], device="cuda:0", dtype=torch.int32 if bits == 32 else torch.int64)
    T = len(ids)
    out, flags = torch.full((T, D), 9.0, device="cuda:0"), torch.zeros(2, dtype=torch.int32, device="cuda:0")
    d = ozd.embedding_desc(T, vocab, D, "f32", bits)
    n = dev.embedding_grad_workspace(d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda:0")
    dout = torch.randn((T, D), device="cuda:0")
    grad = torch.full((vocab, D), 9.0, device="cuda:0")
    torch.cuda.synchronize()
    dev.embedding(d, Ptr(table), Ptr(ids), Ptr(out), Ptr(flags))
    dev.embedding_grad(d, Ptr(dout), Ptr(ids), Ptr(grad), Ptr(flags[1:]), Ptr(work), n)
    dev.sync()
    assert bool((out[0] == 2).all()) and bool((out[-1] == 2).all()) and not out[1:-1].any()
    assert flags.tolist() == [1, 1]
    want = torch.zeros((vocab, D), device="cuda:0")
    want[3] = dout[0] + dout[-1]
    assert torch.equal(grad, want)


def gradient(dev, kind, T, vocab, D, t="bf16", dw="f32", bits=32, scale=0.3, accumulate=False, padding=-1, pad=0, shift=0, seed=4):
    ids = tokens(kind, T, vocab, bits, seed)
    g = generator(seed + 1)
    dout = window(torch.randn((T, D), device="cuda:0", generator=g).to(DTYPE[t]), pad, shift)[0]
    before = torch.randn((vocab, D), device="cuda:0", generator=g).to(DTYPE[dw])
    table, around = window(before, pad, shift, fill=5.0)
    d = ozd.embedding_desc(T, vocab, D, t, bits, scale=scale, grad_type=dw, accumulate=accumulate, padding=padding, ldt=D + pad, ldo=D + pad)
    n = dev.embedding_grad_workspace(d)
    work = torch.full((max(n, 16),), 0x7F, dtype=torch.uint8, device="cuda:0")
    flags = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    torch.cuda.synchronize()
    dev.embedding_grad(d, Ptr(dout), Ptr(ids), Ptr(table), Ptr(flags), Ptr(work), n)
    dev.sync()
    # the sums on the host: added up on the GPU, a million values of one row wait for each other
    keep = (ids.long() != padding).cpu()
    idx, x = ids.long().cpu()[keep], dout.double().cpu()[keep]
    count = torch.bincount(idx, minlength=vocab).double()[:, None].cuda()
    add = lambda v: torch.zeros((vocab, D), dtype=torch.float64).index_add_(0, idx, v).cuda()  # noqa: E731
    s = float(torch.tensor(scale))
    want, size = s * add(x), s * add(x.abs())
    bound = (count + 2) * U32 * size
    if accumulate:
        want, bound = want + before.double(), bound + U32 * (want.abs() + before.double().abs())
    within(table, want, bound + rounded(want.abs() + bound, dw), "dTable")
    if not accumulate:
        assert not table[(count == 0).flatten()].any()
    got = table.clone()
    table.fill_(5.0)
    assert bool((around == 5.0).all()) and not int(flags)
    return got


# from no token to lists longer than a tile, and vocabularies of one to three digits
@pytest.mark.parametrize("kind", ["random", "same", "frequent", "sorted"])
@pytest.mark.parametrize("T,vocab,D", [(0, 6, 8), (1, 1, 1), (2, 70, 520), (31, 9, 64), (32, 40, 7), (33, 400, 8), (65, 600, 1032),
                                       (700, 70, 500), (4095, 511, 64), (4097, 513, 72), (9000, 3000, 136), (40000, 300000, 8),
                                       (70000, 1 << 17, 16), (1100000, 70000, 8)])
def test_gradient(dev, kind, T, vocab, D):
    print("embedding_grad", kind, T, vocab, D, flush=True)
    gradient(dev, kind, T, vocab, D)


@pytest.mark.parametrize("t,dw", [("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_forms(dev, t, dw, bits, accumulate):
    for pad, shift, padding in ((0, 0, -1), (8, 0, 20), (3, 1, 41)):
        print("embedding_grad", t, dw, bits, accumulate, pad, shift, padding, flush=True)
        gradient(dev, "frequent", 500, 123, 200, t, dw, bits, accumulate=accumulate, pad=pad, shift=shift, padding=padding)


def test_all_padding(dev):
    got = gradient(dev, "same", 300, 40, 24, padding=20)
    assert not got.any()


def test_same_bits_again(dev):
    a = [gradient(dev, "frequent", 5000, 700, 264, "bf16", "f32") for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_gradient_against_differences(dev):
    """The lookup is linear in the table: the difference of the outputs for two tables, times dOut, is the
    gradient times the tables' difference, to FP32 rounding of the two sums of T D terms."""
    T, vocab, D = 300, 50, 64
    g = generator(8)
    ids = tokens("frequent", T, vocab, 64, 9)
    a, b, c = (torch.randn(s, device="cuda:0", generator=g) for s in ((vocab, D), (vocab, D), (T, D)))
    oa, ob, grad = torch.zeros_like(c), torch.zeros_like(c), torch.zeros_like(a)
    d = ozd.embedding_desc(T, vocab, D, "f32", 64, scale=0.5)
    n = dev.embedding_grad_workspace(d)
    work = torch.zeros(n, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.embedding(d, Ptr(a), Ptr(ids), Ptr(oa))
    dev.embedding(d, Ptr(b), Ptr(ids), Ptr(ob))
    dev.embedding_grad(d, Ptr(c), Ptr(ids), Ptr(grad), None, Ptr(work), n)
    dev.sync()
    left = float(((oa.double() - ob.double()) * c.double()).sum())
    right = float((grad.double() * (a.double() - b.double())).sum())
    size = float(((oa.double().abs() + ob.double().abs()) * c.double().abs()).sum())
    assert abs(left - right) <= T * U32 * size


def test_refusals_name_what_is_wrong(dev):
    x = torch.zeros(4096, device="cuda:0")
    p, odd = Ptr(x), Ptr(x.view(torch.uint8)[1:])
    d = ozd.embedding_desc(4, 8, 16, "f32", 32)
    for what, call in (
            ("null operand", lambda: dev.embedding(d, Ptr(None), p, p)),
            ("addresses", lambda: dev.embedding(d, p, odd, p)),
            ("ids' type", lambda: dev.embedding(ozd.embedding_desc(4, 8, 16, "f32", 16), p, p, p)),
            ("leading dimension", lambda: dev.embedding(ozd.embedding_desc(4, 8, 16, "f32", ldt=15), p, p, p)),
            ("workspace", lambda: dev.embedding_grad(d, p, p, p)),
            ("gradient's type", lambda: dev.embedding_grad(ozd.embedding_desc(4, 8, 16, "bf16", grad_type="f16"), p, p, p))):
        with pytest.raises(RuntimeError, match=what):
            call()
    dev.sync()
    assert not x.any()
