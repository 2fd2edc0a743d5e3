"""oz_embedding and oz_embedding_grad at the ends of their range: more tokens than one row of a grid holds, tables past 4 GiB, and
vocabularies whose tokens take four digits of the sort."""
import pytest
import torch

from oztt_amd import device as ozd
from tests.operator_cases import DTYPE, Ptr, generator

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    """Up to 40 GB a test are given back."""
    yield
    torch.cuda.empty_cache()


def test_lookups_beyond_a_row_of_a_grid(dev):
    """2^25 tokens and more, a wave each: every row is its token's."""
    T, vocab, D = 2**25 + 41, 200, 264
    print("embedding", T, vocab, D, flush=True)
    table = torch.randn((vocab, D), device="cuda:0", generator=generator(1)).bfloat16()
    ids = torch.randint(0, vocab, (T,), device="cuda:0", dtype=torch.int32, generator=generator(2))
    out = torch.zeros((T, D), dtype=torch.bfloat16, device="cuda:0")
    torch.cuda.synchronize()
    dev.embedding(ozd.embedding_desc(T, vocab, D, "bf16", 32), Ptr(table), Ptr(ids), Ptr(out))
    dev.sync()
    for i in range(0, T, 2**22):
        assert torch.equal(out[i : i + 2**22], table[ids[i : i + 2**22].long()])


def test_gradient_beyond_a_row_of_a_grid(dev):
    """2^30 tokens and more, all but some of them padding."""
    T, vocab, D = 2**30 + 77, 1000, 2
    print("embedding_grad", T, vocab, D, flush=True)
    ids = torch.full((T,), 999, dtype=torch.int32, device="cuda:0")
    at = torch.cat([torch.randint(0, T, (1000,), device="cuda:0", generator=generator(3)), torch.tensor([0, 2**30 - 1, 2**30, T - 1], device="cuda:0")]).unique()
    ids[at] = torch.randint(0, 999, (len(at),), device="cuda:0", dtype=torch.int32, generator=generator(4))
    dout = torch.full((T, D), 100.0, dtype=torch.bfloat16, device="cuda:0")
    dout[at] = torch.randint(-8, 9, (len(at), D), device="cuda:0", generator=generator(5)).bfloat16()
    table = torch.full((vocab, D), 9.0, device="cuda:0")
    d = ozd.embedding_desc(T, vocab, D, "bf16", 32, grad_type="f32", padding=999)
    n = dev.embedding_grad_workspace(d)
    work = torch.empty(n, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.embedding_grad(d, Ptr(dout), Ptr(ids), Ptr(table), None, Ptr(work), n)
    dev.sync()
    # small whole numbers: every order gives the same sum
    want = torch.zeros((vocab, D), device="cuda:0").index_add_(0, ids[at].long(), dout[at].float())
    assert torch.equal(table, want)


@pytest.mark.parametrize("T", [700, 3000])
def test_tokens_of_four_digits(dev, T):
    vocab, D = 2**27 + 3, 3
    print("embedding_grad", T, vocab, D, flush=True)
    g = generator(T)
    ids = torch.randint(0, vocab, (T,), device="cuda:0", generator=g)
    ids[:4] = torch.tensor([vocab - 1, 0, 2**27, vocab - 1], device="cuda:0")
    ids[T // 2 :: 3] = ids[5]
    dout = torch.randint(-8, 9, (T, D), device="cuda:0", generator=g).float()
    table = torch.full((vocab, D), 9.0, device="cuda:0")
    d = ozd.embedding_desc(T, vocab, D, "f32", 64)
    n = dev.embedding_grad_workspace(d)
    work = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda:0")
    torch.cuda.synchronize()
    dev.embedding_grad(d, Ptr(dout), Ptr(ids), Ptr(table), None, Ptr(work), n)
    dev.sync()
    assert torch.equal(table, torch.zeros((vocab, D), device="cuda:0").index_add_(0, ids, dout))


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_tables_past_4_gib(dev, t):
    """Rows on either side of 2^31 and 2^32 bytes, looked up and written, in rows apart by more than their length."""
    D, ld = 520, 2**21 if t == "bf16" else 2**20
    vocab = 2**33 // (ld * DTYPE[t].itemsize)
    print("embedding", vocab, D, ld, t, flush=True)
    table = torch.zeros(vocab * ld, dtype=DTYPE[t], device="cuda:0").view(vocab, ld)
    table[:, :D] = torch.randint(-8, 9, (vocab, D), device="cuda:0", generator=generator(7)).to(DTYPE[t])
    ids = torch.cat([torch.arange(vocab, device="cuda:0"), torch.full((900,), vocab - 1, device="cuda:0")])
    T = len(ids)
    out = torch.zeros((T, D), dtype=DTYPE[t], device="cuda:0")
    d = ozd.embedding_desc(T, vocab, D, t, 64, ldt=ld)
    torch.cuda.synchronize()
    dev.embedding(d, Ptr(table), Ptr(ids), Ptr(out))
    dev.sync()
    assert torch.equal(out, table[:, :D][ids])
    n = dev.embedding_grad_workspace(d)
    work = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda:0")
    want = torch.zeros((vocab, D), device="cuda:0").index_add_(0, ids, out.float()).to(DTYPE[t])
    table[:, :D] = 7.0
    torch.cuda.synchronize()
    dev.embedding_grad(d, Ptr(out), Ptr(ids), Ptr(table), None, Ptr(work), n)
    dev.sync()
    assert torch.equal(table[:, :D], want) and not table[:, D:].any()
