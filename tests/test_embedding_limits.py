"""Embedding: tokens and types outside what it takes, on every path, and very many tokens."""
import pytest
import torch

import lm_oracle as O
from grace_amd.ops.embedding import _plain, embedding

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ---------------------------------------------------------------------------- tokens outside the table
def outside_case(device, n=60, rows=7, d=5):
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(-2, rows + 2, (4, n), generator=g)
    ids[0, 0] = 2**40
    w = torch.randn(rows, d, generator=g).to(device).requires_grad_()
    return ids.to(device), w, torch.randn(4, n, d, generator=g).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [None, 3])
def test_tokens_outside_the_table_without_the_kernels(pad, monkeypatch):
    """GRACE_AMD_FORCE_TORCH=1 on a GPU: rows of NaN and no gradient, as the kernels give, and no access behind the
    table."""
    ids, w, dy = outside_case("cuda")
    results = []
    for forced in ("1", "0"):
        monkeypatch.setenv("GRACE_AMD_FORCE_TORCH", forced)
        y = embedding(ids, w, 1.5, pad)
        dw, = torch.autograd.grad(y, w, dy)
        ry, yb, rdw, dwb = O.embedding(ids, w.detach(), 1.5, pad, dy)
        O.within(y, ry, yb, "y")
        O.within(dw, rdw, dwb, "dw")
        results.append((y.isnan(), dw == 0))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("pad", [None, 3])
def test_plain_form_of_tokens_outside_the_table(pad):
    ids, w, dy = outside_case("cpu")
    y = _plain(ids, w, 1.5, pad, F32)
    dw, = torch.autograd.grad(y, w, dy)
    ry, yb, rdw, dwb = O.embedding(ids, w.detach(), 1.5, pad, dy)
    O.within(y, ry, yb, "y")
    O.within(dw, rdw, dwb, "dw")
    with pytest.raises(IndexError):
        embedding(ids, w)


# ---------------------------------------------------------------------------- types
@pytest.mark.parametrize("device", DEVICES)
def test_embedding_refuses_other_types(device):
    ids, w = torch.tensor([1, 0], device=device), torch.ones(3, 4, device=device)
    for table, out in ((w.long(), None), (w.bool(), F32), (w, torch.int32), (w, torch.bool), (w.to(torch.complex64), None)):
        with pytest.raises(TypeError):
            embedding(ids, table, dtype=out)
    if device == "cpu":
        assert embedding(ids, w.double(), 0.5).dtype == F64 and embedding(ids, w, dtype=F64).dtype == F64


# ---------------------------------------------------------------------------- very many tokens
@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,d,out,index", [
    (131073, 70000, 3, F32, torch.int64),    # eight pairs to a thread of the sort, over three passes
    (140001, 300, 481, BF16, torch.int64),   # 128 MB and more of gradients, read past the caches, at odd addresses
    (4300007, 1 << 24, 1, F32, torch.int32),  # counts scanned in a launch of their own, four passes
    (4300007, 257, 5, F16, torch.int64)])
def test_gradient_of_many_tokens(n, vocab, d, out, index):
    g = torch.Generator("cuda").manual_seed(0)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    ids[torch.rand(n, generator=g, device="cuda") < 0.1] = vocab - 1  # a run over many chunks
    ids[::1001] = -1
    ids[n // 2] = vocab
    w = torch.zeros(vocab, d, device="cuda", requires_grad=True)
    flat = torch.randn(n * d + 1, generator=g, device="cuda").to(out)
    dy = flat[1:].view(n, d)  # one element behind an aligned address
    pad = 7
    y = embedding(ids.to(index), w, 1.5, pad, out)
    dw, = torch.autograd.grad(y, w, dy)
    _, _, want, bound = O.embedding(ids.cpu(), w.detach().cpu(), 1.5, pad, dy.cpu())
    O.within(dw.cpu(), want, bound, "dw")
    again, = torch.autograd.grad(embedding(ids.to(index), w, 1.5, pad, out), w, dy)
    assert torch.equal(dw, again)


@pytest.mark.gpu
def test_sorted_gradient_of_far_rows():
    """A gradient of more than 2^31 elements whose tokens are sorted, and its last rows."""
    vocab, d, n = 2**20 + 5, 2100, 3000
    g = torch.Generator("cuda").manual_seed(1)
    rows = torch.tensor([0, 3, 2**20 - 1, 2**20, 2**20 + 4], device="cuda")
    at = torch.randint(0, 5, (n,), generator=g, device="cuda")
    w = torch.zeros(vocab, d, dtype=BF16, device="cuda", requires_grad=True)
    dy = torch.randn(n, d, generator=g, device="cuda").to(BF16)
    dw, = torch.autograd.grad(embedding(rows[at], w), w, dy)
    _, _, want, bound = O.embedding(at, torch.zeros(5, d, device="cuda"), 1.0, None, dy)
    O.within(dw[rows], want, bound, "dw")
    assert int(dw.any(1).sum()) == 5


@pytest.mark.gpu
def test_gradient_of_the_most_tokens():
    """2^31 - 2 tokens: every row's sum of ones is a whole number below 2^24, which fp32 holds in any order."""
    n, vocab = 2**31 - 2, 300
    ids = torch.arange(n, device="cuda", dtype=torch.int32).remainder_(vocab)
    w = torch.zeros(vocab, 1, device="cuda", requires_grad=True)
    y = embedding(ids, w, dtype=F16)
    dw, = torch.autograd.grad(y, w, torch.ones(n, 1, dtype=F16, device="cuda"))
    want = n // vocab + (torch.arange(vocab, device="cuda") < n % vocab).long()
    assert torch.equal(dw[:, 0].double(), want.double())
