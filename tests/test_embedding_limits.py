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
