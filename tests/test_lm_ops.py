"""Embedding, residual norm and gradient clipping on the CPU: values and gradients against fp64, and every
refusal (the arguments are checked before the device is looked at, so these hold on a GPU too)."""
import math

import pytest
import torch
import torch.nn as nn

from grace_amd.ops.embedding import ScaledEmbedding, embedding
from grace_amd.ops.norm import ResidualNorm, residual_norm
from grace_amd.parallel import FusedSGD, clip_grad_norm_, grad_norm

import lm_oracle as O

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]  # a GPU's refusals come from the host too


# ---------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("table,out", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("pad", [None, 0, -1])
def test_embedding_cpu(table, out, pad):
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 11, (3, 7), generator=g)
    w = torch.randn(11, 5, generator=g).to(table).requires_grad_()
    dy = torch.randn(3, 7, 5, generator=g).to(out)
    y = embedding(ids, w, 1.7, pad, out)
    assert y.dtype == out
    dw, = torch.autograd.grad(y, w, dy)
    ry, yb, rdw, dwb = O.embedding(ids, w.detach(), 1.7, None if pad is None else pad % 11, dy)
    O.within(y, ry, yb, "y")
    O.within(dw, rdw, dwb, "dw")


def test_embedding_gradcheck_and_module():
    w = torch.randn(6, 3, dtype=F64, requires_grad=True)
    ids = torch.tensor([[0, 5], [5, 2]])
    # row 4 is padding and unused: a used one has a zero gradient by definition, which differences do not see
    assert torch.autograd.gradcheck(lambda v: embedding(ids, v, 0.3, 4), (w,))
    a, b = nn.Embedding(6, 3, padding_idx=1), ScaledEmbedding(6, 3, padding_idx=1, scale=2.0)
    b.load_state_dict(a.state_dict())
    torch.testing.assert_close(b(ids), a(ids) * 2, rtol=0, atol=0)


@pytest.mark.parametrize("device", DEVICES)
def test_embedding_refusals(device):
    w, ids = torch.randn(4, 3, device=device), torch.tensor([1, 2], device=device)
    for bad in (ids.float(), ids.to(torch.int16), ids.bool()):
        with pytest.raises(TypeError):
            embedding(bad, w)
    with pytest.raises(ValueError):
        embedding(ids, w[0])
    with pytest.raises(ValueError):
        embedding(ids, torch.empty(0, 3, device=device))
    for pad in (4, -5):
        with pytest.raises(ValueError):
            embedding(ids, w, padding_idx=pad)
    if device == "cpu":
        with pytest.raises(IndexError):
            embedding(torch.tensor([4]), w)
    for kw in (dict(max_norm=1.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        with pytest.raises(ValueError):
            ScaledEmbedding(4, 3, **kw)
    assert embedding(ids.new_empty(0, 2), w).shape == (0, 2, 3)


# ---------------------------------------------------------------------------- residual norm
GATES = {"none": None, "channel": lambda b, t, d: (d,), "sample": lambda b, t, d: (b, 1, d),
         "full": lambda b, t, d: (b, t, d)}


def norm_inputs(b, t, d, tx, ty, gate, post, bias, device="cpu", param=F32, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*shape, dtype=F32, mean=0.0, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale + mean).to(dtype).to(device)

    v = dict(y=r(b, t, d, dtype=ty), x=None if tx is None else r(b, t, d, dtype=tx, mean=0.3),
             weight=r(d, dtype=param, mean=1.0, scale=0.2), bias=r(d, dtype=param, scale=0.2) if bias else None,
             gate=None if GATES[gate] is None else r(*GATES[gate](b, t, d), dtype=ty, mean=0.7, scale=0.4),
             post_weight=r(d, dtype=param, mean=1.0, scale=0.2) if post else None,
             post_bias=r(d, dtype=param, scale=0.2) if post and bias else None)
    return v, r(b, t, d, dtype=ty), r(b, t, d, dtype=ty if tx is None else tx)


def norm_case(v, dh, ds, kind, alpha, post, eps=1e-5):
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    h, s = residual_norm(leaves["y"], leaves.get("x"), leaves.get("weight"), leaves.get("bias"), kind=kind, eps=eps,
                         gate=leaves.get("gate"), alpha=alpha, post=post, post_weight=leaves.get("post_weight"),
                         post_bias=leaves.get("post_bias"), return_sum=True)
    outs = [(o, d) for o, d in ((h, dh), (s, ds)) if d is not None]
    grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [d for _, d in outs], allow_unused=True)
    ref = O.residual_norm(v["y"], v["x"], v["weight"], v["bias"], v["gate"], v["post_weight"], v["post_bias"],
                          kind == "rms", eps, alpha, post, dh, ds)
    assert h.dtype == v["y"].dtype and s.dtype == (v["y"] if v["x"] is None else v["x"]).dtype
    got = {"h": h, "s": s, **{"d" + k: g for k, g in zip(leaves, grads)}}
    for k, (value, bound) in ref.items():
        if got[k] is None:  # no path from the outputs that have a gradient
            assert not value.abs().max() > 0, k
            continue
        if k[0] == "d":
            assert got[k].dtype == leaves[k[1:]].dtype
        O.within(got[k], value, bound, k)
    return got


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("tx,ty", [(F32, F32), (None, F32), (BF16, BF16), (F32, F16)])
def test_residual_norm_cpu(kind, gate, post, tx, ty):
    v, dh, ds = norm_inputs(3, 5, 9, tx, ty, gate, post, True)
    norm_case(v, dh, ds, kind, 1.0 if tx is None else 1.5, post)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_residual_norm_gradcheck(kind):
    v, _, _ = norm_inputs(2, 3, 5, F64, F64, "sample", True, True, param=F64)
    v = {k: t.requires_grad_() for k, t in v.items()}

    def f(y, x, w, b, g, pw, pb):
        return residual_norm(y, x, w, b, kind=kind, gate=g, alpha=0.7, post=True, post_weight=pw, post_bias=pb,
                             return_sum=True)

    assert torch.autograd.gradcheck(f, [v[k] for k in ("y", "x", "weight", "bias", "gate", "post_weight", "post_bias")])


def test_residual_norm_module_loads_layer_norm():
    a, b = nn.LayerNorm(12), ResidualNorm(12)
    with torch.no_grad():
        a.weight.normal_()
        a.bias.normal_()
    b.load_state_dict(a.state_dict())
    x, y = torch.randn(4, 12), torch.randn(4, 12)
    torch.testing.assert_close(b(y, x), a(x + y), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(b(y), a(y), rtol=1e-5, atol=1e-5)
    h, s = b(y, return_sum=True)
    assert s is y
    assert ResidualNorm(12, bias=False, post=True).post_bias is None


@pytest.mark.parametrize("device", DEVICES)
def test_residual_norm_refusals(device):
    def ones(*shape):
        return torch.ones(shape, device=device)

    y, x, w = ones(2, 3, 4), ones(2, 3, 4), ones(4)
    for bad in (ones(3), ones(3, 4), ones(1, 3, 4), ones(2, 3, 1), ones(2, 1, 1, 4), ones()):
        with pytest.raises(ValueError):
            residual_norm(y, x, w, gate=bad)
    for kw in (dict(kind="batch"), dict(post_weight=w), dict(post_bias=w)):
        with pytest.raises(ValueError):
            residual_norm(y, x, w, **kw)
    with pytest.raises(ValueError):
        residual_norm(y, None, w, alpha=2.0)
    with pytest.raises(ValueError):
        residual_norm(y, x[:1], w)
    with pytest.raises(ValueError):
        residual_norm(y, x, ones(5))
    with pytest.raises(ValueError):
        residual_norm(y, x, w, ones(1, 4))
    with pytest.raises(ValueError):
        residual_norm(ones())
    with pytest.raises(TypeError):
        residual_norm(y, x.bfloat16(), w)
    with pytest.raises(TypeError):
        residual_norm(y.bfloat16(), x.half(), w)
    with pytest.raises(TypeError):
        residual_norm(y.bfloat16(), x, w.half())
    with pytest.raises(TypeError):
        residual_norm(y.long())
    with pytest.raises(ValueError):
        ResidualNorm(4, kind="batch")
    h, s = residual_norm(y[:0], x[:0], w, return_sum=True)
    assert h.shape == s.shape == (0, 3, 4)


# ---------------------------------------------------------------------------- clipping
def grads_like(shapes, dtypes, device="cpu", seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    ps = []
    for i, s in enumerate(shapes):
        t = dtypes[i % len(dtypes)]
        p = nn.Parameter(torch.zeros(s, dtype=t, device=device))
        p.grad = (torch.randn(s, generator=g) * scale).to(t).to(device)
        ps.append(p)
    return ps


def norm64(grads, p):
    flat = torch.cat([g.detach().double().reshape(-1).cpu() for g in grads])
    return flat.abs().max() if p == math.inf else flat.abs().sum() if p == 1 else flat.square().sum().sqrt()


def check_clip(ps, max_norm, p=2.0, **kw):
    before = [q.grad.clone() for q in ps]
    want = norm64(before, p)
    got = clip_grad_norm_(ps, max_norm, p, **kw)
    assert got.dim() == 0
    # the norm is summed in fp64 and rounded once; one more rounding of slack for the square root
    assert abs(got.double().cpu() - want) <= 2 * O.U * want + 1e-300
    factor = min(1.0, max_norm / (float(want) + 1e-6))
    for q, b in zip(ps, before):
        if factor == 1.0:
            assert torch.equal(q.grad, b)
        else:  # the factor to fp32, and the product
            O.within(q.grad, b.double() * factor, 2 * O.U * b.double().abs() * factor, "gradient")
    return got


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clip_cpu(p, max_norm):
    check_clip(grads_like([(3, 4), (7,), (0,), (), (2, 3, 5)], [F32, BF16, F32]), max_norm, p)


def test_clip_matches_torch_and_shared_parameters():
    a, b = grads_like([(5, 5), (9,)], [F32]), grads_like([(5, 5), (9,)], [F32])
    na, nb = torch.nn.utils.clip_grad_norm_(a, 0.7), clip_grad_norm_(b + b[:1], 0.7)  # a shared one once
    torch.testing.assert_close(nb, na, rtol=1e-6, atol=0)
    for x, y in zip(a, b):
        torch.testing.assert_close(y.grad, x.grad, rtol=1e-6, atol=0)
    one = grads_like([(3,)], [F64])
    assert clip_grad_norm_(one[0], 1.0).dtype == F64
    assert clip_grad_norm_([], 1.0) == 0 and clip_grad_norm_([nn.Parameter(torch.ones(2))], 1.0) == 0
    assert grad_norm([]) == 0
    assert abs(float(grad_norm(torch.full((4,), 2.0))) - 4) < 1e-6


def test_clip_nonfinite():
    for bad in (math.inf, math.nan):
        a, b = grads_like([(4,), (3,)], [F32]), grads_like([(4,), (3,)], [F32])
        for ps in (a, b):
            ps[0].grad[1] = bad
        torch.nn.utils.clip_grad_norm_(a, 1.0)
        keep = [p.grad.clone() for p in b]
        with pytest.raises(RuntimeError):
            clip_grad_norm_(b, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(p.grad, k) or k.isnan().any() for p, k in zip(b, keep))
        clip_grad_norm_(b, 1.0)
        for x, y in zip(a, b):
            torch.testing.assert_close(y.grad, x.grad, rtol=0, atol=0, equal_nan=True)


def test_clip_refusals():
    ps = grads_like([(4,)], [F32])
    for p in (0.0, 3.0, -math.inf):
        with pytest.raises(ValueError):
            clip_grad_norm_(ps, 1.0, p)
    for bound in (-1.0, math.nan):
        with pytest.raises(ValueError):
            clip_grad_norm_(ps, bound)
    q = nn.Parameter(torch.zeros(3, 4))
    q.grad = torch.ones(1, 4).expand(3, 4)
    with pytest.raises(ValueError):
        clip_grad_norm_([q], 1.0)
    with pytest.raises(TypeError):
        grad_norm([torch.ones(3, dtype=torch.int64)])
    with pytest.raises(TypeError):
        grad_norm([torch.ones(3, 3).to_sparse()])
    with pytest.raises(ValueError):
        FusedSGD(ps, lr=0.1, max_grad_norm=-1.0)
    with pytest.raises(ValueError):
        FusedSGD(ps, lr=0.1, max_grad_norm=math.nan)


@pytest.mark.parametrize("kw", [dict(), dict(momentum=0.9, weight_decay=0.01), dict(momentum=0.9, nesterov=True)])
def test_clipped_sgd_cpu(kw):
    a, b = grads_like([(5, 7), (11,)], [F32], seed=1), grads_like([(5, 7), (11,)], [F32], seed=1)
    oa, ob = torch.optim.SGD(a, lr=0.1, **kw), FusedSGD(b, lr=0.1, max_grad_norm=0.5, **kw)
    keep = [p.grad.clone() for p in b]
    for _ in range(3):
        for p, k in zip(a, keep):
            p.grad = k.clone()
        n = torch.nn.utils.clip_grad_norm_(a, 0.5)
        oa.step()
        ob.step()
        torch.testing.assert_close(ob.grad_norm, n, rtol=1e-6, atol=0)
    for x, y, k in zip(a, b, keep):
        torch.testing.assert_close(y, x, rtol=1e-6, atol=1e-7)
        assert torch.equal(y.grad, k)
    ref = torch.optim.SGD(a, lr=0.1, **kw)
    ref.load_state_dict(ob.state_dict())
