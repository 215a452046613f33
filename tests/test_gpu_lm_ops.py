"""GPU: embedding, residual norm and gradient clipping (csrc/kernels/{embed,resnorm*,gradnorm}.hip) against
fp64, at the sizes, layouts and values where they can go wrong; captured graphs, streams, determinism."""
import math

import pytest
import torch
import torch.nn as nn

import lm_oracle as O
from grace_amd.ops import _native
from grace_amd.ops.embedding import embedding
from grace_amd.ops.norm import residual_norm
from grace_amd.parallel import FusedSGD, clip_grad_norm_, grad_norm
from test_lm_ops import check_clip, grads_like, norm64, norm_case, norm_inputs

pytestmark = pytest.mark.gpu
F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64


def test_native_library():
    assert _native.available()


# ---------------------------------------------------------------------------- embedding
def tokens(n, vocab, how, seed=0):
    g = torch.Generator().manual_seed(seed)
    if how == "same":
        return torch.full((n,), vocab // 2, dtype=torch.int64)
    if how == "falling":
        return (vocab - 1 - torch.arange(n) % vocab).long()
    ids = torch.randint(0, vocab, (n,), generator=g)
    if how == "heavy":  # a third one token, runs over several chunks
        ids[torch.rand(n, generator=g) < 0.33] = vocab - 1
    if how == "outside":
        ids[torch.rand(n, generator=g) < 0.2] = -1
        ids[torch.rand(n, generator=g) < 0.2] = vocab
        ids[:1] = 2**40
    return ids


EMBED = [(n, v, d, how) for n, v, d in [
    (1, 1, 1), (1, 5, 3), (31, 7, 64), (32, 2, 65), (33, 300, 257), (64, 255, 650), (65, 256, 768), (700, 10000, 650),
    (2047, 3, 5), (4097, 30522, 100), (8192, 70000, 9), (8193, 70000, 9), (20001, 257, 33)]
    for how in ("any", "heavy")] + [(3000, 1, 4, "same"), (9000, 17, 300, "same"), (5000, 1000, 12, "falling"),
                                    (777, 50, 40, "outside"), (8500, 600, 40, "outside")]


@pytest.mark.parametrize("n,vocab,d,how", EMBED)
@pytest.mark.parametrize("table,out,index", [(F32, F32, torch.int64), (F32, BF16, torch.int32), (F16, F16, torch.int64),
                                             (BF16, F32, torch.int64)])
def test_embedding(n, vocab, d, how, table, out, index):
    if how == "outside" and index == torch.int32:
        ids = tokens(n, vocab, how).clamp(-2, vocab + 3).to(index).cuda()
    else:
        ids = tokens(n, vocab, how).to(index).cuda()
    g = torch.Generator().manual_seed(1)
    w = torch.randn(vocab, d, generator=g).to(table).cuda().requires_grad_()
    dy = torch.randn(n, d, generator=g).to(out).cuda()
    pad = 0 if vocab > 1 and n % 2 else None
    y = embedding(ids, w, 3.1, pad, out)
    dw, = torch.autograd.grad(y, w, dy)
    assert dw.dtype == table and y.dtype == out
    ry, yb, rdw, dwb = O.embedding(ids, w.detach(), 3.1, pad, dy)
    O.within(y, ry, yb, "y")
    O.within(dw, rdw, dwb, "dw")
    assert torch.equal(dw, torch.autograd.grad(embedding(ids, w, 3.1, pad, out), w, dy)[0])  # every time the same


def test_embedding_is_a_copy_at_scale_one():
    w = torch.randn(50, 33, device="cuda").bfloat16()
    ids = torch.randint(0, 50, (4, 9), device="cuda")
    assert torch.equal(embedding(ids, w), w[ids])


def test_embedding_layouts():
    base = torch.randn(41, 80, device="cuda")
    g = torch.randn(6, 10, 31, device="cuda")
    ids = torch.randint(0, 40, (10, 6), device="cuda").t()
    for w in (base[1:, 7:38], base[:40, :31], torch.randn(31, 40, device="cuda").t(),
              base.reshape(-1)[3:3 + 40 * 31].view(40, 31)):
        w = w.detach().requires_grad_()
        for dy in (g, g.transpose(0, 1).contiguous().transpose(0, 1), g[:1, :1].expand(6, 10, 31)):
            y = embedding(ids, w, 0.5)
            dw, = torch.autograd.grad(y, w, dy)
            ry, yb, rdw, dwb = O.embedding(ids, w.detach(), 0.5, None, dy)
            O.within(y, ry, yb)
            O.within(dw, rdw, dwb)
    y = embedding(ids[:0], w)
    assert y.shape == (0, 10, 31) and not torch.autograd.grad(y, w, g[:0])[0].any()
    assert embedding(ids, torch.empty(40, 0, device="cuda")).shape == (6, 10, 0)
    with pytest.raises(TypeError):
        embedding(ids, w.double())
    with pytest.raises(ValueError):
        embedding(ids.cpu(), w)
    with pytest.raises(ValueError):
        embedding(ids, torch.empty(40, 1, device="cuda").expand(40, 2**21 + 1))


def test_embedding_far_rows():
    """A table of more than 2^31 elements, and its last rows."""
    w = torch.zeros(2**20 + 5, 2100, dtype=BF16, device="cuda")
    ids = torch.tensor([2**20 + 4, 3, 2**20 + 4, 2**20], device="cuda")
    w[ids] = torch.randn(4, 2100, device="cuda").bfloat16()
    w.requires_grad_()
    y = embedding(ids, w)
    assert torch.equal(y, w.detach()[ids])
    dy = torch.randn(4, 2100, device="cuda").bfloat16()
    dw, = torch.autograd.grad(y, w, dy)
    assert torch.equal(dw[2**20 + 4], (dy[0].float() + dy[2].float()).bfloat16())
    assert torch.equal(dw[3], dy[1]) and torch.equal(dw[2**20], dy[3])
    assert int(dw.any(1).sum()) == 3


def test_embedding_many_tokens():
    """More threads than a dimension of a grid takes: 2^26 wave-wide rows and some."""
    n = 2**26 + 77
    w = torch.randn(3, 260, device="cuda").bfloat16()
    ids = torch.arange(n, device="cuda", dtype=torch.int32) % 3
    y = embedding(ids, w)
    for at in (0, 2**25 - 5, 2**26 - 5, n - 60):
        assert torch.equal(y[at:at + 60], w[ids[at:at + 60]])


# ---------------------------------------------------------------------------- residual norm
NORM = [  # batch, length, width, residual, block
    (1, 1, 1, F32, F32), (1, 1, 7, BF16, BF16), (2, 3, 63, F32, F32), (4, 1, 768, BF16, BF16), (35, 21, 651, F16, F16),
    (3, 50, 768, F32, BF16), (2, 3, 1024, F32, F32), (2, 5, 1025, BF16, BF16), (1, 300, 33, F32, F16),
    (2, 9, 4096, BF16, BF16), (3, 3, 4099, F32, F32), (2, 3, 16384, BF16, BF16), (1, 2, 8191, F32, F32),
    (2, 5, 9001, BF16, BF16), (1, 300, 9000, F32, F16), (2, 9, 12000, F32, F32),
    (1100, 2, 20, F32, F32), (7, 900, 12, BF16, BF16), (300, 30, 16, None, BF16), (5, 3, 130, None, F32)]


@pytest.mark.parametrize("b,t,d,tx,ty", NORM)
@pytest.mark.parametrize("kind,gate,post,bias", [
    ("layer", "none", False, True), ("rms", "none", False, False), ("rms", "sample", True, False),
    ("layer", "channel", True, True), ("layer", "full", False, True), ("rms", "channel", False, True),
    ("layer", "none", True, True), ("layer", "sample", False, True)])
def test_residual_norm(b, t, d, tx, ty, kind, gate, post, bias):
    v, dh, ds = norm_inputs(b, t, d, tx, ty, gate, post, bias, "cuda", param=ty if b == 2 else F32)
    norm_case(v, dh, ds, kind, 1.0 if tx is None or b == 4 else 1.5, post)


@pytest.mark.parametrize("gate,post", [("none", False), ("sample", True)])
@pytest.mark.parametrize("which", ["h", "s"])
def test_residual_norm_one_gradient(gate, post, which):
    v, dh, ds = norm_inputs(3, 7, 100, F32, F32, gate, post, True, "cuda")
    norm_case(v, dh if which == "h" else None, ds if which == "s" else None, "layer", 1.0, post)


def test_residual_norm_repeats_and_shares_no_gradient():
    v, dh, _ = norm_inputs(5, 60, 768, F32, F32, "none", False, True, "cuda")
    first = None
    for _ in range(3):
        x, y, w, b = (v[k].clone().requires_grad_() for k in ("x", "y", "weight", "bias"))
        residual_norm(y, x, w, b).backward(dh)
        assert x.grad.data_ptr() != y.grad.data_ptr()
        got = [t.grad for t in (x, y, w, b)]
        assert first is None or all(torch.equal(p, q) for p, q in zip(first, got))
        first = got


def test_residual_norm_layouts():
    v, dh, ds = norm_inputs(6, 10, 40, F32, F32, "none", False, True, "cuda")
    for f in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: torch.cat([t, t], -1)[..., :40],
              lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(6, 10, 40)):
        w = {k: f(t) if t is not None and t.dim() == 3 else t for k, t in v.items()}
        norm_case(w, f(dh), f(ds), "layer", 1.0, False)
    norm_case(v, dh[:1, :1].expand(6, 10, 40), ds, "rms", 1.0, False)


@pytest.mark.parametrize("d", [24, 64, 130, 200, 650, 651, 2050])
def test_residual_norm_16_bit_views(d):
    """Every tensor, weights too, one element behind an aligned address; many gates in a workgroup."""
    v, dh, ds = norm_inputs(70, 3, d, BF16, BF16, "sample", True, True, "cuda", param=BF16)

    def off(t):
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    w = {k: off(t) for k, t in v.items()}
    norm_case(w, off(dh), off(ds), "layer", 1.5, True)
    leaves = {k: t.detach().requires_grad_() for k, t in w.items()}

    def run():
        h, s = residual_norm(leaves["y"], leaves["x"], leaves["weight"], leaves["bias"], gate=leaves["gate"], post=True,
                             post_weight=leaves["post_weight"], post_bias=leaves["post_bias"], return_sum=True)
        return [h, s, *torch.autograd.grad([h, s], list(leaves.values()), [dh, ds])]

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_residual_norm_frozen_parts():
    v, dh, _ = norm_inputs(4, 6, 50, BF16, BF16, "channel", True, True, "cuda")
    for k in ("y", "x", "weight", "gate", "post_bias"):
        t = {n: p.clone() for n, p in v.items()}
        t[k].requires_grad_()
        h = residual_norm(t["y"], t["x"], t["weight"], t["bias"], gate=t["gate"], post=True,
                          post_weight=t["post_weight"], post_bias=t["post_bias"])
        got, = torch.autograd.grad(h, t[k], dh)
        ref = O.residual_norm(v["y"], v["x"], v["weight"], v["bias"], v["gate"], v["post_weight"], v["post_bias"],
                              False, 1e-5, 1.0, True, dh, None)
        O.within(got, *ref["d" + k], k)


def test_residual_norm_special_values():
    y = torch.randn(6, 300, device="cuda")
    x = torch.randn(6, 300, device="cuda")
    y[0, 5], y[1, 7], x[2, 9] = math.inf, math.nan, -math.inf
    y[3], x[3] = 2.0, 1.0  # no deviation
    y[4], x[4] = 0.0, 0.0
    for kind in ("layer", "rms"):
        h, s = residual_norm(y, x, kind=kind, return_sum=True)
        assert h[:3].isnan().any(1).all() and torch.isfinite(h[3:]).all()
        assert torch.isfinite(s[3:]).all()
        if kind == "layer":
            assert not h[3].any()
        assert not h[4].any()
    big = torch.full((2, 64), 1e4, device="cuda") + torch.randn(2, 64, device="cuda")  # the mean is subtracted first
    ref = O.residual_norm(big, None, None, None, None, None, None, False, 1e-5, 1.0, False, None, None)
    O.within(residual_norm(big), *ref["h"])
    with pytest.raises(ValueError):
        residual_norm(torch.zeros(1, 16385, device="cuda"))
    with pytest.raises(TypeError):
        residual_norm(torch.zeros(1, 4, device="cuda", dtype=F64))


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("d", [96, 651, 1100, 4099])
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_of_a_large_constant(d, t, post):
    """mean / deviation overflows fp32, but no value of the row has it: h = 0 and
    dy = r (dh - mean dh), once for each norm, with r = 1 / sqrt(eps)."""
    y = torch.full((3, d), 2.0**110, dtype=t, device="cuda", requires_grad=True)  # the sums over the row are exact
    w = torch.ones(d, device="cuda", requires_grad=True)
    g = torch.Generator("cuda").manual_seed(d)
    dh = torch.randn(3, d, device="cuda", generator=g).to(t)
    h = residual_norm(y, None, w, eps=1e-12, post=post)
    assert not h.any()
    dy, dw = torch.autograd.grad(h, [y, w], dh)
    assert not dw.any()
    r = 1e6 ** (1 + post)
    a = dh.double()
    mass = a.abs() + a.abs().mean(1, keepdim=True)
    O.within(dy, r * (a - a.mean(1, keepdim=True)), 2 * O.K * O.U * r * mass)


@pytest.mark.parametrize("tx,ty", [(F32, F32), (BF16, BF16), (F32, F16)])
def test_residual_norm_empty_batch(tx, ty):
    for gate in ("none", "sample", "full", "channel"):
        v, dh, ds = norm_inputs(0, 3, 20, tx, ty, gate, True, True, "cuda")
        leaves = {k: t.requires_grad_() for k, t in v.items() if t is not None}
        h, s = residual_norm(v["y"], v["x"], v["weight"], v["bias"], gate=v["gate"], post=True,
                             post_weight=v["post_weight"], post_bias=v["post_bias"], return_sum=True)
        assert h.shape == s.shape == (0, 3, 20)
        for g, p in zip(torch.autograd.grad([h, s], list(leaves.values()), [dh, ds]), leaves.values()):
            assert g.shape == p.shape and not g.any()


@pytest.mark.parametrize("weight,bias", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_without_weights(weight, bias, post):
    v, dh, ds = norm_inputs(3, 5, 200, BF16, BF16, "none", post, True, "cuda")
    for on, names in ((weight, ("weight", "post_weight")), (bias, ("bias", "post_bias"))):
        for n in names:
            v[n] = v[n] if on else None
    norm_case(v, dh, ds, "layer", 1.0, post)


def test_residual_norm_of_a_sum_with_itself():
    y = torch.randn(7, 90, device="cuda", requires_grad=True)
    dh = torch.randn(7, 90, device="cuda")
    got, = torch.autograd.grad(residual_norm(y, y), y, dh)
    z = y.detach().requires_grad_()
    a, = torch.autograd.grad(residual_norm(z, y.detach()), z, dh)
    # both ways into the sum carry the same gradient: their fp32 sum is exact
    assert torch.equal(got, a + a)
    y.grad = None
    residual_norm(y, y).backward(dh)
    assert torch.equal(y.grad, a + a)


def test_differentiable_once():
    w = torch.randn(30, 8, device="cuda", requires_grad=True)
    ids = torch.randint(0, 30, (5,), device="cuda")
    for f in (lambda: embedding(ids, w), lambda: residual_norm(w)):
        out = f()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out.sum(), w, create_graph=True)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(w.detach(), torch.ones_like(w))
            with pytest.raises((RuntimeError, NotImplementedError)):
                embedding(ids, dual)
            with pytest.raises((RuntimeError, NotImplementedError)):
                residual_norm(dual)
    y = w.detach().clone().requires_grad_()
    h = residual_norm(y * 1.0, w)
    with torch.no_grad():
        w.add_(1.0)
    got, = torch.autograd.grad(h.sum(), y)  # fp32 keeps the sum, not its parts
    assert torch.isfinite(got).all()
    x = w.detach().bfloat16().requires_grad_()
    z = x * 1.0
    h = residual_norm(z, x)
    with torch.no_grad():
        z.add_(1.0)  # a saved tensor has changed
    with pytest.raises(RuntimeError):
        torch.autograd.grad(h.sum(), x)


def test_residual_norm_far_rows():
    """More than 2^31 elements: the last rows are where they belong."""
    y = torch.zeros(2**20 + 3, 2100, dtype=BF16, device="cuda")
    y[-3:] = torch.randn(3, 2100, device="cuda").bfloat16()
    h = residual_norm(y)
    ref = O.residual_norm(y[-3:], None, None, None, None, None, None, False, 1e-5, 1.0, False, None, None)
    O.within(h[-3:], *ref["h"])
    assert not h[:-3].any()


# ---------------------------------------------------------------------------- clipping
SHAPES = [[(5,)], [(4096,), (4097,), (1,), (0,), (3, 5, 7)], [(100003,), (64, 129)], [(3,)] * 300 + [(9999,)],
          [(70, 1000)] * 7 + [(1,)] * 11]


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("dtypes", [[F32], [BF16, F32, F16], [F16]])
@pytest.mark.parametrize("p,max_norm", [(2.0, 0.5), (2.0, 1e9), (1.0, 3.0), (math.inf, 0.1)])
def test_clip(shapes, dtypes, p, max_norm):
    check_clip(grads_like(shapes, dtypes, "cuda"), max_norm, p)


def test_clip_memory_layouts():
    flat = torch.randn(5000, device="cuda")
    ps = []
    for at, n in ((1, 999), (1000, 1001), (2001, 7), (2008, 2500)):  # views of one bucket, end to end
        p = nn.Parameter(torch.zeros(n, device="cuda"))
        p.grad = flat[at:at + n]
        ps.append(p)
    for g in (torch.randn(8, 4, 5, 5, device="cuda").contiguous(memory_format=torch.channels_last),
              torch.randn(30, 20, device="cuda").t(), torch.randn(30, 40, device="cuda")[:, ::2]):
        p = nn.Parameter(torch.empty_strided(g.shape, g.stride(), device="cuda"))
        p.grad = g
        ps.append(p)
    keep = flat[4508:].clone(), flat[:1].clone()
    check_clip(ps, 0.5)
    assert torch.equal(flat[4508:], keep[0]) and torch.equal(flat[:1], keep[1])  # nothing around them


def test_clip_repeated_and_overlapping():
    p, q = grads_like([(100,), (100,)], [F32], "cuda")
    q.grad = p.grad
    before = p.grad.clone()
    n = clip_grad_norm_([p, q, p], 0.5)  # once
    O.within(p.grad, before.double() * (0.5 / (float(norm64([before], 2)) + 1e-6)), 2 * O.U * before.double().abs())
    assert abs(float(n) - float(norm64([before], 2))) <= 4 * O.U * float(n)
    q.grad = p.grad.view(10, 10).view(-1)  # another view of the same memory: once, too
    assert abs(float(grad_norm([p.grad, q.grad])) - float(norm64([p.grad], 2))) <= 4 * O.U
    flat = torch.randn(150, device="cuda")
    p.grad, q.grad = flat[:100], flat[50:]
    with pytest.raises(RuntimeError):
        clip_grad_norm_([p, q], 0.5)


def test_clip_wide_values():
    ps = grads_like([(1000,), (50,)], [F32], "cuda", scale=1e25)  # squares overflow fp32
    check_clip(ps, 1.0)
    ps = grads_like([(1000,), (50,)], [F32], "cuda", scale=1e-30)  # and underflow
    check_clip(ps, 1.0)
    for bad in (math.inf, math.nan):
        a, b = (grads_like([(5000,), (3,)], [F32], d) for d in ("cpu", "cuda"))
        for p in (a, b):
            p[0].grad[4321] = bad
        assert not torch.isfinite(clip_grad_norm_(b, 1.0))
        clip_grad_norm_(a, 1.0)
        for x, y in zip(a, b):
            torch.testing.assert_close(y.grad.cpu(), x.grad, rtol=0, atol=0, equal_nan=True)
        assert grad_norm([p.grad for p in b], math.inf).isnan()  # inf * 0 and NaN alike are NaN by now
        with pytest.raises(RuntimeError):
            clip_grad_norm_(b, 1.0, error_if_nonfinite=True)


def test_clip_two_devices_and_types():
    ps = grads_like([(100,), (7, 9)], [F32], "cuda") + grads_like([(30,)], [F32], "cpu", seed=1) \
        + grads_like([(20,)], [F64], "cuda", seed=2)
    got = check_clip(ps, 0.5)
    assert got.dtype == F64


def test_clip_long_tensor():
    """More elements than one table entry holds."""
    p = nn.Parameter(torch.empty(2**29 + 4099, dtype=F16, device="cuda"))
    p.grad = torch.zeros_like(p)
    p.grad[-3:] = 2.0
    p.grad[2**29 - 1] = 1.0
    n = clip_grad_norm_([p], 1.0)
    assert abs(float(n) - math.sqrt(13.0)) < 1e-6
    f = 1.0 / (math.sqrt(13.0) + 1e-6)
    O.within(p.grad[-4:], torch.tensor([0.0, 2 * f, 2 * f, 2 * f], device="cuda"), torch.tensor(4 * O.U, device="cuda"))
    O.within(p.grad[2**29 - 1:2**29 + 1], torch.tensor([f, 0.0], device="cuda"), torch.tensor(4 * O.U, device="cuda"))


@pytest.mark.parametrize("kw", [dict(), dict(momentum=0.9, weight_decay=0.01), dict(momentum=0.9, nesterov=True),
                                dict(momentum=0.5, maximize=True)])
@pytest.mark.parametrize("bound", [0.5, 1e9])
def test_clipped_sgd(kw, bound):
    shapes = [(64, 33), (4097,), (3,)] + [(5,)] * 70
    a, b = grads_like(shapes, [F32], "cuda", seed=1), grads_like(shapes, [F32], "cuda", seed=1)
    a = [nn.Parameter(p.detach().double()) for p in a]
    oa, ob = torch.optim.SGD(a, lr=0.1, **kw), FusedSGD(b, lr=0.1, max_grad_norm=bound, **kw)
    norm = norm64([p.grad for p in b], 2)
    f = min(1.0, bound / (float(norm) + 1e-6))
    keep = [p.grad.clone() for p in b]
    for step in range(3):
        for p, k in zip(a, keep):
            p.grad = k.double() * f
        oa.step()
        ob.step()
        assert abs(float(ob.grad_norm) - float(norm)) <= 2 * O.U * float(norm)
        # the weight has moved by at most lr (1 + ... ) times the gradients so far: some 12 roundings a step
        for x, y, k in zip(a, b, keep):
            O.within(y, x.detach(), 12 * O.U * (step + 1) * (x.detach().abs() + 0.1 * 4 * (step + 1) * k.abs() * f))
    assert all(torch.equal(p.grad, k) for p, k in zip(b, keep))


# ---------------------------------------------------------------------------- graphs and streams
def _training_calls(dev="cuda"):
    """Leaves and a function that runs all operators on them, as a step does."""
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 97, (4, 50), generator=g).to(dev)
    table = torch.randn(97, 72, generator=g).to(dev)
    w, b = torch.randn(72, generator=g).to(dev), torch.randn(72, generator=g).to(dev)
    gate = torch.randn(4, 1, 72, generator=g).to(dev)
    dy = torch.randn(4, 50, 72, generator=g).to(dev)

    def run():
        leaves = [t.detach().requires_grad_() for t in (table, w, b, gate)]
        x = embedding(ids, leaves[0], 2.0)
        h, s = residual_norm(x.tanh(), x, leaves[1], leaves[2], gate=leaves[3], post=True, return_sum=True)
        grads = torch.autograd.grad(h + s, leaves, dy)
        params = [nn.Parameter(t.detach()) for t in leaves]
        for p, q in zip(params, grads):
            p.grad = q
        n = clip_grad_norm_(params, 0.7)
        return [h.detach(), s.detach(), n] + [p.grad for p in params]

    return (ids, table, w, b, gate, dy), run


def test_operators_in_a_graph():
    inputs, run = _training_calls()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            run()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):  # two graphs alive together
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graphs.append((graph, outs))
    for k in range(5):
        with torch.no_grad():
            inputs[1].mul_(1.1)
            inputs[5].add_(0.1)
            inputs[0].copy_((inputs[0] + 13 * k) % 97)
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for a, e in zip(outs, want):
                assert torch.equal(a, e)


def test_captured_backward_beside_an_eager_graph():
    """An eager graph on the default stream that holds a leaf: the captured backward is refused, and runs without it."""
    ids = torch.arange(40, device="cuda") % 7
    w = torch.randn(7, 24, device="cuda", requires_grad=True)
    y = torch.randn(40, 24, device="cuda", requires_grad=True)
    dy = torch.randn(40, 24, device="cuda")
    for f, leaf in ((lambda: embedding(ids, w), w), (lambda: residual_norm(y), y)):
        eager = f()
        want, = torch.autograd.grad(eager, leaf, dy, retain_graph=True)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(f(), leaf, dy)
        torch.cuda.synchronize()
        assert torch.equal(torch.autograd.grad(eager, leaf, dy)[0], want)
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(f(), leaf, dy)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_operators_on_another_stream():
    _, run = _training_calls()
    want = [t.clone() for t in run()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for outs in got:
        for a, e in zip(outs, want):
            assert torch.equal(a, e)


def test_wide_rows_in_a_graph():
    """The widest LDS use, and a graph as the first call of its kernels."""
    v, dh, ds = norm_inputs(2, 40, 3000, BF16, BF16, "sample", True, True, "cuda")

    def run():
        t = {k: p.detach().requires_grad_() for k, p in v.items()}
        h, s = residual_norm(t["y"], t["x"], t["weight"], t["bias"], gate=t["gate"], post=True,
                             post_weight=t["post_weight"], post_bias=t["post_bias"], return_sum=True)
        return [h.detach(), s.detach(), *torch.autograd.grad([h, s], list(t.values()), [dh, ds])]

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for _ in range(3):
        with torch.no_grad():
            v["y"].mul_(1.25)
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(outs, want):
            assert torch.equal(a, e)


def test_clipped_sgd_in_a_graph():
    shapes = [(300, 33), (77,)]
    a, b = grads_like(shapes, [F32], "cuda"), grads_like(shapes, [F32], "cuda")
    oa, ob = (FusedSGD(p, lr=0.1, momentum=0.9, max_grad_norm=0.5) for p in (a, b))
    for o in (oa, ob):
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for k in range(4):
        for ps in (a, b):
            for p in ps:
                p.grad.mul_(0.3 if k % 2 else 2.0)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa.grad_norm, ob.grad_norm)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
