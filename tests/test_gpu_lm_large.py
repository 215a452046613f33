"""GPU: the forms that residual norms and the clipped SGD update take by their size: nontemporal accesses, more than 2^31
elements."""
import pytest
import torch
import torch.nn as nn

import lm_oracle as O
from grace_amd.ops.norm import residual_norm
from grace_amd.parallel import FusedSGD
from test_lm_ops import norm64

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def values(*shape, dtype=F32, mean=0.0, scale=1.0, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(mean).to(dtype)


@pytest.mark.parametrize("rows,d,tx,ty", [
    (33600, 1000, F32, F32), (65538, 1024, BF16, BF16), (270000, 256, F16, F16), (8200, 8192, BF16, BF16),
    (44745, 1000, F32, BF16), (5600, 12000, BF16, BF16)])
@pytest.mark.parametrize("gate,post", [(False, False), (True, True)])
def test_backward_that_stores_past_the_caches(rows, d, tx, ty, gate, post):
    size = {F32: 4, BF16: 2, F16: 2}
    assert rows * d * (size[tx] + size[ty]) * 2 > 512 << 20
    v = dict(y=values(rows, d, dtype=ty), x=values(rows, d, dtype=tx, mean=0.3, seed=1),
             weight=values(d, mean=1.0, scale=0.2, seed=2), bias=values(d, scale=0.2, seed=3))
    v["gate"] = values(d, dtype=ty, mean=0.7, scale=0.4, seed=4) if gate else None
    v["post_weight"] = values(d, mean=1.0, scale=0.2, seed=5) if post else None
    v["post_bias"] = values(d, scale=0.2, seed=6) if post else None
    dh, ds = torch.randint(-4, 5, (rows, d), device="cuda").to(ty), values(rows, d, dtype=tx, seed=8)
    leaves = {k: t.requires_grad_() for k, t in v.items() if t is not None}
    h, s = residual_norm(v["y"], v["x"], v["weight"], v["bias"], gate=v["gate"], alpha=1.5, post=post,
                         post_weight=v["post_weight"], post_bias=v["post_bias"], return_sum=True)
    got = dict(zip(leaves, torch.autograd.grad([h, s], list(leaves.values()), [dh, ds])))
    plain = {k: None if t is None else t.detach() for k, t in v.items()}
    # row by row; the sums over rows below.  16-bit sums are made again, so the bound is that of fp32 values
    some = torch.cat([torch.arange(0, 40), torch.arange(rows // 2, rows // 2 + 40), torch.arange(rows - 40, rows)]).cuda()

    def oracle(at):
        rest = [None if plain[k] is None else plain[k].float() for k in ("weight", "bias", "gate", "post_weight", "post_bias")]
        return O.residual_norm(plain["y"][at].float(), plain["x"][at].float(), *rest, False, 1e-5, 1.5, post,
                               dh[at].float(), ds[at].float())

    want = oracle(some)
    for k, t in (("h", h), ("s", s), ("dx", got["x"]), ("dy", got["y"])):
        O.within(t[some], *want[k], k)
    total = {}
    for part in torch.arange(rows, device="cuda").split(8192):  # sums of sums: no more roundings than serial ones
        for k, (value, bound) in oracle(part).items():
            if k in ("h", "s", "dx", "dy"):
                continue
            a, b = total.get(k, (0.0, 0.0))
            total[k] = a + value, b + bound
    for k, (value, bound) in total.items():
        O.within(got[k[1:]], value, bound, k)
    # those bounds are too wide to show a row left out; sums of whole numbers below 2^24 are exact in any order
    assert torch.equal(got["bias"].double(), total["dbias"][0])


def test_backward_of_far_rows():
    """More than 2^31 elements: the last rows' gradients, and sums that only they take part in."""
    rows, d = 2**20 + 3, 2100
    y = torch.zeros(rows, d, dtype=BF16, device="cuda")
    y[-3:] = values(3, d, dtype=BF16)
    dh = torch.zeros(rows, d, dtype=BF16, device="cuda")
    dh[-3:] = values(3, d, dtype=BF16, seed=1)
    w = values(d, mean=1.0, scale=0.2, seed=2).requires_grad_()
    y.requires_grad_()
    dy, dw = torch.autograd.grad(residual_norm(y, None, w), [y, w], dh)
    want = O.residual_norm(y.detach()[-3:], None, w.detach(), None, None, None, None, False, 1e-5, 1.0, False, dh[-3:], None)
    O.within(dy[-3:], *want["dy"])
    assert not dy[:-3].any()
    O.within(dw, *want["dweight"])


@pytest.mark.parametrize("kw", [dict(momentum=0.9, weight_decay=0.01), dict(momentum=0.9, nesterov=True), dict()])
@pytest.mark.parametrize("bound", [0.5, 1e9])
def test_clipped_update_past_the_caches(kw, bound):
    sizes = [22500003, 4099, 5, 12000002] if kw else [33600001, 4099, 5, 7]
    assert sum(sizes) * 4 * (3 if kw else 2) > 256 << 20
    flat, grads = values(sum(sizes) + 3, scale=0.05), values(sum(sizes) + 3, scale=0.01, seed=1)
    ps, at = [], 3  # views at odd places: in the first neither vector accesses nor whole ones
    for n in sizes:
        p = nn.Parameter(flat[at:at + n])
        p.grad = grads[at:at + n]
        ps.append(p)
        at += n
    aligned = nn.Parameter(values(10000001, scale=0.05, seed=2))
    aligned.grad = values(10000001, scale=0.01, seed=3)
    ps.append(aligned)
    edge = flat[:3].clone()
    opt = FusedSGD(ps, lr=0.1, max_grad_norm=bound, **kw)
    norm = norm64([p.grad for p in ps], 2)
    f = min(1.0, bound / (float(norm) + 1e-6))
    ref = [nn.Parameter(p.detach().double()) for p in ps]
    wide = torch.optim.SGD(ref, lr=0.1, **kw)
    for step in range(2):
        for r, p in zip(ref, ps):  # anew: torch's nesterov step adds the momentum to the gradients in place
            r.grad = p.grad.double() * f
        opt.step()
        wide.step()
        assert abs(float(opt.grad_norm) - float(norm)) <= 2 * O.U * float(norm)
        # as for small tensors: some 12 roundings a step of the weight and of what it has moved by
        for p, r in zip(ps, ref):
            O.within(p, r.detach(), 12 * O.U * (step + 1) * (r.detach().abs() + 0.4 * (step + 1) * p.grad.abs() * f))
    assert torch.equal(flat[:3], edge)


def test_the_most_rows():
    """2^31 - 2 rows of one value.  The rms norm of +-1 with eps = 0 is +-1 in fp32, so with weight 2 and bias 1 h is 3 or
    -1, and dweight and dbias are whole numbers."""
    n = 2**31 - 2
    y = torch.ones(n, 1, dtype=BF16, device="cuda")
    y[1::2] = -1.0
    w = torch.full((1,), 2.0, device="cuda", requires_grad=True)
    b = torch.full((1,), 1.0, device="cuda", requires_grad=True)
    h = residual_norm(y, None, w, b, kind="rms", eps=0.0)
    assert bool((h.view(-1, 2) == torch.tensor([3.0, -1.0], dtype=BF16, device="cuda")).all())
    dh = torch.zeros(n, 1, dtype=BF16, device="cuda")
    dh[::2], dh[-3:] = 1.0, 4.0
    dw, db = torch.autograd.grad(h, [w, b], dh)
    # the last three rows have 4 each, two of them with y = -1; sums of whole numbers, each rounded at most 40 times
    ones = n // 2 - 1
    assert abs(float(db) - (ones + 12)) <= 40 * O.U * (ones + 12)
    assert abs(float(dw) - (ones + 4 - 8)) <= 40 * O.U * (ones + 12)
    # and with whole numbers below 2^24 exactly
    dh.zero_()
    dh[::1024], dh[-3:] = 1.0, 4.0
    dw, db = torch.autograd.grad(residual_norm(y, None, w, b, kind="rms", eps=0.0), [w, b], dh)
    assert float(db) == n // 1024 + 1 + 12 and float(dw) == n // 1024 + 1 + 4 - 8
