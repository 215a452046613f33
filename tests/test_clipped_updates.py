"""Clipping inside the SGD update and over views: 16-bit parameters, copies, pickles and state dicts of the optimizer,
steps without gradients, gradients that share memory."""
import copy
import math
import pickle

import pytest
import torch
import torch.nn as nn

import lm_oracle as O
from grace_amd.parallel import FusedSGD, clip_grad_norm_, grad_norm

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def parameter(grad):
    p = nn.Parameter(torch.zeros_like(grad))
    p.grad = grad
    return p


# ---------------------------------------------------------------------------- 16-bit parameters
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("t", [BF16, F16])
def test_the_factor_keeps_its_bits(t, device):
    """A step of lr 1 from zero is the clipped gradient with its sign turned: one rounding to the weights' type, and the
    roundings of the fp32 factor and of the fp32 product before it."""
    g = torch.Generator().manual_seed(0)
    for n, bound in ((1000, 1.0), (4097, 0.37), (3, 0.01)):
        p = parameter(torch.randn(n, generator=g).to(t).to(device))
        opt = FusedSGD([p], lr=1.0, max_grad_norm=bound)
        opt.step()
        grad = p.grad.double()
        want = -grad * (bound / (grad.norm() + 1e-6))
        O.within(p, want, 3 * O.U * want.abs(), f"{t} {n}")


# ---------------------------------------------------------------------------- copies, pickles, state dicts
def stepped(opt, grads):
    """The weights after a step with these gradients."""
    params = [p for group in opt.param_groups for p in group["params"]]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    opt.step()
    return [p.detach().clone() for p in params]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("how", ["copy", "pickle"])
@pytest.mark.parametrize("bound", [0.25, None])
def test_a_copy_clips_as_its_original(how, bound, device):
    grads = [torch.full((5,), 2.0, device=device), torch.full((3, 2), -1.0, device=device)]
    opt = FusedSGD([parameter(g) for g in grads], lr=0.5, momentum=0.9, max_grad_norm=bound)
    stepped(opt, grads)
    other = copy.deepcopy(opt) if how == "copy" else pickle.loads(pickle.dumps(opt))
    assert other.max_grad_norm == bound
    for a, b in zip(stepped(opt, grads), stepped(other, grads)):
        assert torch.equal(a, b)


def test_state_dicts_hold_the_bound():
    grads = [torch.full((5,), 2.0)]

    def made(cls=FusedSGD, **kw):
        return cls([parameter(g) for g in grads], lr=0.5, momentum=0.9, **kw)

    opt = made(max_grad_norm=0.25)
    stepped(opt, grads)
    plain = made()
    plain.load_state_dict(opt.state_dict())
    assert plain.max_grad_norm == 0.25
    opt.load_state_dict(made(max_grad_norm=0.5).state_dict())
    assert opt.max_grad_norm == 0.5
    # torch's optimizer loads it, and its state dict, which has no bound, leaves the one that there is
    ref = made(torch.optim.SGD)
    ref.load_state_dict(opt.state_dict())
    opt.load_state_dict(made(torch.optim.SGD).state_dict())
    assert opt.max_grad_norm == 0.5
    opt.load_state_dict(made().state_dict())
    assert opt.max_grad_norm is None


def test_one_bound_for_all_groups():
    a, b, c = (parameter(torch.full((4,), 3.0)) for _ in range(3))
    opt = FusedSGD([{"params": [a]}, {"params": [b], "lr": 0.1}], lr=1.0, max_grad_norm=1.0)
    opt.add_param_group({"params": [c]})
    opt.step()
    assert abs(float(opt.grad_norm) - 108 ** 0.5) < 1e-5
    opt.max_grad_norm = 2.0
    assert opt.max_grad_norm == 2.0 and all(group["max_grad_norm"] == 2.0 for group in opt.param_groups)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            opt.max_grad_norm = bad
    assert opt.max_grad_norm == 2.0
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [parameter(torch.ones(2))], "max_grad_norm": 1.0})
    with pytest.raises(ValueError):
        FusedSGD([{"params": [a], "max_grad_norm": 1.0}, {"params": [b]}], lr=1.0)
    state = opt.state_dict()
    state["param_groups"][1]["max_grad_norm"] = 1.0
    with pytest.raises(ValueError):
        opt.load_state_dict(state)
    assert opt.max_grad_norm == 2.0


# ---------------------------------------------------------------------------- steps without gradients
@pytest.mark.parametrize("device", DEVICES)
def test_the_norm_is_the_last_steps(device):
    p = parameter(torch.ones(3, device=device))
    opt = FusedSGD([p], lr=0.1, max_grad_norm=1.0)
    opt.step()
    assert abs(float(opt.grad_norm) - 3 ** 0.5) < 1e-6
    opt.zero_grad(set_to_none=True)
    before = p.detach().clone()
    opt.step()
    assert opt.grad_norm.shape == () and opt.grad_norm.device == p.device and float(opt.grad_norm) == 0.0
    assert torch.equal(p, before)
    p.grad = torch.full((3,), 2.0, device=device)
    opt.step()
    assert abs(float(opt.grad_norm) - 12 ** 0.5) < 1e-6
    opt.max_grad_norm = None  # an unclipped step takes no norm
    opt.step()
    assert opt.grad_norm is None


def test_a_step_without_parameters():
    opt = FusedSGD([{"params": []}], lr=0.1, max_grad_norm=1.0)
    opt.step()
    assert float(opt.grad_norm) == 0.0
    p = parameter(torch.full((4,), 2.0))
    opt.add_param_group({"params": [p]})
    opt.step()
    assert float(opt.grad_norm) == 4.0
    want = torch.full((4,), -0.1 * 2.0 / (4.0 + 1e-6), dtype=F64)
    O.within(p, want, 8 * O.U * want.abs())  # lr, factor and two products


# ---------------------------------------------------------------------------- gradients that share memory
VIEWS = {"the same": lambda g: g, "a view": lambda g: g.view(2, 2).view(4), "a part of its storage": lambda g: g[:],
         "a permuted one": lambda g: g.view(2, 2).t()}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("raises", [False, True])  # two ways through the host code
@pytest.mark.parametrize("view", list(VIEWS))
def test_views_of_one_gradient_count_once(view, raises, device):
    a, b = parameter(torch.ones(4, device=device)), nn.Parameter(torch.zeros(4, device=device))
    grad = VIEWS[view](a.grad)
    b = nn.Parameter(torch.zeros_like(grad))
    b.grad = grad
    assert float(grad_norm([a.grad, grad])) == 2.0
    assert float(clip_grad_norm_([a, b], 1.0, error_if_nonfinite=raises)) == 2.0
    want = torch.full((4,), 1.0 / (2.0 + 1e-6), dtype=F64, device=device)
    O.within(a.grad, want, 2 * O.U * want)
    opt = FusedSGD([a, b], lr=0.1, max_grad_norm=1e9)
    opt.step()
    assert abs(float(opt.grad_norm) - 1.0) <= 1e-6  # 2 x the factor, 1 / (2 + 1e-6)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("raises", [False, True])
def test_views_with_gaps_count_once(raises, device):
    m = torch.ones(3, 8, device=device)
    ps = [nn.Parameter(torch.empty_strided((3, 4), (8, 2), device=device)) for _ in range(3)]
    ps[0].grad, ps[1].grad, ps[2].grad = m[:, ::2], m.view(3, 4, 2)[..., 0], m[:, 1::2]  # the third lies between
    assert abs(float(clip_grad_norm_(ps, 1.0, error_if_nonfinite=raises)) - 24 ** 0.5) <= 2e-6
    want = torch.full((3, 8), 1.0 / (24 ** 0.5 + 1e-6), dtype=F64, device=device)
    O.within(m, want, 3 * O.U * want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("raises", [False, True])
def test_overlapping_gradients_are_refused(raises, device):
    flat = torch.ones(150, device=device)
    ps = [nn.Parameter(torch.zeros(100, device=device)) for _ in range(2)]
    ps[0].grad, ps[1].grad = flat[:100], flat[50:]
    for call in (lambda: grad_norm([p.grad for p in ps]), lambda: clip_grad_norm_(ps, 1.0, error_if_nonfinite=raises),
                 lambda: FusedSGD(ps, lr=0.1, max_grad_norm=1.0).step()):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    assert torch.equal(flat, torch.ones_like(flat))
    other = nn.Parameter(torch.zeros(100, dtype=BF16, device=device))
    other.grad = flat.view(BF16)[20:120]  # another type over the first's bytes
    wide = nn.Parameter(torch.zeros(3, 50, device=device))
    wide.grad = flat.view(3, 50)
    gaps = nn.Parameter(torch.empty_strided((3, 10), (50, 1), device=device))
    gaps.grad = wide.grad[:, 5:15]
    for pair in ([ps[0], other], [wide, gaps], [gaps, wide]):
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grad_norm_(pair, 1.0, error_if_nonfinite=raises)
    assert torch.equal(flat, torch.ones_like(flat))


# ---------------------------------------------------------------------------- the wrapped optimizer
def test_the_bound_through_the_distributed_optimizer():
    from grace_amd import grace_from_params
    from grace_amd.parallel import DistributedOptimizer

    def wrapped(cls, **kw):
        p = nn.Parameter(torch.zeros(4))
        opt = DistributedOptimizer(cls([p], lr=1.0, **kw), grace_from_params(
            {"compressor": "none", "memory": "none", "communicator": "allreduce", "world_size": 1}))
        (p * torch.full((4,), 2.0)).sum().backward()
        return p, opt

    p, opt = wrapped(FusedSGD, max_grad_norm=8.0)
    assert opt.max_grad_norm == 8.0
    opt.max_grad_norm = 1.0
    opt.step()
    want = torch.full((4,), -2.0 / (4.0 + 1e-6), dtype=F64)
    O.within(p, want, 4 * O.U * want.abs())
    _, plain = wrapped(torch.optim.SGD)
    for call in (lambda: plain.max_grad_norm, lambda: setattr(plain, "max_grad_norm", 1.0)):
        with pytest.raises(AttributeError):
            call()
