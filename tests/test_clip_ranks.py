"""Clipping by the norm of the exchanged gradients on CPU ranks (gloo, W = 2): the same norm and the same weights on every
rank, inside the update, as a call of its own, and with bf16 working copies."""
import os
import sys

import pytest
import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(__file__))
from dist_utils import run_distributed  # noqa: E402

BOUND, STEPS = 0.05, 3


def _net():
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(7, 9), nn.Tanh(), nn.Linear(9, 3))


def _data(rank):
    g = torch.Generator().manual_seed(10 + rank)
    return torch.randn(5, 7, generator=g), torch.randn(5, 3, generator=g)


def _reference(world):
    """(norms, weights) in fp64: the mean gradient over ranks, torch's clipping and SGD."""
    net = _net().double()
    opt = torch.optim.SGD(net.parameters(), lr=0.5, momentum=0.9)
    norms = []
    for _ in range(STEPS):
        opt.zero_grad()
        for rank in range(world):
            x, y = (t.double() for t in _data(rank))
            ((net(x) - y).square().mean() / world).backward()
        norms.append(float(torch.nn.utils.clip_grad_norm_(net.parameters(), BOUND)))
        opt.step()
    return norms, [p.detach() for p in net.parameters()]


def _body(rank, world, inside, working):
    import torch.distributed as dist

    from grace_amd import grace_from_params
    from grace_amd.parallel import DistributedOptimizer, FusedSGD, clip_grad_norm_
    from grace_amd.parallel.precision import BF16Weights

    net = _net()
    weights = BF16Weights(net) if working else None
    named = list(weights.named_master_parameters(net) if working else net.named_parameters())
    params = [p for _, p in named]
    opt = DistributedOptimizer(FusedSGD(params, lr=0.5, momentum=0.9, max_grad_norm=BOUND if inside else None),
                               grace_from_params({"compressor": "none", "memory": "none", "communicator": "allreduce",
                                                  "world_size": world}), named_parameters=named, weights=weights)
    x, y = _data(rank)
    norms = []
    for _ in range(STEPS):
        opt.zero_grad()
        with torch.autocast("cpu", dtype=torch.bfloat16, enabled=working):
            out = net(x)
        (out.float() - y).square().mean().backward()
        if inside:
            opt.step()
            norms.append(float(opt.grad_norm))
        else:
            opt.synchronize()
            norms.append(float(clip_grad_norm_(params, BOUND)))
            with opt.skip_synchronize():
                opt.step()
    mine = torch.cat([torch.tensor(norms), *(p.detach().reshape(-1) for p in params)])
    everyone = [torch.empty_like(mine) for _ in range(world)]
    dist.all_gather(everyone, mine)
    assert all(torch.equal(t, mine) for t in everyone)
    want, ref = _reference(world)
    # fp32 against fp64, or bf16 weights and activations (2^-8 each) of two layers
    tol = 0.05 if working else 1e-5
    for a, b in zip(norms, want):
        assert b > BOUND and abs(a - b) <= tol * b, (a, b)
    start = [p.detach() for p in _net().double().parameters()]
    for p, r, s in zip(params, ref, start):
        assert float((p.detach().double() - r).norm()) <= tol * float((r - s).norm()) + 1e-6
    if working:
        for _, _, master, work in weights.entries:
            assert torch.equal(work, master.to(torch.bfloat16))


@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("working", [False, True])
def test_clipped_steps_of_two_ranks(inside, working):
    run_distributed(_body, 2, inside, working)
