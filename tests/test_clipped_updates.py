"""Clipping inside the SGD update and over views: 16-bit parameters, copies, pickles and state dicts of the optimizer,
steps without gradients, gradients that share memory."""
import pytest
import torch
import torch.nn as nn

import lm_oracle as O
from grace_amd.parallel import FusedSGD

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
