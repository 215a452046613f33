"""Residual norms with a 16-bit residual: the sum is made again in fp32 for the backward, never read back in 16 bits, and
every row takes part in the sums over rows.

The bounds are lm_oracle's for the same values held in fp32: with fp32 inputs it allows the kept sum one fp32
rounding, with 16-bit ones a 16-bit rounding, which is 2^13 (fp16) or 2^16 (bf16) times as wide and would hide both faults.
lm_oracle takes sums over rows as serial.  With the at most 9000 rows here they are not: a workgroup's slot of rows adds
at most 36 of them (9000 rows in 256 workgroups and more), a workgroup 16 slots, the fold 16 partial rows to a slice
and then 4 and 16 slices; torch's sum on the CPU cascades by 16.  DEEP = 128 roundings cover both.
"""
import pytest
import torch

import lm_oracle as O
from grace_amd.ops.norm import residual_norm
from test_lm_ops import norm_inputs

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NAMES = ("y", "x", "weight", "bias", "gate", "post_weight", "post_bias")
FEW = [(1, 1, 7, BF16, BF16), (2, 3, 1025, BF16, BF16), (1, 5, 96, F16, F16), (1, 3, 16384, BF16, BF16), (2, 2, 651, F16, F16),
       (2, 3, 130, BF16, BF16)]
MANY = [(7, 900, 12, BF16, BF16), (300, 30, 16, None, BF16), (35, 21, 651, F16, F16), (3, 700, 200, BF16, BF16)]
FORMS = [("layer", "none", False), ("rms", "channel", True), ("layer", "sample", True), ("layer", "channel", False),
         ("rms", "full", True)]


def made(b, t, d, tx, ty, kind, gate, post, device, gate_type=None):
    v, dh, ds = norm_inputs(b, t, d, tx, ty, gate, post, True, device, seed=b + t + d)
    if gate_type is not None and v["gate"] is not None:
        v["gate"] = v["gate"].to(gate_type)
    return v, dh, ds, 1.0 if tx is None else 1.5


DEEP = 128


def bounds(v, dh, ds, kind, alpha, post):
    """lm_oracle's, and the terms of dweight; dweight's and dbias' bounds for sums of DEEP roundings."""
    wide = [None if v[k] is None else v[k].float() for k in NAMES]
    out = O.residual_norm(*wide, kind == "rms", 1e-5, alpha, post, dh.float(), ds.float())
    s = out["s"][0]
    mean = 0.0 if kind == "rms" else s.mean(-1, keepdim=True)
    rstd = 1 / ((s - mean).square().mean(-1, keepdim=True) + 1e-5).sqrt()
    terms = dh.double() * (s - mean) * rstd
    rows = dh.numel() // dh.shape[-1]
    for k, t in (("dweight", terms), ("dbias", dh.double())):
        value, bound = out[k]
        out[k] = value, bound - max(0, rows + 4 - DEEP) * O.U * t.abs().sum((0, 1))
    return out, terms, mean, rstd


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,gate,post,gate_type", [(*f, g) for f in FORMS for g in (None, F32) if g is None or f[1] != "none"])
@pytest.mark.parametrize("b,t,d,tx,ty", FEW + MANY)
def test_gradients(b, t, d, tx, ty, kind, gate, post, gate_type, device):
    v, dh, ds, alpha = made(b, t, d, tx, ty, kind, gate, post, device, gate_type)
    leaves = {k: u.detach().requires_grad_() for k, u in v.items() if u is not None}
    h, s = residual_norm(leaves["y"], leaves.get("x"), leaves["weight"], leaves["bias"], kind=kind, gate=leaves.get("gate"),
                         alpha=alpha, post=post, post_weight=leaves.get("post_weight"),
                         post_bias=leaves.get("post_bias"), return_sum=True)
    got = dict(zip(leaves, torch.autograd.grad([h, s], list(leaves.values()), [dh, ds])))
    want = bounds(v, dh, ds, kind, alpha, post)[0]
    for k, g in got.items():
        assert g.dtype == v[k].dtype
        if device == "cpu" and k == "y" and tx is None and gate == "none" and not post:
            continue  # s is y: torch adds the two rounded gradients of y, and rounds again
        O.within(g, *want["d" + k], k)


def rejected(value, want, bound):
    try:
        O.within(value.float(), want, bound)
    except AssertionError:
        return True
    return False


@pytest.mark.parametrize("kind,gate,post", FORMS)
@pytest.mark.parametrize("b,t,d,tx,ty", FEW + MANY)
def test_the_bounds_reject(b, t, d, tx, ty, kind, gate, post):
    """dweight of a 16-bit sum that was read back (few rows: the bound grows with them, the fault with their root), and
    sums over rows that leave one out."""
    v, dh, ds, alpha = made(b, t, d, tx, ty, kind, gate, post, "cpu")
    ref, terms, mean, rstd = bounds(v, dh, ds, kind, alpha, post)
    want, bound = ref["dweight"]
    assert not rejected(terms.sum((0, 1)), want, bound)
    if (b, t, d, tx, ty) in FEW:
        back = ref["s"][0].to(ty).double()
        assert rejected((dh.double() * (back - mean) * rstd).sum((0, 1)), want, bound)
    assert rejected(want - terms[-1, -1], want, bound)
    assert rejected(ref["dbias"][0] - dh[-1, -1].double(), *ref["dbias"])
