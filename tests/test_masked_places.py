"""What stands in the masked places of a weight does not reach the layer's
results: infinities and NaN there are as good as zeros."""

import math

import pytest
import torch

from turboprune_amd.ops import functional as TF

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("wt,ct", [(F32, BF16), (F32, FP16), (BF16, BF16)])
@pytest.mark.parametrize("keep", [None, "e4m3"])
def test_linear(dev, wt, ct, keep):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(70, 40, generator=g).to(dev, ct)
    w = torch.randn(24, 40, generator=g).to(dev, wt)
    m = (torch.rand(24, 40, generator=g) < 0.6).float().to(dev)
    m[3] = 0                               # a row of nothing
    dy = torch.randn(70, 24, generator=g).to(dev, ct)
    out = []
    for filled in (False, True):
        v = torch.where(m != 0, w, torch.zeros_like(w))
        if filled:
            bad = torch.tensor([math.nan, math.inf, -math.inf, 1e30],
                               device=dev).repeat(240).reshape(24, 40).to(wt)
            v = torch.where(m != 0, w, bad)
        leaves = [x.clone().requires_grad_(), v.requires_grad_()]
        y = TF.masked_linear_act(*leaves, m, act="gelu", compute_dtype=ct,
                                 keep=keep)
        with torch.no_grad():
            z = TF.masked_linear_act(*leaves, m, act="gelu",
                                     compute_dtype=ct)
        out.append([y.detach(), z, *torch.autograd.grad(y, leaves, dy)])
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert (out[0][0][:, 3] == 0).all() and (out[0][3][m == 0] == 0).all()
