"""The plain forms compute in 32 bits, also where autocast would have their
products in 16: they are what the kernels are held against."""

import pytest
import torch

from test_operators_traced import data
from turboprune_amd.ops import functional as TF
from turboprune_amd.ops.norm_act import add_rms_norm, gelu

BF16 = torch.bfloat16


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("compute", [BF16, torch.float32])
def test_linear(grad, compute):
    def run(amp):
        d = data("cpu", 0)
        leaves = [d[k].requires_grad_(grad) for k in ("x", "w", "b", "r2")]
        with torch.autocast("cpu", BF16, enabled=amp):
            y = TF.masked_linear_act(d["x"], d["w"], d["m"], d["b"], d["r2"],
                                     "gelu", compute_dtype=compute,
                                     keep="e4m3")
            # a backward pass under autocast as well
            return [y.detach()] + (list(torch.autograd.grad(
                y, leaves, torch.ones_like(y))) if grad else [])
    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))


def test_norm_and_gelu():
    def run(amp):
        d = data("cpu", 0)
        leaves = [d[k].requires_grad_() for k in ("x", "r", "nw")]
        with torch.autocast("cpu", BF16, enabled=amp):
            y, h, kept = add_rms_norm(d["x"], d["r"], d["nw"], keep="e4m3")
            z = gelu(y, keep="e4m3")
            return [y.detach(), h.detach(), kept.codes.float()] + list(
                torch.autograd.grad((z, h), leaves, (torch.ones_like(z),
                                                     torch.ones_like(h))))
    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))
