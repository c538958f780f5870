"""What the operators keep goes through the hooks on saved tensors: kept on the
host meanwhile, or made anew by a second forward pass."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_operators_traced import data
from turboprune_amd.ops import functional as TF
from turboprune_amd.ops.norm_act import add_rms_norm, gelu

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16 = torch.bfloat16


def block(x, r, nw, w, m, b):
    y, h, kept = add_rms_norm(x, r, nw, keep="e4m3")
    z = TF.masked_linear_act(y, w, m, b, act="gelu", compute_dtype=BF16,
                             keep="e4m3", kept=kept)
    z = TF.masked_linear_act(z, w.t(), m.t(), residual=h, act="gelu",
                             compute_dtype=BF16)
    return gelu(z, keep="e4m3")


@pytest.mark.parametrize("dev", DEVICES)
def test_kept_elsewhere(dev):
    d = data(dev, 0)
    args = [d[k].requires_grad_(k != "m") for k in ("x", "r", "nw", "w", "m",
                                                    "b")]
    leaves = [t for t in args if t.requires_grad]
    torch.manual_seed(1)
    dy = torch.randn_like(d["r"])
    y = block(*args)
    ref = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    with torch.autograd.graph.save_on_cpu():
        y = block(*args)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    for reentrant in (False, True):
        y = checkpoint(block, *args, use_reentrant=reentrant)
        got = [y.detach()]
        y.backward(dy)
        got += [t.grad for t in leaves]
        # a forward pass without gradients may add few rows in another order
        tol = 2.0 ** -6 if reentrant else 0
        for a, b in zip(ref, got):
            assert (a.double() - b.double()).norm() <= tol * a.double().norm()
        for t in leaves:
            t.grad = None
