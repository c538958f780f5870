"""Forward-mode differentiation, which the kernels do not offer: the calls say
so, and do not hand out results without the tangent."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_operators_traced import (data, linear, linear_16, norm, norm_alone,
                                   norm_kept)
from turboprune_amd.ops.norm_act import add_rms_norm, gelu


@pytest.mark.gpu
def test_refused_on_a_gpu():
    d = data("cuda", 0)
    ops = {norm: "x r nw", norm_kept: "x r nw", norm_alone: "r nw",
           linear: "x w b r2", linear_16: "x w"}
    for op, names in ops.items():
        for name in names.split():
            for grad in (False, True):
                with fwd.dual_level():
                    e = {k: v.clone().requires_grad_(grad and k != "m")
                         for k, v in d.items()}
                    e[name] = fwd.make_dual(e[name],
                                            torch.ones_like(e[name]))
                    with pytest.raises(NotImplementedError):
                        op(e)
    with fwd.dual_level():
        x = d["x"].clone().requires_grad_()
        with pytest.raises(NotImplementedError):
            gelu(fwd.make_dual(x, torch.ones_like(x)), keep="e4m3")
    norm(d), linear(d)           # and without a tangent as ever


def test_plain_form():
    """CPU tensors without reverse-mode gradients: elementary operations,
    which carry tangents."""
    d = data("cpu", 0)
    t = torch.randn_like(d["r"])
    with fwd.dual_level():
        e = dict(d, r=fwd.make_dual(d["r"], t))
        y, h = norm(e)
        got = fwd.unpack_dual(y).tangent
    eps = 1e-3
    up, down = (add_rms_norm(d["x"].double().float(), d["r"] + s * t,
                             d["nw"])[0].double() for s in (eps, -eps))
    assert (got.double() - (up - down) / (2 * eps)).abs().max() < 0.05
