"""The outputs of the operators with nodes of their own are ordinary tensors:
they can be changed in place, as those of the elementary operations can."""

import pytest
import torch

from turboprune_amd.ops import functional as TF
from turboprune_amd.ops.mask_layers import Conv1dMask
from turboprune_amd.ops.norm_act import add_rms_norm, gelu

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
F32, BF16 = torch.float32, torch.bfloat16


def inputs(lead, res, dev):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(*lead, 40, generator=g).to(dev, BF16)
    w = (torch.randn(24, 40, generator=g) * 0.2).to(dev)
    m = (torch.rand(24, 40, generator=g) < 0.6).float().to(dev)
    b = torch.randn(24, generator=g).to(dev)
    r = None if res is None else torch.randn(*lead, 24, generator=g).to(dev,
                                                                       res)
    dy = torch.randn(*lead, 24, generator=g).to(dev, res or BF16)
    return x, w, m, b, r, dy


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("lead", [(6,), (2, 3), (), (0,), (2, 0)])
@pytest.mark.parametrize("res", [None, BF16, F32])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear(dev, lead, res, act):
    x, w, m, b, r, dy = inputs(lead, res, dev)
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_()

    def run():
        return TF.masked_linear_act(x, w, m, b, r, act, compute_dtype=BF16,
                                    keep="e4m3")
    y = run()
    want = y.detach().add(1).mul(2)
    # a power of two, so that dy's rounding does not go by the order
    ref = torch.autograd.grad(y, leaves, 2 * dy)
    y = run()
    y.add_(1).mul_(2)
    assert torch.equal(y.detach(), want)
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("lead", [(6,), (2, 3), (70, 70)])
def test_linear_without_gradient(dev, lead):
    """What a call without gradients returns may meet one afterwards."""
    x, w, m, b, r, _ = inputs(lead, F32, dev)
    with torch.no_grad():
        y = TF.masked_linear_act(x, w, m, b, r, compute_dtype=BF16)
    p = torch.ones(24, device=dev, requires_grad=True)
    y.add_(p)
    y.sum().backward()
    assert (p.grad == y.numel() // 24).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_layer_before_in_place_modules(dev):
    torch.manual_seed(0)
    layer = Conv1dMask(in_features=40, out_features=24, bias=True).to(dev)
    layer.enable_cache(BF16)
    x = torch.randn(2, 5, 40, device=dev, dtype=BF16)
    y = torch.nn.functional.relu(layer.fused(x), inplace=True)
    z = torch.nn.functional.dropout(layer.fused(x), 0.5, inplace=True)
    (y.float().sum() + z.float().sum()).backward()
    assert layer.weight.grad.isfinite().all()


@pytest.mark.parametrize("dev", DEVICES)
def test_norm_and_gelu(dev):
    x, _, _, _, _, _ = inputs((2, 3), F32, dev)
    r = torch.randn(2, 3, 40, device=dev).requires_grad_()
    w = torch.rand(40, device=dev).requires_grad_()
    x.requires_grad_()
    dy = torch.randn(2, 3, 40, device=dev).to(BF16)
    y, _, _ = add_rms_norm(x, r, w, keep="e4m3")
    ref = torch.autograd.grad(y, (x, r, w), 2 * dy)
    y, _, _ = add_rms_norm(x, r, w, keep="e4m3")
    y.add_(1).mul_(2)
    got = torch.autograd.grad(y, (x, r, w), dy)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    ref, = torch.autograd.grad(gelu(x, keep="e4m3"), x, 2 * dy)
    y = gelu(x, keep="e4m3")
    y.add_(1).mul_(2)
    got, = torch.autograd.grad(y, x, dy)
    assert torch.equal(got, ref)
