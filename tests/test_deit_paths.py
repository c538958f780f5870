"""The fused blocks of the transformer models: what they compute beside what
their modules' own calls would."""

import pytest
import torch

from test_deit_kept import step, vit
from turboprune_amd.ops.norm_act import FusedRMSNorm

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
def test_codes_only_where_they_are_kept(dev, monkeypatch):
    """The norms write 8-bit rows for the product behind them, which keeps them
    only for its weight's gradient."""
    seen = []
    add = FusedRMSNorm.add

    def spy(self, *a, **k):
        out = add(self, *a, **k)
        seen.append(out[2] is not None)
        return out
    monkeypatch.setattr(FusedRMSNorm, "add", spy)
    m = vit(dev, norm="rms", keep="e4m3")

    def run(**kw):
        del seen[:]
        step(m, dev)
        return seen[:4]
    assert run() == [True] * 4
    for layer in (m.blocks[0].attn.qkv, m.blocks[1].mlp.fc1):
        layer.weight.requires_grad_(False)
    seen.clear()
    with torch.autocast(dev, torch.bfloat16, enabled=dev == "cuda"):
        m(torch.randn(2, 3, 32, 32, device=dev)).float().sum().backward()
    assert seen[:4] == [False, True, True, False]
    seen.clear()
    with torch.no_grad(), torch.autocast(dev, torch.bfloat16,
                                         enabled=dev == "cuda"):
        m.eval()(torch.randn(2, 3, 32, 32, device=dev))
    assert seen[:4] == [False] * 4
