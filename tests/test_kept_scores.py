"""Pruning scores of models that keep activations in 8 bits: the gradients at
the activations' own values."""

import pytest
import torch

from test_deit_kept import vit
from turboprune_amd.ops.mask_layers import masked_modules
from turboprune_amd.pruning.prune import prune_snip, prune_synflow


@pytest.mark.parametrize("prune", [prune_snip, prune_synflow])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_masks_do_not_go_by_what_is_kept(prune, norm):
    torch.manual_seed(7)
    batch = [(torch.randn(8, 3, 32, 32), torch.randint(0, 10, (8,)))]
    masks = []
    for keep in (None, "e4m3"):
        m = vit("cpu", norm=norm, keep=keep)
        prune(m, 0.3, batch)
        masks.append([layer.mask.clone() for _, layer in masked_modules(m)])
        assert all(b.keep == keep and b.mlp.act.keep == keep
                   for b in m.blocks)
    assert all(torch.equal(a, b) for a, b in zip(*masks))


def test_an_error_leaves_the_model_as_it_was():
    m = vit("cpu", keep="e4m3")
    with pytest.raises(RuntimeError):
        prune_snip(m, 0.3, [(torch.randn(8, 4, 32, 32),
                             torch.randint(0, 10, (8,)))])
    assert all(b.keep == "e4m3" and b.mlp.act.keep == "e4m3"
               for b in m.blocks)


def test_other_modules_keep_is_their_own():
    class Scale(torch.nn.Module):
        keep = 0.5

        def forward(self, x):
            return x * self.keep
    m = vit("cpu", keep="e4m3")
    m.blocks.append(Scale())
    prune_snip(m, 0.3, [(torch.randn(8, 3, 32, 32),
                         torch.randint(0, 10, (8,)))])
    assert m.blocks[2].keep == 0.5
