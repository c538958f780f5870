"""Each tile of the linear layer's products against the formulas: which of them
a size goes to is asked of the rule itself, so that a rule that is measured
anew cannot leave one of them untested."""

import pytest
import torch

from test_linear_act import BF16, F32, FP16, check, make

SIZES = {(64, 64): [(300, 72, 200), (1025, 100, 1001)],
         (128, 128): [(5000, 136, 500)],
         (160, 128): [(9000, 200, 500), (12608, 72, 383)],
         (256, 256): [(9000, 384, 1536), (9000, 136, 1501), (8960, 72, 1535)]}


def tile(M, N):
    from turboprune_amd.ops._backend import extension
    return tuple(extension().linear_act_tile(M, N))


@pytest.mark.gpu
def test_sizes_reach_their_tiles():
    for want, sizes in SIZES.items():
        for M, _, N in sizes:
            assert tile(M, N) == want


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [s for v in SIZES.values() for s in v])
@pytest.mark.parametrize("keep", [None, "e4m3"])
@pytest.mark.parametrize("res", [None, BF16, F32])
def test_gelu(M, K, N, keep, res):
    check(make(M, K, N, BF16, res, "cuda"), BF16, "gelu", keep)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [v[-1] for v in SIZES.values()])
@pytest.mark.parametrize("res", [None, FP16, F32])
def test_half_and_without_activation(M, K, N, res):
    check(make(M, K, N, FP16, res, "cuda"), FP16, "gelu", "e4m3")
    check(make(M, K, N, BF16, BF16 if res == FP16 else res, "cuda"), BF16,
          None, "e4m3")


# rows, K, N: the weight's gradient in each of its tiles, whole and in slabs
WEIGHTS = {(64, False): [(60, 130, 70)], (64, True): [(900, 72, 200)],
           (128, False): [(300, 1900, 1100)], (128, True): [(3000, 500, 900)],
           (256, False): [(200, 2050, 2300)], (256, True): [(5000, 1000, 1001)]}


@pytest.mark.gpu
def test_weights_reach_their_tiles():
    from turboprune_amd.ops._backend import extension
    for (want, split), sizes in WEIGHTS.items():
        for M, K, N in sizes:
            t, slabs = extension().linear_act_split(M, N, K)
            assert (t, slabs > 1) == (want, split), (M, K, N, t, slabs)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [s for v in WEIGHTS.values() for s in v])
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("keep", [None, "e4m3"])
@pytest.mark.parametrize("weight", [F32, "same"])
def test_weight_gradients(M, K, N, t, keep, weight):
    check(make(M, K, N, t, None, "cuda",
               weight=t if weight == "same" else F32), t, None, keep)


def test_sizes_of_nothing_are_refused():
    from turboprune_amd.ops import _backend
    if not _backend.has_extension():
        pytest.skip("needs the extension, but no GPU")
    ext = _backend.extension()
    for bad in (lambda: ext.linear_act_tile(0, 64),
                lambda: ext.linear_act_tile(64, -1),
                lambda: ext.linear_act_tile(1 << 40, 64),
                lambda: ext.linear_act_split(0, 64, 64),
                lambda: ext.linear_act_split(64, 0, 64),
                lambda: ext.linear_act_split(64, 64, 1 << 21)):
        with pytest.raises(RuntimeError):
            bad()
