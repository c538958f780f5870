"""Functional masked ops with reference-exact semantics.

The observable contract (reference: utils/mask_layers.py:23-34,59-70,
104-119): forward computes with ``mask * weight``; the autograd chain
therefore multiplies the weight gradient by the mask. Raw (unmasked)
weights keep receiving weight-decay/momentum updates — they are nullified
at forward time only — and checkpoints contain the raw weights.

MI355X design: ``mask_apply`` is a single fused HIP kernel producing the
compute-dtype masked weight (no fp32 temp + separate autocast cast), and
layers may hold a *cached* masked weight maintained by the fused SGD
kernel so steady-state forwards skip the multiply entirely.
"""

from __future__ import annotations

import os
from typing import Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from turboprune_amd.ops import _backend
from turboprune_amd.ops import act8
from turboprune_amd.ops.act8 import Act8


def mask_apply(weight: torch.Tensor, mask: torch.Tensor,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """out = (mask != 0) ? weight : 0, cast to out_dtype. No autograd."""
    out_dtype = out_dtype or weight.dtype
    if _backend.use_native(weight, mask):
        return _backend.extension().mask_apply(weight, mask, out_dtype)
    return (weight * mask).to(out_dtype)


def grad_mask_apply(grad: torch.Tensor, mask: torch.Tensor,
                    out_dtype: torch.dtype) -> torch.Tensor:
    """grad_weight = mask ⊙ grad, cast to the raw weight dtype."""
    if _backend.use_native(grad, mask):
        return _backend.extension().mask_apply(grad, mask, out_dtype)
    return (grad * mask.to(grad.dtype)).to(out_dtype)


class MaskedWeight(torch.autograd.Function):
    """Differentiable masked weight: forward yields ``mask ⊙ weight`` (or a
    pre-computed cache of it), backward applies the mask to the gradient and
    casts to the raw weight's dtype."""

    @staticmethod
    def forward(ctx, weight: torch.Tensor, mask: torch.Tensor,
                cache: Optional[torch.Tensor], compute_dtype: Optional[torch.dtype]):
        ctx.save_for_backward(mask)
        ctx.weight_dtype = weight.dtype
        if cache is not None:
            return cache
        return mask_apply(weight, mask, compute_dtype or weight.dtype)

    @staticmethod
    def backward(ctx, grad):
        (mask,) = ctx.saved_tensors
        return grad_mask_apply(grad, mask, ctx.weight_dtype), None, None, None


def masked_weight(weight: torch.Tensor, mask: torch.Tensor,
                  cache: Optional[torch.Tensor] = None,
                  compute_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return MaskedWeight.apply(weight, mask, cache, compute_dtype)


def masked_conv2d(x, weight, mask, bias=None, stride=1, padding=0,
                  dilation=1, groups=1, cache=None, compute_dtype=None):
    w = masked_weight(weight, mask, cache, compute_dtype)
    return F.conv2d(x, w, bias, stride, padding, dilation, groups)


def masked_linear(x, weight, mask, bias=None, cache=None, compute_dtype=None):
    w = masked_weight(weight, mask, cache, compute_dtype)
    if w.dtype == torch.bfloat16 and x.dtype != w.dtype:
        # the bf16 masked-weight cache defines the compute dtype; cast
        # the activations like autocast would inside F.linear (also
        # required OUTSIDE autocast — F.linear raises on mixed dtypes)
        x = x.to(torch.bfloat16)
    # TURBOPRUNE_GEMM: auto (default, per-shape routing) | native
    # (always in-house MFMA GEMM) | library (always hipBLASLt)
    mode = os.environ.get("TURBOPRUNE_GEMM", "auto")
    if (mode != "library" and _backend.use_native(x, w) and x.dim() >= 2):
        ext = _backend.extension()
        if ext is not None and hasattr(ext, "masked_linear_available") \
                and ext.masked_linear_available(x, w) \
                and (mode == "native" or _gemm_shape_native_wins(x, w)):
            return _MaskedLinearGemm.apply(x, w, bias)
    return F.linear(x, w, bias)


def _gemm_shape_native_wins(x, w) -> bool:
    """Per-shape routing from the round-1 PMC table
    (profiles/r01_gemm_mfma_pmc.md): the in-house 128² MFMA GEMM beats
    hipBLASLt on tall token-GEMMs (M ≥ tens of thousands, N,K ≤ ~2k —
    every DeiT training shape, incl. its split-K grad_w at 2.1×) and
    loses on big squares (8192³: 901 vs 1565 TF) and on small-M
    classifier heads (ResNet50 fc 512×1000×2048: 48 vs 100 TF). Routing
    at the Function level is enough: when (M,N,K) is in the token
    regime, both backward GEMMs (M×K×N and the deep-K N×K×M) are in
    regimes ours wins too."""
    K = x.shape[-1]
    M = x.numel() // K
    N = w.shape[0]
    return M >= 4096 and N <= 2048 and K <= 2048


class _MaskedLinearGemm(torch.autograd.Function):
    """Linear on the in-house MFMA GEMM kernel (y = x @ w^T + b).

    Forward/backward both route through the HIP GEMM; backward grads:
      grad_x = grad_y @ w ; grad_w = grad_y^T @ x ; grad_b = sum(grad_y).
    """

    @staticmethod
    def forward(ctx, x, w, bias):
        ctx.save_for_backward(x, w)
        ctx.bias_dtype = bias.dtype if bias is not None else None
        ext = _backend.extension()
        return ext.linear_fwd(x, w, bias)

    @staticmethod
    def backward(ctx, grad_y):
        x, w = ctx.saved_tensors
        ext = _backend.extension()
        gy = grad_y.contiguous()
        grad_x, grad_w = ext.linear_bwd(gy, x, w)
        grad_b = None
        if ctx.bias_dtype is not None:
            gy2 = gy.reshape(-1, gy.shape[-1])
            if gy2.dtype == torch.bfloat16 and gy2.shape[-1] % 8 == 0:
                # one streaming HIP pass (the eager reduce was 5.5% of
                # the DeiT step, profiles/r02_bench_final.md)
                grad_b = ext.colsum_bf16(gy2).to(ctx.bias_dtype)
            else:
                grad_b = gy2.sum(0).to(ctx.bias_dtype)
        return grad_x, grad_w, grad_b


ACTS = (None, "gelu")


class _MaskedLinearAct(torch.autograd.Function):
    """One node from the raw weight: product, bias, activation and residual
    forward; dx, masked dw, db and dresidual backward. The node for CPU tensors,
    in the plain form, and for torch.jit.trace; on a GPU the node is else the
    extension's."""

    @staticmethod
    def forward(ctx, x, w, weight, mask, bias, residual, act, keep, codes,
                scales):
        # the pre-activation is needed by the slope, the input only by dw
        need = ctx.needs_input_grad
        need_x, need_z = need[2], need[0] or need[2] or need[4]
        keep_x = keep is not None and codes is None and need_x
        y, z, zs, xc, xs = _linear_act_fwd(
            x, w, bias, residual, act,
            0 if not need_z else 1 if keep is None else 2, keep_x)
        if keep_x:
            codes, scales = xc, xs
        kept = (None, None) if not need_x else \
            (x, None) if keep is None else (codes, scales)
        ctx.save_for_backward(w, z, zs, *kept, mask if need_x else None)
        ctx.weight, ctx.bias = (weight.dtype, weight.shape), \
            None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, z, zs, xk, xs, mask = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[2] or need[4]:
            bwd = _backend.extension().linear_act_bwd \
                if _backend.use_native(w) else _linear_act_bwd_plain
            dx, dw, db = bwd(
                dy, z, zs, xk, xs, w, mask, need[0],
                ctx.weight[0] if need[2] else None,
                ctx.bias if need[4] else None)
        if dw is not None:
            dw = dw.reshape(ctx.weight[1])
        return (dx, None, dw, None, db, dy if need[5] else None, None, None,
                None, None)


def _linear_act_fwd(x, w, bias, residual, act, keep, keep_x):
    """(y, z, its scales, x's codes, their scales)."""
    if _backend.use_native(x):
        return _backend.extension().linear_act_fwd(
            x, w, bias, residual, act is not None, keep, keep_x)
    return (*_linear_act_fwd_plain(x, w, bias, residual, act, keep),
            *(act8.quantize_act8(x) if keep_x else (None, None)))


def _product32(a, b):
    """In 32 bits, whatever autocast says."""
    with torch.autocast(a.device.type, enabled=False):
        return a.float() @ b.float()


def _linear_act_fwd_plain(x, w, bias, residual, act, keep):
    from turboprune_amd.ops.norm_act import gelu_plain
    z = _product32(x, w.t())
    if bias is not None:
        z = z + bias.float()
    y = z if act is None else gelu_plain(z)
    if residual is not None:
        y = y + residual.float()
    y = y.to(x.dtype if residual is None else residual.dtype)
    if act is None or keep == 0:
        return y, None, None
    if keep == 2:
        return y, *act8.quantize_act8(z)
    if x.dtype == torch.float16:    # an infinity would have no slope
        z = z.clamp(-65504.0, 65504.0)
    return y, z.to(x.dtype), None


def _linear_act_bwd_plain(dy, z, zs, xk, xs, w, mask, want_dx, dw_type, db_type):
    from turboprune_amd.ops.norm_act import gelu_slope
    dz = dy.float()
    if z is not None:
        z = z.float() if zs is None else \
            act8.dequantize_act8(Act8(z, zs), torch.float32)
        dz = dz * gelu_slope(z)
    dx = dw = db = None
    if want_dx:
        dx = _product32(dz, w).to(w.dtype)
    if dw_type is not None:
        x = xk.float() if xs is None else \
            act8.dequantize_act8(Act8(xk, xs), torch.float32)
        dw = _product32(dz.t(), x)
        if mask is not None:
            dw = torch.where(mask.reshape(dw.shape) != 0, dw,
                             torch.zeros_like(dw))
        dw = dw.to(dw_type)
    if db_type is not None:
        db = dz.sum(0).to(db_type)
    return dx, dw, db


def masked_linear_act(x: torch.Tensor, weight: torch.Tensor,
                      mask: Optional[torch.Tensor],
                      bias: Optional[torch.Tensor] = None,
                      residual: Optional[torch.Tensor] = None,
                      act: Optional[str] = None,
                      cache: Optional[torch.Tensor] = None,
                      compute_dtype: Optional[torch.dtype] = None,
                      keep: Optional[str] = None,
                      kept: Optional[Act8] = None) -> torch.Tensor:
    """``act(x @ (mask * weight)^T + bias) + residual`` with everything after
    the product in its epilogue.

    ``x`` is ``(..., K)``, ``weight`` ``(N, K)``; ``mask`` float32 of its shape,
    or None; ``bias`` ``(N,)``; ``residual`` of the output's shape, in the
    compute type or float32, which is then the output's type too; ``act`` None
    or ``"gelu"`` (exact). ``cache`` and ``compute_dtype`` are
    ``masked_linear``'s: the masked weight in the compute type, and that type
    where there is no cache. The compute type is bfloat16 or float16 on a GPU
    (also float32 on the CPU); an ``x`` of another type is cast to it. For
    float32 products on a GPU there is ``masked_linear``: the matrix
    instructions that this kernel is made of take 16-bit operands. At most 2^30
    rows, and 2^20 values in a row of ``x`` and of the output.

    For the backward pass the input and, with an activation, the
    pre-activation are kept: in the compute type, or with ``keep="e4m3"`` in
    the 8-bit format of ``ops.act8`` (the gradients are then taken at the
    values it stands for). ``kept`` is ``x`` already in that format, as
    ``add_rms_norm`` hands it on. The weight's gradient is masked and has the
    weight's type. The gradient of the pre-activation is rounded to the compute
    type (on a GPU) before the products that give ``x``'s and the weight's, as
    between two layers of that type; the bias's is summed before that rounding.
    Sums are in 32 bits, in an order that does not change from call to call.
    Neither gradients of gradients nor, on a GPU, forward-mode derivatives.
    """
    native = _backend.use_native(x)
    tracing = torch.jit.is_tracing()
    if native and not tracing:
        codes, scales = kept if kept is not None else (None, None)
        return _backend.extension().masked_linear_act(
            x, weight, mask, bias, residual, act, cache, compute_dtype, keep,
            codes, scales)
    act8.check_keep(keep)
    if act not in ACTS:
        raise ValueError(f"act={act!r}: one of {ACTS}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("masked_linear_act: x (..., K) and weight (N, K) "
                         f"expected, not {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    N, K = weight.shape
    for name, t, shape in (("mask", mask, (N, K)), ("bias", bias, (N,)),
                           ("cache", cache, (N, K)),
                           ("residual", residual, x.shape[:-1] + (N,))):
        if t is not None and t.shape != torch.Size(shape):
            raise ValueError(f"masked_linear_act: {name} of shape "
                             f"{tuple(shape)} expected, not {tuple(t.shape)}")
    for name, t in (("weight", weight), ("mask", mask), ("bias", bias),
                    ("cache", cache), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"masked_linear_act: {name} on {t.device}, x on "
                             f"{x.device}")
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None:
            act8.check_float(name, t)
    if mask is not None and mask.dtype != torch.float32:
        raise TypeError(f"masked_linear_act: mask is {mask.dtype}: float32 "
                        "expected")
    if cache is not None:
        w = cache.detach()
    else:
        ct = compute_dtype or (weight.dtype if weight.dtype != torch.float32
                               else x.dtype)
        with torch.no_grad():
            w = _masked_compute(weight.detach(), mask, ct)
    ct = w.dtype
    act8.check_float("the compute type", w)
    if native and ct == torch.float32:
        raise TypeError("masked_linear_act computes in bfloat16 or float16 on "
                        "a GPU")
    if residual is not None and residual.dtype not in (ct, torch.float32):
        raise TypeError(f"masked_linear_act: residual in {ct} or float32 "
                        f"expected, not {residual.dtype}")
    if kept is not None:
        if keep is None:
            raise ValueError("masked_linear_act: kept needs keep='e4m3'")
        act8.check_act8(kept, like=x)
    if x.dtype != ct:
        x = x.to(ct)
    if bias is not None and bias.dtype not in (ct, torch.float32):
        bias = bias.to(ct)
    lead = x.shape[:-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    r2 = residual if residual is None or residual.dim() == 2 else \
        residual.reshape(-1, N)
    if x2.numel() == 0 or N == 0:
        y = _linear_of_nothing(x2, weight, bias, r2, ct)
    elif native or torch.is_grad_enabled() and any(
            t is not None and t.requires_grad
            for t in (x, weight, bias, residual)):
        codes, scales = (None, None) if kept is None else \
            (kept.codes.reshape(x2.shape), kept.scales.reshape(
                x2.shape[0], -1))
        y = _MaskedLinearAct.apply(x2, w, weight, mask, bias, r2, act, keep,
                                   codes, scales)
    else:
        y = _linear_act_fwd_plain(x2, w, bias, r2, act, 0)[0]
    if x.dim() == 2:
        return y
    if tracing:                       # the sizes are variables of the trace
        return y.reshape(lead + (N,))
    # no view: one made without gradients could not be changed in place later
    return torch.ops.aten._unsafe_view(y, lead + (N,))


def _masked_compute(weight, mask, dtype):
    if mask is None:
        return weight.to(dtype)
    if _backend.use_native(weight, mask) and weight.dtype == torch.float32 \
            and dtype == torch.bfloat16:
        if torch.jit.is_tracing():
            return MaskedWeight.apply(weight, mask, None, dtype)
        return mask_apply(weight, mask, dtype)
    # chosen, not multiplied: an infinity in a masked place stays there
    return torch.where(mask != 0, weight, torch.zeros_like(weight)).to(dtype)


def _linear_of_nothing(x, weight, bias, residual, dtype):
    """No rows, or rows of nothing: the sum is empty and no kernel runs."""
    if x.shape[1] == 0 or weight.shape[0] == 0:
        if x.shape[0] and weight.shape[0]:
            raise ValueError("masked_linear_act: rows of at least one value")
    y = x.new_empty((x.shape[0], weight.shape[0]), dtype=dtype)
    # keeps every input in the graph, so that each gets a gradient of zeros
    y = y + (x.sum() + weight.sum()
             + (bias.sum() if bias is not None else 0)).to(dtype) * 0
    return y if residual is None else (y + residual).to(residual.dtype)


def synflow_linearize_(t: torch.Tensor):
    """t <- |t| in place; returns the sign tensor (reference
    pruning_utils.py:223-248). GPU: one fused HIP pass emitting int8
    signs; CPU oracle: torch sign + abs_."""
    if _backend.use_native(t) and t.dtype == torch.float32 \
            and t.is_contiguous():
        return _backend.extension().sign_abs_(t)
    s = torch.sign(t)
    t.abs_()
    return s


def synflow_restore_(t: torch.Tensor, sign: torch.Tensor):
    """t <- t * sign in place (signs from synflow_linearize_)."""
    if _backend.use_native(t) and t.dtype == torch.float32 \
            and sign.dtype == torch.int8 and t.is_contiguous():
        _backend.extension().mul_sign_(t, sign)
        return t
    return t.mul_(sign.to(t.dtype))


def bernoulli_mask_(mask: torch.Tensor, p: float,
                    seed: Optional[int] = None) -> torch.Tensor:
    """In-place Bernoulli(p) fill of a mask buffer (reference:
    mask_layers.py:43 ``zeros_like(weight).bernoulli_(p)``).

    On GPU a Philox counter-based HIP kernel is used (seeded from torch's
    RNG unless an explicit seed is given)."""
    if _backend.use_native(mask):
        if seed is None:
            seed = int(torch.randint(0, 2**31 - 1, (1,)).item())
        _backend.extension().bernoulli_mask_(mask, float(p), seed)
        return mask
    return mask.zero_().bernoulli_(p)


def kth_smallest(values: torch.Tensor, k: int) -> float:
    """k-th smallest (1-based) of a 1-D tensor — the pruning threshold
    primitive (reference: torch.kthvalue at utils/pruning_utils.py:79).

    GPU path: multi-pass radix select HIP kernel (no full sort)."""
    assert values.dim() == 1
    assert 1 <= k <= values.numel(), (k, values.numel())
    if _backend.use_native(values):
        return float(_backend.extension().kth_smallest(values, k))
    return float(torch.kthvalue(values.float().cpu(), k).values)


def mask_from_threshold_(mask: torch.Tensor, score: torch.Tensor,
                         threshold: float) -> torch.Tensor:
    """mask = where(score <= threshold, 0, 1) in place (reference:
    utils/pruning_utils.py:82-88)."""
    if _backend.use_native(mask, score):
        _backend.extension().mask_from_threshold_(mask, score, float(threshold))
        return mask
    mask.copy_(torch.where(score <= threshold,
                           torch.zeros_like(mask), torch.ones_like(mask)))
    return mask


def masked_abs_score(weight: torch.Tensor, mask: torch.Tensor,
                     other: Optional[torch.Tensor] = None) -> torch.Tensor:
    """|mask * weight| (magnitude) or |mask * weight * other| (SNIP/SynFlow
    style with other=grad). Reference: utils/pruning_utils.py:75,189-191."""
    if _backend.use_native(weight, mask):
        return _backend.extension().masked_abs_score(
            weight, mask, other if other is not None else torch.Tensor())
    s = (mask * weight).detach()
    if other is not None:
        s = s * other
    return s.abs()


def cross_entropy(logits: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """Mean-reduction cross-entropy. GPU: fused log-softmax+NLL fwd/bwd HIP
    kernel (one pass over logits each way); CPU: torch reference."""
    if _backend.use_native(logits) and logits.dim() == 2:
        return _FusedCrossEntropy.apply(logits.contiguous(), target)
    return F.cross_entropy(logits, target)


class _FusedCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target):
        ext = _backend.extension()
        loss, lse = ext.ce_fwd(logits, target)
        ctx.save_for_backward(logits, target, lse)
        return loss

    @staticmethod
    def backward(ctx, grad_out):
        logits, target, lse = ctx.saved_tensors
        ext = _backend.extension()
        grad_logits = ext.ce_bwd(logits, target, lse, grad_out)
        return grad_logits, None


def accuracy_count(logits: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """Number of argmax(logits)==target hits, as a device tensor (reference:
    torchmetrics Accuracy, base_harness.py:54-60 — synced per epoch here)."""
    if _backend.use_native(logits) and logits.dim() == 2:
        return _backend.extension().accuracy_count(logits.contiguous(), target)
    return (logits.argmax(dim=-1) == target).sum()
