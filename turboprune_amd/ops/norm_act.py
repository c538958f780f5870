"""Fused LayerNorm + exact GELU modules (ViT path). Drop-in for
nn.LayerNorm / nn.GELU; torch fallbacks on CPU and unsupported shapes
are the numerics oracles (see csrc/layernorm_gelu.hip).

``add_rms_norm`` / ``FusedRMSNorm`` add the residual, normalise by the root
mean square and can hand on the rows in 8 bits as well (csrc/rms_norm.hip);
``gelu(keep="e4m3")`` / ``FusedGELU(keep="e4m3")`` keep their input for the
backward pass in 8 bits (csrc/act8.hip). The 8-bit format is ops/act8.py's.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import os

import torch.nn.functional as F

from typing import Optional, Tuple

from torch.autograd.function import once_differentiable

from turboprune_amd.ops import _backend
from turboprune_amd.ops import act8
from turboprune_amd.ops.act8 import Act8


class _LNFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        ext = _backend.extension()
        y, mean, rstd = ext.ln_fwd(x, gamma, beta, eps)
        ctx.save_for_backward(x, gamma, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gamma, mean, rstd = ctx.saved_tensors
        ext = _backend.extension()
        dx, dgamma, dbeta = ext.ln_bwd(x, dy, gamma, mean, rstd)
        return dx, dgamma.to(gamma.dtype), dbeta.to(gamma.dtype), None


class FusedLayerNorm(nn.LayerNorm):
    """nn.LayerNorm with a fused HIP path for last-dim normalization of
    bf16/f32 tensors (state dict identical)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        vn = 8 if x.dtype == torch.bfloat16 else 4
        if (os.environ.get("TURBOPRUNE_LN", "native") == "native"
                and x.is_cuda and len(self.normalized_shape) == 1
                and x.dtype in (torch.bfloat16, torch.float32)
                and x.shape[-1] == self.normalized_shape[0]
                and x.shape[-1] % vn == 0
                and self.weight is not None and self.bias is not None
                and _backend.use_native(x)):
            return _LNFn.apply(x, self.weight, self.bias, self.eps)
        return super().forward(x)


class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ext = _backend.extension()
        ctx.save_for_backward(x)
        return ext.gelu_fwd(x)

    @staticmethod
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        ext = _backend.extension()
        return ext.gelu_bwd(x, dy)


class _GeluKeep8Fn(torch.autograd.Function):
    """The node for CPU tensors, in the plain form, and for torch.jit.trace; on
    a GPU the node is else the extension's."""

    @staticmethod
    def forward(ctx, x):
        if _backend.use_native(x):
            y, *kept = _backend.extension().gelu_keep8_fwd(x)
        else:
            y = gelu_plain(x.float()).to(x.dtype)
            kept = act8.quantize_act8(x)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        if _backend.use_native(codes):
            return _backend.extension().gelu_keep8_bwd(codes, scales, dy)
        z = act8.dequantize_act8(Act8(codes, scales), torch.float32)
        return (dy.float() * gelu_slope(z)).to(dy.dtype)


def gelu_plain(z: torch.Tensor) -> torch.Tensor:
    """Exact GELU, z Phi(z), by erfc: 1 + erf cancels for negative z."""
    return z * (0.5 * torch.special.erfc(-z * 0.5 ** 0.5))


def gelu_slope(z: torch.Tensor) -> torch.Tensor:
    """The derivative of exact GELU: Phi(z) + z phi(z)."""
    cdf = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    return cdf + z * (torch.exp(-0.5 * z * z) * 0.3989422804014327)


def gelu(x: torch.Tensor, keep: Optional[str] = None) -> torch.Tensor:
    """Exact (erf) GELU. With ``keep="e4m3"`` the input is held for the
    backward pass in the 8-bit format of ``ops.act8`` (1.03 bytes a value)
    and the slope is taken at the value it then stands for; without a
    gradient to come, nothing is kept. float32, bfloat16 and float16 tensors
    of any shape with at least one dimension."""
    act8.check_keep(keep)
    if keep is None or not (torch.is_grad_enabled() and x.requires_grad):
        return _gelu(x)
    if _backend.use_native(x) and not torch.jit.is_tracing():
        return _backend.extension().gelu_keep8(x)
    act8.check_float("x", x)
    if x.dim() < 1:
        raise ValueError("gelu(keep=...): a tensor of at least one dimension")
    return _GeluKeep8Fn.apply(x)


def _gelu(x: torch.Tensor) -> torch.Tensor:
    vn = 8 if x.dtype == torch.bfloat16 else 4
    if (os.environ.get("TURBOPRUNE_GELU", "native") == "native"
            and x.is_cuda and x.dtype in (torch.bfloat16, torch.float32)
            and x.numel() % vn == 0 and _backend.use_native(x)):
        return _GeluFn.apply(x)
    return F.gelu(x)


class FusedGELU(nn.Module):
    """Exact (erf) GELU with fused HIP fwd/bwd; ``keep="e4m3"`` holds the
    input for the backward pass in 8 bits."""

    def __init__(self, keep: Optional[str] = None):
        super().__init__()
        act8.check_keep(keep)
        self.keep = keep

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gelu(x, self.keep)

    def extra_repr(self) -> str:
        return "" if self.keep is None else f"keep={self.keep!r}"


class _AddRMSNormFn(torch.autograd.Function):
    """The node for CPU tensors, in the plain form, and for torch.jit.trace."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, out_dtype, keep):
        ctx.set_materialize_grads(False)
        y, h, rstd, codes, scales = _rms_fwd(x, residual, weight, eps,
                                             out_dtype, keep)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.x_dtype, ctx.residual = x.dtype, residual is not None
        if codes is not None:
            ctx.mark_non_differentiable(codes, scales)
        return y, h, codes, scales

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh, *_):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:            # only the sum was used
            dx = None if dh is None else dh.to(ctx.x_dtype)
            return dx, dh, None, None, None, None
        bwd = _backend.extension().rms_bwd if _backend.use_native(h) \
            else _rms_bwd_plain
        dx, dr, dw = bwd(dy, dh, h, weight, rstd, ctx.x_dtype, ctx.residual)
        return dx, dr, dw.to(weight.dtype), None, None, None


def _rms_fwd(x, residual, weight, eps, out_dtype, keep):
    if _backend.use_native(x):
        return _backend.extension().rms_fwd(x, residual, weight, eps,
                                            out_dtype, True, keep is not None)
    return _rms_fwd_plain(x, residual, weight, eps, out_dtype, keep)


def _rms_fwd_plain(x, residual, weight, eps, out_dtype, keep):
    h = None if residual is None else \
        (x.float() + residual.float()).to(residual.dtype)
    hf = (x if h is None else h).float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + eps)
    yf = hf * rstd * weight.float()
    kept = (None, None) if keep is None else act8.quantize_act8(yf)
    return (yf.to(out_dtype), h, rstd.reshape(-1), *kept)


def _rms_bwd_plain(dy, dh, h, weight, rstd, x_dtype, has_residual):
    g = dy.float()
    rstd = rstd.reshape(h.shape[:-1] + (1,))
    hat = h.float() * rstd
    gw = g * weight.float()
    d = rstd * (gw - hat * (gw * hat).mean(-1, keepdim=True))
    if dh is not None:
        d = d + dh.float()
    dw = (g * hat).reshape(-1, h.shape[-1]).sum(0)
    return d.to(x_dtype), d.to(h.dtype) if has_residual else None, dw


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor],
                 weight: torch.Tensor, eps: float = 1e-6,
                 keep: Optional[str] = None,
                 out_dtype: Optional[torch.dtype] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor, Optional[Act8]]:
    """``h = x + residual`` and ``y = h * rsqrt(mean(h^2) + eps) * weight``
    over the last dimension, in one pass.

    Returns ``(y, h, kept)``. ``h`` has the residual's type and is rounded to
    it before it is normalised (without a residual ``h`` is ``x`` itself);
    ``y`` has ``out_dtype``, ``x``'s type by default; ``kept`` is None, or with
    ``keep="e4m3"`` the unrounded ``y`` in the 8-bit format of ``ops.act8``,
    which ``functional.masked_linear_act(kept=...)`` takes in place of
    quantising its input again. ``y`` and ``h`` are differentiable, ``kept``
    is not.

    ``x`` is float32, bfloat16 or float16; the residual has ``x``'s shape and
    its type or float32; ``out_dtype`` is ``x``'s type, or a 16-bit type where
    ``x`` is float32; ``weight`` is a vector of the last dimension's length
    in any of the three types. Rows may lie at any distance. Statistics and
    the weight's gradient are summed in float32, in a fixed order. Neither
    gradients of gradients nor, on a GPU, forward-mode derivatives.
    """
    native = _backend.use_native(x)
    if native and not torch.jit.is_tracing():
        y, h, codes, scales = _backend.extension().add_rms_norm(
            x, residual, weight, eps, keep, out_dtype)
        return y, h, None if codes is None else Act8(codes, scales)
    act8.check_keep(keep)
    act8.check_float("x", x)
    act8.check_float("weight", weight)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("add_rms_norm: x needs rows of at least one value, "
                         f"not shape {tuple(x.shape)}")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"add_rms_norm: weight of shape {(x.shape[-1],)} "
                         f"expected, not {tuple(weight.shape)}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("add_rms_norm: residual of shape "
                             f"{tuple(x.shape)} expected, not "
                             f"{tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"add_rms_norm: residual in {x.dtype} or float32 "
                            f"expected, not {residual.dtype}")
    out_dtype = out_dtype or x.dtype
    if out_dtype != x.dtype and not (
            x.dtype == torch.float32
            and out_dtype in (torch.bfloat16, torch.float16)):
        raise TypeError(f"add_rms_norm: out_dtype {out_dtype} for x in "
                        f"{x.dtype}")
    for name, t in (("residual", residual), ("weight", weight)):
        if t is not None and t.device != x.device:
            raise ValueError(f"add_rms_norm: {name} on {t.device}, x on "
                             f"{x.device}")
    if native or torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad
            or (residual is not None and residual.requires_grad)):
        y, h, codes, scales = _AddRMSNormFn.apply(x, residual, weight, eps,
                                                  out_dtype, keep)
    else:
        y, h, _, codes, scales = _rms_fwd_plain(x, residual, weight, eps,
                                                out_dtype, keep)
    return (y, x if h is None else h,
            None if codes is None else Act8(codes, scales))


class FusedRMSNorm(nn.Module):
    """RMS norm over the last dimension, as a norm layer of the transformer
    models: ``norm(x)`` is the normalised tensor; ``norm.add(x, residual,
    keep)`` is ``add_rms_norm``'s triple. Under autocast a float32 stream is
    normalised straight to the autocast type."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def _out(self, x: torch.Tensor) -> torch.dtype:
        if x.dtype == torch.float32 and torch.is_autocast_enabled(
                x.device.type):
            return torch.get_autocast_dtype(x.device.type)
        return x.dtype

    def add(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
            keep: Optional[str] = None):
        return add_rms_norm(x, residual, self.weight, self.eps, keep,
                            self._out(x))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.add(x)[0]

    def extra_repr(self) -> str:
        return f"{self.weight.numel()}, eps={self.eps}"
