"""Activations kept in 8 bits.

The format (csrc/act8.h): a row is cut into blocks of 32 values; a block
holds e4m3 codes and one power of two, the smallest within 2^-126 .. 2^126
that brings its largest finite magnitude to 448 or less (a magnitude within
6 % of the largest float takes the code below, so that it stays finite). A value is off by at
most 2^-4 of itself (half a step of e4m3), or by 2^-10 of its block's scale
where it is that small. NaN and infinities become NaN. 1.03 bytes a value,
against 2 in bfloat16.

Dequantised values are exact in bfloat16, so reading them as such for the matrix
products of a backward pass (``functional.masked_linear_act``) adds nothing to
the error of keeping. What those products add is the rounding of the gradient
that they multiply them by to the compute type.

CPU tensors take the plain PyTorch form below, which is also the kernels'
numerics oracle.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from turboprune_amd.ops import _backend

BLOCK = 32
KEEP = (None, "e4m3")
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def check_keep(keep: Optional[str]) -> None:
    if keep not in KEEP:
        raise ValueError(f"keep={keep!r}: one of {KEEP}")


def check_float(name: str, t: torch.Tensor) -> None:
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name} is {t.dtype}: float32, bfloat16 or float16 "
                        "expected")


class Act8(NamedTuple):
    """A tensor in the 8-bit format: ``codes`` (float8_e4m3fn, the tensor's
    shape) and ``scales`` (float8_e8m0fnu, one for every 32 values of the
    last dimension, from 2^-126 to 2^126)."""

    codes: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the codes stand for, within ``dtype``'s finite
        range."""
        return dequantize_act8(self, dtype)


def quantize_act8(x: torch.Tensor) -> Act8:
    """``x`` in the 8-bit format, blocks along its last dimension. No
    autograd."""
    check_float("x", x)
    if x.dim() < 1:
        raise ValueError("quantize_act8: a tensor of at least one dimension")
    x = x.detach()
    if _backend.use_native(x):
        return Act8(*(_QuantizeFn.apply(x) if torch.jit.is_tracing()
                      else _backend.extension().act8_quantize(x)))
    return _quantize_plain(x)


class _QuantizeFn(torch.autograd.Function):
    """A native call as one node of a trace, without gradients: a trace records
    the allocation of such a call's outputs, but not the kernel that fills
    them, and a Function as a whole."""

    @staticmethod
    def forward(ctx, x):
        codes, scales = _backend.extension().act8_quantize(x)
        ctx.mark_non_differentiable(codes, scales)
        return codes, scales

    @staticmethod
    def backward(ctx, *_):
        return None


class _DequantizeFn(torch.autograd.Function):
    """The same for the way back."""

    @staticmethod
    def forward(ctx, codes, scales, dtype):
        values = _dequantize_native(codes, scales, dtype)
        ctx.mark_non_differentiable(values)
        return values

    @staticmethod
    def backward(ctx, _):
        return None, None, None


def dequantize_act8(kept: Act8, dtype: torch.dtype = torch.bfloat16
                    ) -> torch.Tensor:
    """The values that ``kept`` stands for."""
    if dtype not in _FLOATS:
        raise TypeError(f"dtype={dtype}: float32, bfloat16 or float16")
    if _backend.use_native(*kept):
        return (_DequantizeFn.apply if torch.jit.is_tracing()
                else _dequantize_native)(*kept, dtype)
    check_act8(kept)
    return _dequantize_plain(kept, dtype)


def _dequantize_native(codes, scales, dtype):
    try:
        return _backend.extension().act8_dequantize(codes, scales, dtype)
    except RuntimeError:
        # which says what is wrong with the arguments
        check_act8(Act8(codes, scales))
        raise


def check_act8(kept: Act8, like: Optional[torch.Tensor] = None) -> None:
    """Refuses what is not in the format, or not of ``like``'s shape."""
    codes, scales = kept
    if codes.dtype != torch.float8_e4m3fn \
            or scales.dtype != torch.float8_e8m0fnu:
        raise TypeError("kept: float8_e4m3fn codes and float8_e8m0fnu "
                        f"scales expected, not {codes.dtype} and "
                        f"{scales.dtype}")
    if codes.dim() < 1:
        raise ValueError("kept: codes of at least one dimension")
    want = codes.shape[:-1] + (-(-codes.shape[-1] // BLOCK),)
    if scales.shape != want:
        raise ValueError(f"kept: scales of shape {tuple(want)} expected for "
                         f"codes of {tuple(codes.shape)}, not "
                         f"{tuple(scales.shape)}")
    if codes.device != scales.device:
        raise ValueError("kept: codes and scales on two devices")
    if like is not None and (codes.shape != like.shape
                             or codes.device != like.device):
        raise ValueError(f"kept: codes of shape {tuple(like.shape)} on "
                         f"{like.device} expected, not "
                         f"{tuple(codes.shape)} on {codes.device}")


def _blocks(x: torch.Tensor) -> torch.Tensor:
    b = F.pad(x, (0, -x.shape[-1] % BLOCK))
    return b.reshape(*x.shape[:-1], b.shape[-1] // BLOCK, BLOCK)


def _quantize_plain(x: torch.Tensor) -> Act8:
    b = _blocks(x.float())
    finite = torch.isfinite(b)
    top = torch.where(finite, b.abs(), torch.zeros_like(b))
    top = top.amax(-1, keepdim=True) if b.numel() else top[..., :1]
    # top = m 2^k with m in [1, 2): 2^(k-8), one more where m > 1.75
    bits = top.view(torch.int32)
    e = (((bits + 0x1FFFFF) >> 23) - 135).clamp(-126, 126)
    inv = ((127 - e) << 23).view(torch.float32)
    most = torch.where(e < 120, 448.0, 240.0)
    q = torch.where(finite, torch.minimum(torch.maximum(b * inv, -most), most),
                    torch.full_like(b, float("nan")))
    q = q.to(torch.float8_e4m3fn).view(torch.uint8)
    q = q.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]] if b.numel() \
        else torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    s = (e + 127).to(torch.uint8).squeeze(-1)
    return Act8(q.contiguous().view(torch.float8_e4m3fn),
                s.contiguous().view(torch.float8_e8m0fnu))


def _dequantize_plain(kept: Act8, dtype: torch.dtype) -> torch.Tensor:
    codes, scales = kept
    if codes.numel() == 0:
        return torch.empty(codes.shape, dtype=dtype, device=codes.device)
    s = (scales.view(torch.uint8).int() << 23).view(torch.float32)
    b = _blocks(codes.float()) * s.unsqueeze(-1)
    v = b.reshape(*codes.shape[:-1], -1)[..., :codes.shape[-1]]
    if dtype == torch.float16:
        v = v.clamp(-65504.0, 65504.0)
    return v.to(dtype)
