"""Linear layers with MXFP4 weights: the product that a quantized model runs.

``linear_mxfp4`` takes what ``mxwave_b200.core.quantize_mxfp4`` returns and
computes ``act(x W^T + bias) + residual`` on the tensor cores' block-scaled
MXFP4 path, from one token to long prompts, without dequantizing the weight.
The reference has no such operator: the consumers of its checkpoints
dequantize (mxwave/core.py:254-278) or bring their own.
"""

from __future__ import annotations

import torch

from . import _lib
from .core import BLOCK_SIZE

ACTIVATIONS = {
    "none": _lib.MXW_ACT_NONE,
    "relu": _lib.MXW_ACT_RELU,
    "silu": _lib.MXW_ACT_SILU,
    "gelu": _lib.MXW_ACT_GELU,  # the erf form
}


def linear_mxfp4(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str = "none",
    residual: torch.Tensor | None = None,
) -> torch.Tensor:
    """``act(x W^T + bias) + residual`` with W [out, in] held in MXFP4.

    x: [..., in] bf16 or f16; packed [out, in//2] and scales [out, in//32]
    uint8 as ``quantize_mxfp4`` returns them; bias [out] and residual
    [..., out] of x's type.  Returns [..., out] of x's type.  Sums are fp32 and
    rounded once, after the residual; the order of additions is fixed, so equal
    calls give equal bits.  A row of x that holds a NaN or an infinity gives
    NaN in all its outputs.  There is no gradient.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unknown activation: {activation}")
    if x.ndim < 1 or packed.ndim != 2 or scales.ndim != 2:
        raise ValueError("x must have a last dimension, packed and scales must be matrices")
    inner, outs = x.shape[-1], packed.shape[0]
    if inner == 0 or inner % BLOCK_SIZE != 0:
        raise ValueError(f"Last dim {inner} not divisible by BLOCK_SIZE={BLOCK_SIZE}")
    if packed.shape[1] != inner // 2 or scales.shape != (outs, inner // BLOCK_SIZE):
        raise ValueError(f"packed {tuple(packed.shape)} and scales {tuple(scales.shape)} do not hold [out, {inner}] weights")
    if packed.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("packed and scales must be uint8")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.device.type != "cuda":
        raise RuntimeError(f"mxwave_b200 runs on CUDA devices only; x is on {x.device} (no CPU fallback)")
    for name, t, shape in (("bias", bias, (outs,)), ("residual", residual, (*x.shape[:-1], outs))):
        if t is not None and (t.shape != shape or t.dtype != x.dtype):
            raise ValueError(f"{name} must be a {x.dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    for name, t in (("packed", packed), ("scales", scales), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, bias, residual)):
        raise RuntimeError("linear_mxfp4 has no gradient: call it under torch.no_grad()")

    from . import ops

    rows = _rows(x, inner)
    args = (rows, packed.contiguous(), scales.contiguous(), None if bias is None else bias.contiguous(),
            None if residual is None else _rows(residual, outs), ACTIVATIONS[activation])
    y = ops._linear_mxfp4(*args) if ops.plain_eager(x) else torch.ops.mxwave_b200.linear_mxfp4(*args)
    return y if x.ndim == 2 else y.reshape(*x.shape[:-1], outs)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """`t` as a matrix whose rows are contiguous and do not overlap."""
    m = t if t.ndim == 2 else t.reshape(-1, width)
    if width > 1 and m.stride(1) != 1 or m.shape[0] > 1 and m.stride(0) < width:
        m = m.contiguous()
    return m


__all__ = ["ACTIVATIONS", "linear_mxfp4"]
