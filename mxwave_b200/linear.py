"""Linear layers with MXFP4 weights: the product that a quantized model runs.

``linear_mxfp4`` takes what ``mxwave_b200.core.quantize_mxfp4`` returns and
computes ``act(x W^T + bias) + residual`` on the tensor cores' block-scaled
MXFP4 path, from one token to long prompts, without dequantizing the weight.
The reference has no such operator: the consumers of its checkpoints
dequantize (mxwave/core.py:254-278) or bring their own.
"""

from __future__ import annotations

import torch

from . import _lib, ops
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
    calls give equal bits.  Products are taken of x as it is where an element is
    at least 2^-13 of the largest of its 32, and of x to within 2^-22 of that
    largest where it is smaller.  A row of x that holds a NaN or an infinity
    gives NaN in all its outputs.  There is no gradient.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"Unknown activation: {activation}")
    if ops.binding is not None and not torch.compiler.is_compiling():
        y = ops.binding.linear(x, packed, scales, bias, residual, act)
        if y is not None:
            return y
    _check(x, packed, scales, bias, residual)
    outs = packed.shape[0]
    args = (_rows(x), packed.contiguous(), scales.contiguous(), None if bias is None else bias.contiguous(),
            None if residual is None else _rows(residual), act)
    y = ops._linear_mxfp4(*args) if ops.plain_eager(x) else torch.ops.mxwave_b200.linear_mxfp4(*args)
    return y if x.ndim == 2 else y.reshape(*x.shape[:-1], outs)


def _check(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None) -> None:
    shape, held, blocks = x.shape, packed.shape, scales.shape
    if len(shape) < 1 or len(held) != 2 or len(blocks) != 2:
        raise ValueError("x must have a last dimension, packed and scales must be matrices")
    inner, outs = shape[-1], held[0]
    if inner == 0 or inner % BLOCK_SIZE != 0:
        raise ValueError(f"Last dim {inner} not divisible by BLOCK_SIZE={BLOCK_SIZE}")
    if held[1] != inner // 2 or blocks[0] != outs or blocks[1] != inner // BLOCK_SIZE:
        raise ValueError(f"packed {tuple(held)} and scales {tuple(blocks)} do not hold [out, {inner}] weights")
    if packed.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("packed and scales must be uint8")
    dtype, device = x.dtype, x.device
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError(f"x must be bfloat16 or float16, got {dtype}")
    if device.type != "cuda":
        raise RuntimeError(f"mxwave_b200 runs on CUDA devices only; x is on {device} (no CPU fallback)")
    if bias is not None and (bias.shape != (outs,) or bias.dtype != dtype):
        raise ValueError(f"bias must be a {dtype} tensor of shape {(outs,)}, got {bias.dtype} {tuple(bias.shape)}")
    if residual is not None and (residual.shape != (*shape[:-1], outs) or residual.dtype != dtype):
        raise ValueError(f"residual must be a {dtype} tensor of shape {(*shape[:-1], outs)}, got {residual.dtype} {tuple(residual.shape)}")
    for t in (packed, scales, bias, residual):
        if t is not None and t.device != device:
            raise ValueError(f"x is on {device}, another argument is on {t.device}")
    if ops.wants_gradient(x, bias, residual):
        raise RuntimeError("linear_mxfp4 has no gradient: call it under torch.no_grad()")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as a matrix whose rows are contiguous and do not overlap."""
    m = t if t.ndim == 2 else t.reshape(-1, t.shape[-1])
    if m.is_contiguous():
        return m
    rows, width = m.shape
    if width > 1 and m.stride(1) != 1 or rows > 1 and m.stride(0) < width:
        m = m.contiguous()
    return m


__all__ = ["ACTIVATIONS", "linear_mxfp4"]
