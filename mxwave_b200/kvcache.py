"""A paged key/value cache in MXFP4, and attention over it.

The cache holds keys and values as the quantizer holds weights: 4-bit codes
and one E8M0 exponent per 32 elements, 4.25 bits per element.  One layer is

* ``codes``  uint8 [pages, 2 (key, value), kv_heads, page_tokens, head_dim // 2]
* ``scales`` uint8 [pages, 2, kv_heads, page_tokens, head_dim // 32]

and token ``slot`` of the pool is token ``slot % page_tokens`` of page ``slot //
page_tokens``.  A row is encoded as ``quantize_mxfp4(row, method="rtn")`` encodes
it (mxwave/core.py:91-104).  The functions below work on one layer (``copy_pages_``
on all); ``PagedKVCache`` owns the layers and keeps the books: which pages are
free, which sequences share them.  The reference quantizes weights only and has
no counterpart.
"""

from __future__ import annotations

from collections.abc import Sequence


import torch

from .core import BLOCK_SIZE

PAGE_TOKENS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_ROW_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _ops():
    from . import ops

    return ops


def _check_pool(codes: torch.Tensor, scales: torch.Tensor, layers: bool = False) -> None:
    """Codes and scales of one layer, or of several with a leading dimension."""
    lead = 1 if layers else 0
    if codes.ndim != 5 + lead or scales.ndim != 5 + lead or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"codes and scales must be {5 + lead}-D uint8 tensors")
    two, _heads, page, half = codes.shape[1 + lead :]
    if two != 2 or page not in PAGE_TOKENS or 2 * half not in HEAD_DIMS:
        raise ValueError(f"codes must be [.., pages, 2, kv_heads, page in {PAGE_TOKENS}, head_dim/2 of {HEAD_DIMS}], got {tuple(codes.shape)}")
    if scales.shape != (*codes.shape[:-1], half * 2 // BLOCK_SIZE):
        raise ValueError(f"scales {tuple(scales.shape)} do not match codes {tuple(codes.shape)}")
    if codes.device.type != "cuda":
        raise RuntimeError(f"mxwave_b200 runs on CUDA devices only; codes is on {codes.device} (no CPU fallback)")
    if scales.device != codes.device:
        raise ValueError(f"scales is on {scales.device}, codes on {codes.device}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("codes and scales must be contiguous")
    if codes.data_ptr() % 16 != 0 or scales.data_ptr() % 16 != 0:
        raise ValueError("codes and scales must be 16-byte aligned")


def _check_index(name: str, t: torch.Tensor, dtype: torch.dtype, ndim: int, device: torch.device) -> None:
    if t.ndim != ndim or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {ndim}-D {dtype} tensor on {device}, got {t.ndim}-D {t.dtype} on {t.device}")


def append_mxfp4_(codes: torch.Tensor, scales: torch.Tensor, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor) -> None:
    """Encode key and value rows [tokens, kv_heads, head_dim] and write them to their slots.

    bf16, f16 or fp32 rows with any token and head stride (slices of a fused
    projection need no copy).  slots: int64 [tokens], distinct; a slot outside
    the pool (-1) skips its row.  Nothing but the named rows is written.
    """
    _check_pool(codes, scales)
    heads, dim = codes.shape[2], 2 * codes.shape[4]
    if key.ndim != 3 or key.shape[1:] != (heads, dim) or value.shape != key.shape:
        raise ValueError(f"key and value must be [tokens, {heads}, {dim}], got {tuple(key.shape)} and {tuple(value.shape)}")
    if key.dtype not in _ROW_TYPES or value.dtype != key.dtype:
        raise ValueError(f"key and value must both be bfloat16, float16 or float32, got {key.dtype} and {value.dtype}")
    if key.device != codes.device or value.device != codes.device:
        raise ValueError(f"key and value must be on {codes.device}")
    _check_index("slots", slots, torch.int64, 1, codes.device)
    if slots.shape[0] != key.shape[0]:
        raise ValueError(f"slots holds {slots.shape[0]} entries for {key.shape[0]} rows")
    ops = _ops()
    args = (codes, scales, _unit_rows(key.detach()), _unit_rows(value.detach()), slots.contiguous())
    if ops.plain_eager(codes):
        ops._kv_append_mxfp4_(*args)
    else:
        torch.ops.mxwave_b200.kv_append_mxfp4_(*args)


def gather_mxfp4(
    codes: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
) -> tuple[torch.Tensor, torch.Tensor]:
    """The key and value rows of `slots` as values, each [tokens, kv_heads, head_dim] of `dtype`.

    bf16 and fp32 hold every MXFP4 value exactly; f16 rounds.  A slot outside
    the pool gives zeros.
    """
    _check_pool(codes, scales)
    if dtype not in _ROW_TYPES:
        raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    _check_index("slots", slots, torch.int64, 1, codes.device)
    ops = _ops()
    args = (codes, scales, slots.contiguous(), dtype)
    return ops._kv_gather_mxfp4(*args) if ops.plain_eager(codes) else torch.ops.mxwave_b200.kv_gather_mxfp4(*args)


def copy_pages_(
    codes: torch.Tensor, scales: torch.Tensor, source: torch.Tensor | Sequence[int], target: torch.Tensor | Sequence[int]
) -> None:
    """Copy pages source[i] to target[i] in every layer of [layers, pages, ...] codes and scales.

    The page numbers are host data (lists or CPU int64 tensors), read during
    the call.  No target may also be a source or appear twice: the copies of
    one call run in no order.
    """
    _check_pool(codes, scales, layers=True)
    source = torch.as_tensor(source, dtype=torch.int64)
    target = torch.as_tensor(target, dtype=torch.int64)
    if source.device.type != "cpu" or target.device.type != "cpu":
        raise ValueError("source and target are page numbers on the host")
    if source.ndim != 1 or source.shape != target.shape:
        raise ValueError(f"source and target must be vectors of one length, got {tuple(source.shape)} and {tuple(target.shape)}")
    ops = _ops()
    args = (codes, scales, source.contiguous(), target.contiguous())
    if ops.plain_eager(codes):
        ops._copy_pages_(*args)
    else:
        torch.ops.mxwave_b200.copy_pages_(*args)


def paged_attention_mxfp4(
    query: torch.Tensor,
    codes: torch.Tensor,
    scales: torch.Tensor,
    table: torch.Tensor,
    lengths: torch.Tensor,
    query_start: torch.Tensor,
    *,
    max_length: int,
    max_queries: int,
    softmax_scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Softmax attention of packed queries over one layer of the cache.

    query: [tokens, heads, head_dim] bf16 or f16, heads a multiple of kv_heads;
    rows query_start[b] .. query_start[b + 1] - 1 are the last tokens of
    sequence b, whose lengths[b] cached tokens (the new ones included: append
    before attending) lie in pages table[b].  table [seqs, width], lengths
    [seqs] and query_start [seqs + 1] are int32 on the device.

    A query sees the keys up to its own position (`causal`), the last `window`
    of them when `window` is positive.  max_length and max_queries bound the
    lengths and the queries of a sequence; they only size the launch.
    softmax_scale defaults to head_dim ** -0.5.  Returns [tokens, heads,
    head_dim] of query's type, and with `return_lse` the fp32 natural log of
    each row's sum of exponentials [tokens, heads].  A query that no key
    reaches, and a row of `query` behind the last sequence, gives zeros (and
    -inf).  Equal calls give equal bits.  There is no gradient.
    """
    _check_pool(codes, scales)
    kv_heads, dim = codes.shape[2], 2 * codes.shape[4]
    if query.ndim != 3 or query.shape[2] != dim or query.shape[1] == 0 or query.shape[1] % kv_heads != 0:
        raise ValueError(f"query must be [tokens, a multiple of {kv_heads} heads, {dim}], got {tuple(query.shape)}")
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"query must be bfloat16 or float16, got {query.dtype}")
    if query.device != codes.device:
        raise ValueError(f"query is on {query.device}, codes on {codes.device}")
    _check_index("table", table, torch.int32, 2, codes.device)
    _check_index("lengths", lengths, torch.int32, 1, codes.device)
    _check_index("query_start", query_start, torch.int32, 1, codes.device)
    seqs = table.shape[0]
    if lengths.shape[0] != seqs or query_start.shape[0] != seqs + 1:
        raise ValueError(f"{seqs} sequences need {seqs} lengths and {seqs + 1} starts, got {lengths.shape[0]} and {query_start.shape[0]}")
    if max_length < 0 or max_queries < 0:
        raise ValueError("max_length and max_queries must not be negative")
    if window < 0 or (window > 0 and not causal):
        raise ValueError("window must not be negative, and needs causal")
    scale = dim**-0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"softmax_scale must be positive and finite, got {softmax_scale}")
    if torch.is_grad_enabled() and query.requires_grad:
        raise RuntimeError("paged_attention_mxfp4 has no gradient: call it under torch.no_grad()")
    ops = _ops()
    if table.stride(1) != 1 or table.stride(0) < table.shape[1]:
        table = table.contiguous()
    args = (_unit_rows(query), codes, scales, table, lengths.contiguous(), query_start.contiguous(), int(max_length), int(max_queries),
            scale, bool(causal), int(window), bool(return_lse))
    fn = ops._paged_attention_mxfp4 if ops.plain_eager(query) else torch.ops.mxwave_b200.paged_attention_mxfp4
    out, lse = fn(*args)
    return (out, lse) if return_lse else out


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with unit stride over its last dimension (other strides may be anything)."""
    return t if t.stride(-1) == 1 else t.contiguous()


__all__ = ["HEAD_DIMS", "PAGE_TOKENS", "append_mxfp4_", "copy_pages_", "gather_mxfp4", "paged_attention_mxfp4"]
