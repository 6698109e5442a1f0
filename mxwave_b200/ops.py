"""torch custom operators over the C ABI (namespace ``mxwave_b200``).

Each operator wraps one entry point of include/mxwave_b200.h with a schema, a
CUDA implementation (allocation through torch's caching allocator on the
input's device, launch on torch's current stream) and a fake implementation,
so callers get shape propagation under FakeTensor / ``torch.compile`` and
``torch.library.opcheck`` coverage.  Argument validation with the
reference's messages stays in the host mirror (``mxwave_b200.core``,
``mxwave_b200.calibration``); these operators only enforce the C ABI's own
contract, and a non-OK status raises (ValueError for MXW_EINVAL).

Operators (reference function each one backs):

* ``quantize_mxfp4(weight, scale_percentile, gamma, hessian, method,
  mse_clip_depth, flags) -> (packed, scales)`` -- mxwave/core.py:114-251;
  ``flags`` is a caller-owned int32 word that receives MXW_FLAG_* bits.
* ``dequant_mxfp4(packed, scales, rows, cols) -> fp32`` -- core.py:254-278.
* ``accumulate_moments_(x, sum_abs, sum_sq)`` -- calibration.py:227-232.
* ``accumulate_activation_stats_(x, sum_abs?, sum_sq?, gram_blocks?)`` --
  calibration.py:226-236 in one read of ``x``.
* ``accumulate_xtx_(x, gram)`` -- the full X^T X on the tensor cores
  (the reference forms only its diagonal blocks, calibration.py:233-236).
* ``finalize_moments(sums, count, root) -> fp32`` -- calibration.py:262-266.
* ``finalize_block_hessian(gram, full, count, damp, mode) -> fp32`` --
  calibration.py:267-270 with core.py:61-69.

Serving operators (no counterpart in the reference; ``mxwave_b200.linear``
and ``mxwave_b200.kvcache`` hold their public functions and argument checks):

* ``linear_mxfp4(x, packed, scales, bias?, residual?, act) -> y`` -- the product
  with quantized weights.
* ``kv_append_mxfp4_(codes, scales, key, value, slots)`` and
  ``kv_gather_mxfp4(codes, scales, slots, dtype) -> (key, value)`` -- rows of a
  paged cache in MXFP4 (``mxwave_b200.kvcache``).
* ``copy_pages_(codes, scales, source, target)`` -- page copies in every layer;
  ``source`` and ``target`` are host tensors.
* ``paged_attention_mxfp4(query, codes, scales, table, lengths, query_start,
  max_length, max_queries, softmax_scale, causal, window, want_lse) -> (out,
  lse)``; lse is empty unless wanted.

Dispatching a custom operator costs more host time than their smallest calls
take on the device, so the public functions have two shorter ways for eager
calls on plain CUDA tensors: ``binding`` (csrc/binding.cpp) takes the ordinary
ones whole, and the functions here with a leading underscore, which the
operators wrap, take the rest.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib

_DTYPE_CODES = {torch.bfloat16: _lib.MXW_BF16, torch.float16: _lib.MXW_F16, torch.float32: _lib.MXW_F32}


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _cuda_2d(x: Tensor, what: str) -> tuple[Tensor, int]:
    """A 2-D view with unit column stride in a native dtype."""
    if x.device.type != "cuda":
        raise RuntimeError(f"mxwave_b200 runs on CUDA devices only; {what} is on {x.device} (no CPU fallback)")
    if x.ndim != 2:
        raise ValueError(f"{what} must be 2-D, got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPE_CODES:
        x = x.to(torch.float32)
    if x.stride(-1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x, _DTYPE_CODES[x.dtype]


def _f32_buffer(t: Tensor, shape: tuple[int, ...], what: str) -> None:
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device.type != "cuda":
        raise ValueError(f"{what} must be a contiguous CUDA float32 tensor of shape {shape}")


# ------------------------------------------------------------------ quantize


@torch.library.custom_op("mxwave_b200::quantize_mxfp4", mutates_args=("flags",))
def quantize_mxfp4(
    weight: Tensor,
    scale_percentile: float,
    gamma: Tensor | None,
    hessian: Tensor | None,
    method: int,
    mse_clip_depth: int,
    flags: Tensor,
) -> tuple[Tensor, Tensor]:
    w, code = _cuda_2d(weight, "the weight")
    rows, cols = w.shape
    packed = torch.empty((rows, cols // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((rows, cols // 32), dtype=torch.uint8, device=w.device)
    if rows == 0:
        return packed, scales
    if flags.dtype != torch.int32 or flags.numel() < 1 or flags.device != w.device:
        raise ValueError("flags must be an int32 tensor on the weight's device")
    lib = _lib.load()
    with torch.cuda.device(w.device):
        status = lib.mxw_quantize_mxfp4(
            w.data_ptr(), code, rows, cols, w.stride(0), float(scale_percentile), _ptr(gamma), _ptr(hessian),
            method, mse_clip_depth, packed.data_ptr(), scales.data_ptr(), flags.data_ptr(), _stream(w.device),
        )
    _lib.check(status, "mxw_quantize_mxfp4")
    return packed, scales


@quantize_mxfp4.register_fake
def _(weight, scale_percentile, gamma, hessian, method, mse_clip_depth, flags):
    rows, cols = weight.shape
    return (weight.new_empty((rows, cols // 2), dtype=torch.uint8),
            weight.new_empty((rows, cols // 32), dtype=torch.uint8))


@torch.library.custom_op("mxwave_b200::dequant_mxfp4", mutates_args=())
def dequant_mxfp4(packed: Tensor, scales: Tensor, rows: int, cols: int) -> Tensor:
    if packed.device.type != "cuda":
        raise RuntimeError(f"mxwave_b200 runs on CUDA devices only; packed is on {packed.device} (no CPU fallback)")
    p = packed.reshape(rows, cols // 2).contiguous()
    s = scales.reshape(rows, cols // 32).to(device=packed.device).contiguous()
    out = torch.empty((rows, cols), dtype=torch.float32, device=packed.device)
    lib = _lib.load()
    with torch.cuda.device(packed.device):
        status = lib.mxw_dequant_mxfp4(p.data_ptr(), s.data_ptr(), rows, cols, out.data_ptr(), _stream(packed.device))
    _lib.check(status, "mxw_dequant_mxfp4")
    return out


@dequant_mxfp4.register_fake
def _(packed, scales, rows, cols):
    return packed.new_empty((rows, cols), dtype=torch.float32)


# ------------------------------------------------------------- calibration


@torch.library.custom_op("mxwave_b200::accumulate_moments_", mutates_args=("sum_abs", "sum_sq"))
def accumulate_moments_(x: Tensor, sum_abs: Tensor, sum_sq: Tensor) -> None:
    xx, code = _cuda_2d(x, "the activation")
    tokens, cols = xx.shape
    _f32_buffer(sum_abs, (cols,), "sum_abs")
    _f32_buffer(sum_sq, (cols,), "sum_sq")
    if tokens == 0:
        return
    lib = _lib.load()
    with torch.cuda.device(xx.device):
        status = lib.mxw_accumulate_moments(xx.data_ptr(), code, tokens, cols, max(xx.stride(0), cols),
                                            sum_abs.data_ptr(), sum_sq.data_ptr(), _stream(xx.device))
    _lib.check(status, "mxw_accumulate_moments")


@accumulate_moments_.register_fake
def _(x, sum_abs, sum_sq):
    return None


@torch.library.custom_op("mxwave_b200::accumulate_activation_stats_",
                         mutates_args=("sum_abs", "sum_sq", "gram_blocks"))
def accumulate_activation_stats_(x: Tensor, sum_abs: Tensor | None, sum_sq: Tensor | None,
                                 gram_blocks: Tensor | None) -> None:
    xx, code = _cuda_2d(x, "the activation")
    tokens, cols = xx.shape
    if sum_abs is not None:
        _f32_buffer(sum_abs, (cols,), "sum_abs")
    if sum_sq is not None:
        _f32_buffer(sum_sq, (cols,), "sum_sq")
    if gram_blocks is not None:
        _f32_buffer(gram_blocks, (cols // 32, 32, 32), "gram_blocks")
    if tokens == 0:
        return
    lib = _lib.load()
    with torch.cuda.device(xx.device):
        status = lib.mxw_accumulate_activation_stats(
            xx.data_ptr(), code, tokens, cols, max(xx.stride(0), cols), _ptr(sum_abs), _ptr(sum_sq),
            _ptr(gram_blocks), None, _stream(xx.device),
        )
    _lib.check(status, "mxw_accumulate_activation_stats")


@accumulate_activation_stats_.register_fake
def _(x, sum_abs, sum_sq, gram_blocks):
    return None


@torch.library.custom_op("mxwave_b200::accumulate_xtx_", mutates_args=("gram",))
def accumulate_xtx_(x: Tensor, gram: Tensor) -> None:
    if x.dtype != torch.bfloat16:
        raise ValueError("accumulate_xtx_ takes bf16 activations")
    xx, _code = _cuda_2d(x, "the activation")
    tokens, cols = xx.shape
    _f32_buffer(gram, (cols, cols), "gram")
    if tokens == 0:
        return
    lib = _lib.load()
    with torch.cuda.device(xx.device):
        status = lib.mxw_accumulate_xtx(xx.data_ptr(), tokens, cols, xx.stride(0), gram.data_ptr(), cols, None,
                                        _stream(xx.device))
    _lib.check(status, "mxw_accumulate_xtx")


@accumulate_xtx_.register_fake
def _(x, gram):
    return None


@torch.library.custom_op("mxwave_b200::finalize_moments", mutates_args=())
def finalize_moments(sums: Tensor, count: int, root: bool) -> Tensor:
    _f32_buffer(sums, (sums.shape[0],), "sums")
    out = torch.empty_like(sums)
    lib = _lib.load()
    cols = sums.shape[0]
    with torch.cuda.device(sums.device):
        if root:
            status = lib.mxw_finalize_moments(None, sums.data_ptr(), cols, count, None, out.data_ptr(),
                                              _stream(sums.device))
        else:
            status = lib.mxw_finalize_moments(sums.data_ptr(), None, cols, count, out.data_ptr(), None,
                                              _stream(sums.device))
    _lib.check(status, "mxw_finalize_moments")
    return out


@finalize_moments.register_fake
def _(sums, count, root):
    return torch.empty_like(sums)


@torch.library.custom_op("mxwave_b200::finalize_block_hessian", mutates_args=())
def finalize_block_hessian(gram: Tensor, full: bool, count: int, damp: float, mode: int) -> Tensor:
    if full:
        cols = gram.shape[-1]
        _f32_buffer(gram, (cols, cols), "gram")
    else:
        cols = gram.shape[0] * 32
        _f32_buffer(gram, (cols // 32, 32, 32), "gram")
    out = torch.empty((cols // 32, 32, 32), dtype=torch.float32, device=gram.device)
    lib = _lib.load()
    with torch.cuda.device(gram.device):
        status = lib.mxw_finalize_block_hessian(gram.data_ptr(), 1 if full else 0, cols, cols, count, float(damp),
                                                mode, out.data_ptr(), _stream(gram.device))
    _lib.check(status, "mxw_finalize_block_hessian")
    return out


@finalize_block_hessian.register_fake
def _(gram, full, count, damp, mode):
    cols = gram.shape[-1] if full else gram.shape[0] * 32
    return gram.new_empty((cols // 32, 32, 32), dtype=torch.float32)


# ----------------------------------------------------------------- serving

try:
    from ._native import _binding as binding  # built with the library; without it calls only take longer
except ImportError:
    binding = None


# What every call dispatches through.  A dispatch mode (FakeTensor, make_fx, before the
# dispatch or in it), torch.jit's tracer and a functorch level (vmap) each add keys.
_UNWATCHED = (torch._C.DispatchKeySet(torch._C.DispatchKey.BackendSelect) | torch._C.DispatchKeySet(torch._C.DispatchKey.ADInplaceOrView)).raw_repr()


def plain_eager(t: Tensor) -> bool:
    """Whether a call on `t` may skip the operator dispatch: an ordinary tensor, and
    nothing (FakeTensor, tracing, compilation, a functorch transform, another dispatch mode) is watching."""
    return (type(t) is Tensor and not torch.compiler.is_compiling()
            and not torch._C._dispatch_tls_local_include_set().raw_repr() & ~_UNWATCHED)


def wants_gradient(*tensors: Tensor | None) -> bool:
    """Whether a derivative is asked for: a backward pass, or the tangents of a forward one."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _call(fn, index: int, args: tuple, what: str) -> None:
    """One call of the C ABI on device `index`, with its current stream as the last argument."""
    current = torch._C._cuda_getDevice()
    if current == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        torch._C._cuda_setDevice(index)
        try:
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
        finally:
            torch._C._cuda_setDevice(current)
    if status != _lib.MXW_OK:
        _lib.check(status, what)


def _linear_mxfp4(x: Tensor, packed: Tensor, scales: Tensor, bias: Tensor | None, residual: Tensor | None,
                  act: int) -> Tensor:
    rows, inner = x.shape
    outs = packed.shape[0]
    y = x.new_empty((rows, outs))
    if rows == 0 or outs == 0:
        return y
    if packed.data_ptr() % 16 != 0:  # a slice that starts inside a 16-byte line
        packed = packed.clone()
    lib = _lib.load()
    code = _DTYPE_CODES[x.dtype]
    nbytes = lib.mxw_linear_workspace_size(rows, inner, code)
    # Up to four rows the kernel needs none: any address will do.
    workspace = packed if nbytes <= 16 else packed.new_empty(nbytes)
    _call(lib.mxw_linear_mxfp4, x.device.index, (
        x.data_ptr(), code, rows, inner, x.stride(0) if rows > 1 else inner, packed.data_ptr(), scales.data_ptr(), outs,
        None if bias is None else bias.data_ptr(), act, None if residual is None else residual.data_ptr(),
        residual.stride(0) if residual is not None and rows > 1 else outs, y.data_ptr(), workspace.data_ptr(), nbytes, None,
    ), "mxw_linear_mxfp4")
    return y


linear_mxfp4 = torch.library.custom_op("mxwave_b200::linear_mxfp4", _linear_mxfp4, mutates_args=())


@linear_mxfp4.register_fake
def _(x, packed, scales, bias, residual, act):
    return x.new_empty((x.shape[0], packed.shape[0]))


def _kv_append_mxfp4_(codes: Tensor, scales: Tensor, key: Tensor, value: Tensor, slots: Tensor) -> None:
    pages, _two, heads, page, half = codes.shape
    tokens = slots.shape[0]
    if tokens == 0 or pages == 0:
        return
    key_token, key_head, _one = key.stride()
    value_token, value_head, _one = value.stride()
    _call(_lib.load().mxw_kv_append, codes.device.index, (
        codes.data_ptr(), scales.data_ptr(), pages, heads, page, 2 * half, key.data_ptr(), value.data_ptr(), _DTYPE_CODES[key.dtype],
        key_token, key_head, value_token, value_head, slots.data_ptr(), tokens,
    ), "mxw_kv_append")


kv_append_mxfp4_ = torch.library.custom_op("mxwave_b200::kv_append_mxfp4_", _kv_append_mxfp4_,
                                           mutates_args=("codes", "scales"))


@kv_append_mxfp4_.register_fake
def _(codes, scales, key, value, slots):
    return None


def _kv_gather_mxfp4(codes: Tensor, scales: Tensor, slots: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    pages, _two, heads, page, half = codes.shape
    tokens = slots.shape[0]
    key = codes.new_empty((tokens, heads, 2 * half), dtype=dtype)
    value = torch.empty_like(key)
    if tokens == 0:
        return key, value
    _call(_lib.load().mxw_kv_gather, codes.device.index, (
        codes.data_ptr(), scales.data_ptr(), pages, heads, page, 2 * half, slots.data_ptr(), tokens, _DTYPE_CODES[dtype], key.data_ptr(),
        value.data_ptr(),
    ), "mxw_kv_gather")
    return key, value


kv_gather_mxfp4 = torch.library.custom_op("mxwave_b200::kv_gather_mxfp4", _kv_gather_mxfp4, mutates_args=())


@kv_gather_mxfp4.register_fake
def _(codes, scales, slots, dtype):
    shape = (slots.shape[0], codes.shape[2], 2 * codes.shape[4])
    return codes.new_empty(shape, dtype=dtype), codes.new_empty(shape, dtype=dtype)


def _copy_pages_(codes: Tensor, scales: Tensor, source: Tensor, target: Tensor) -> None:
    layers, pages, two, heads, page, half = codes.shape
    n = source.shape[0]
    if n == 0 or layers == 0:
        return
    rows = two * heads * page
    _call(_lib.load().mxw_copy_pages, codes.device.index, (
        codes.data_ptr(), scales.data_ptr(), layers, pages, rows * half, rows * scales.shape[5], source.data_ptr(), target.data_ptr(), n,
    ), "mxw_copy_pages")


copy_pages_ = torch.library.custom_op("mxwave_b200::copy_pages_", _copy_pages_, mutates_args=("codes", "scales"))


@copy_pages_.register_fake
def _(codes, scales, source, target):
    return None


def _paged_attention_mxfp4(query: Tensor, codes: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, query_start: Tensor,
                           max_length: int, max_queries: int, softmax_scale: float, causal: bool, window: int,
                           lse: Tensor | None) -> Tensor:
    tokens, heads, dim = query.shape
    pages, _two, kv_heads, page, _half = codes.shape
    seqs, width = table.shape
    if tokens == 0 or seqs == 0:
        if lse is not None:
            lse.fill_(float("-inf"))
        return query.new_zeros((tokens, heads, dim))
    out = query.new_empty((tokens, heads, dim))
    lib = _lib.load()
    nbytes = lib.mxw_paged_attention_workspace_size(seqs, heads, kv_heads, dim, max_length, max_queries)
    workspace = codes if nbytes <= 16 else codes.new_empty(nbytes)  # (prompts need none: any address will do)
    q_token, q_head, _one = query.stride()
    _call(lib.mxw_paged_attention, query.device.index, (
        query.data_ptr(), _DTYPE_CODES[query.dtype], tokens, heads, q_token, q_head, codes.data_ptr(), scales.data_ptr(), pages, kv_heads,
        page, dim, table.data_ptr(), table.stride(0), width, lengths.data_ptr(), query_start.data_ptr(), seqs, max_length, max_queries,
        softmax_scale, causal, window, out.data_ptr(), None if lse is None else lse.data_ptr(), workspace.data_ptr(), nbytes, None,
    ), "mxw_paged_attention")
    return out


def _new_lse(query: Tensor, want: bool) -> Tensor:
    return query.new_empty(query.shape[:2] if want else (0,), dtype=torch.float32)


@torch.library.custom_op("mxwave_b200::paged_attention_mxfp4", mutates_args=())
def paged_attention_mxfp4(query: Tensor, codes: Tensor, scales: Tensor, table: Tensor, lengths: Tensor, query_start: Tensor,
                          max_length: int, max_queries: int, softmax_scale: float, causal: bool, window: int,
                          want_lse: bool) -> tuple[Tensor, Tensor]:
    lse = _new_lse(query, want_lse)
    out = _paged_attention_mxfp4(query, codes, scales, table, lengths, query_start, max_length, max_queries, softmax_scale, causal, window,
                                 lse if want_lse else None)
    return out, lse


@paged_attention_mxfp4.register_fake
def _(query, codes, scales, table, lengths, query_start, max_length, max_queries, softmax_scale, causal, window,
      want_lse):
    return query.new_empty(query.shape), _new_lse(query, want_lse)


OPS = (
    quantize_mxfp4,
    dequant_mxfp4,
    accumulate_moments_,
    accumulate_activation_stats_,
    accumulate_xtx_,
    finalize_moments,
    finalize_block_hessian,
    linear_mxfp4,
    kv_append_mxfp4_,
    kv_gather_mxfp4,
    copy_pages_,
    paged_attention_mxfp4,
)

__all__ = [
    "OPS",
    "accumulate_activation_stats_",
    "accumulate_moments_",
    "accumulate_xtx_",
    "copy_pages_",
    "dequant_mxfp4",
    "finalize_block_hessian",
    "finalize_moments",
    "kv_append_mxfp4_",
    "kv_gather_mxfp4",
    "linear_mxfp4",
    "paged_attention_mxfp4",
    "quantize_mxfp4",
]
