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

import heapq
from collections.abc import Iterable, Sequence
from dataclasses import dataclass, field
from operator import index

import torch

from . import ops
from .core import BLOCK_SIZE

PAGE_TOKENS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_ROW_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_pool(codes: torch.Tensor, scales: torch.Tensor, layers: bool = False) -> None:
    """Codes and scales of one layer, or of several with a leading dimension."""
    shape, blocks = codes.shape, scales.shape
    ndim = 6 if layers else 5
    if len(shape) != ndim or len(blocks) != ndim or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"codes and scales must be {ndim}-D uint8 tensors")
    half = shape[-1]
    if shape[-4] != 2 or shape[-2] not in PAGE_TOKENS or 2 * half not in HEAD_DIMS:
        raise ValueError(f"codes must be [.., pages, 2, kv_heads, page in {PAGE_TOKENS}, head_dim/2 of {HEAD_DIMS}], got {tuple(shape)}")
    if blocks[:-1] != shape[:-1] or blocks[-1] * BLOCK_SIZE != 2 * half:
        raise ValueError(f"scales {tuple(blocks)} do not match codes {tuple(shape)}")
    device = codes.device
    if device.type != "cuda":
        raise RuntimeError(f"mxwave_b200 runs on CUDA devices only; codes is on {device} (no CPU fallback)")
    if scales.device != device:
        raise ValueError(f"scales is on {scales.device}, codes on {device}")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError("codes and scales must be contiguous")
    if ops.plain_eager(codes) and (codes.data_ptr() % 16 != 0 or scales.data_ptr() % 16 != 0):
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
    if ops.binding is not None and not torch.compiler.is_compiling() and ops.binding.append(codes, scales, key, value, slots):
        return
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
    args = (codes, scales, _unit_rows(key.detach()), _unit_rows(value.detach()), slots.contiguous())
    if ops.plain_eager(codes):
        ops._kv_append_mxfp4_(*args)
        _written(codes, scales)
    else:
        torch.ops.mxwave_b200.kv_append_mxfp4_(*args)


def gather_mxfp4(
    codes: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
) -> tuple[torch.Tensor, torch.Tensor]:
    """The key and value rows of `slots` as values, each [tokens, kv_heads, head_dim] of `dtype`.

    bf16 and fp32 hold every MXFP4 value exactly; f16 rounds.  A slot outside
    the pool gives zeros.
    """
    if ops.binding is not None and not torch.compiler.is_compiling():
        rows = ops.binding.gather(codes, scales, slots, dtype)
        if rows is not None:
            return rows
    _check_pool(codes, scales)
    if dtype not in _ROW_TYPES:
        raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    _check_index("slots", slots, torch.int64, 1, codes.device)
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
    if ops.binding is not None and not torch.compiler.is_compiling() and ops.binding.copy_pages(codes, scales, source, target):
        return
    source, target = _page_numbers("source", source), _page_numbers("target", target)
    _check_pool(codes, scales, layers=True)
    if source.ndim != 1 or source.shape != target.shape:
        raise ValueError(f"source and target must be vectors of one length, got {tuple(source.shape)} and {tuple(target.shape)}")
    args = (codes, scales, source.contiguous(), target.contiguous())
    if ops.plain_eager(codes):
        ops._copy_pages_(*args)
        _written(codes, scales)
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

    Scores, statistics and sums are fp32 (long prompts take queries as
    ``linear_mxfp4`` takes x); values times their scales are exact,
    and probabilities are held to 2^-11 of themselves and 2^-32 of their row's
    largest (f16).  A key that a row's mask hides has no say in it, however
    large its value.  Where the scales of the values that the rows of a head see
    span more than 2^20 within 32 channels, or 2^27 over all, those rows take
    fp32 throughout, which is far slower.
    """
    if ops.binding is not None and not torch.compiler.is_compiling():
        got = ops.binding.attention(query, codes, scales, table, lengths, query_start, max_length, max_queries, softmax_scale, causal, window,
                                    return_lse)
        if got is not None:
            return got
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
    if ops.wants_gradient(query):
        raise RuntimeError("paged_attention_mxfp4 has no gradient: call it under torch.no_grad()")
    if table.stride(1) != 1 or table.stride(0) < table.shape[1]:
        table = table.contiguous()
    args = (_unit_rows(query), codes, scales, table, lengths.contiguous(), query_start.contiguous(), int(max_length), int(max_queries),
            scale, bool(causal), int(window))
    if ops.plain_eager(query):
        lse = ops._new_lse(query, True) if return_lse else None
        out = ops._paged_attention_mxfp4(*args, lse)
    else:
        out, lse = torch.ops.mxwave_b200.paged_attention_mxfp4(*args, bool(return_lse))
    return (out, lse) if return_lse else out


def _written(*tensors: torch.Tensor) -> None:
    """What an in-place operator does to its tensors' version counters (inference tensors have none)."""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _page_numbers(name: str, pages: torch.Tensor | Sequence[int]) -> torch.Tensor:
    """Page numbers as a host tensor of int64."""
    if not isinstance(pages, torch.Tensor):
        pages = torch.tensor([index(page) for page in pages], dtype=torch.int64)
    if pages.dtype == torch.bool or pages.dtype.is_floating_point or pages.dtype.is_complex:
        raise ValueError(f"{name} must hold whole numbers, got {pages.dtype}")
    if pages.device.type != "cpu":
        raise ValueError(f"{name} holds page numbers on the host, got a tensor on {pages.device}")
    return pages.to(torch.int64)


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with unit stride over its last dimension (other strides may be anything)."""
    return t if t.stride(-1) == 1 else t.contiguous()


@dataclass
class _Held:
    """One sequence: its pages in order, and how many tokens of them it has."""

    pages: list[int] = field(default_factory=list)
    length: int = 0


class PageBooks:
    """Which pages are free, which sequences hold which, and what has to be copied.

    Host bookkeeping without tensors.  Pages are shared by reference; a page
    that more than one sequence holds is never written: the writer gets a copy
    first (``grow`` names the copies).
    """

    def __init__(self, pages: int, page_tokens: int) -> None:
        if pages <= 0 or page_tokens <= 0:
            raise ValueError("pages and page_tokens must be positive")
        self.pages = pages
        self.page_tokens = page_tokens
        self._holders = [0] * pages
        self._free = list(range(pages))  # a heap: low pages first keeps the pool compact
        self._held: dict[int, _Held] = {}
        self._next_id = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def sequences(self) -> list[int]:
        return list(self._held)

    def _get(self, seq: int) -> _Held:
        try:
            return self._held[seq]
        except KeyError:
            raise KeyError(f"no sequence {seq}") from None

    def length(self, seq: int) -> int:
        return self._get(seq).length

    def pages_of(self, seq: int) -> list[int]:
        return list(self._get(seq).pages)

    def add(self) -> int:
        """A new, empty sequence."""
        seq = self._next_id
        self._next_id += 1
        self._held[seq] = _Held()
        return seq

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens: it shares every page."""
        held = self._get(seq)
        new = self.add()
        self._held[new] = _Held(list(held.pages), held.length)
        for page in held.pages:
            self._holders[page] += 1
        return new

    def free(self, seq: int) -> None:
        """Drop a sequence; pages that nobody else holds are free again."""
        for page in self._get(seq).pages:
            self._drop(page)
        del self._held[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Drop the tokens from `length` on."""
        held, length = self._get(seq), index(length)
        if not 0 <= length <= held.length:
            raise ValueError(f"length must be in [0, {held.length}], got {length}")
        keep = -(-length // self.page_tokens)
        for page in held.pages[keep:]:
            self._drop(page)
        del held.pages[keep:]
        held.length = length

    def grow(self, seqs: Sequence[int], tokens: Sequence[int]) -> list[tuple[int, int]]:
        """Room for tokens[i] more tokens of each sequence; returns the (source, target) page copies due first.

        Raises, and changes nothing, when the free pages do not suffice.
        """
        tokens = [index(n) for n in tokens]
        if len(seqs) != len(tokens):
            raise ValueError(f"{len(seqs)} sequences, {len(tokens)} token counts")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        if any(n < 1 for n in tokens):
            raise ValueError("every sequence needs at least one new token")
        held = [self._get(seq) for seq in seqs]
        need = 0
        holders = {}  # of shared last pages, as the copies below will leave them
        for h, n in zip(held, tokens):
            need += -(-(h.length + n) // self.page_tokens) - len(h.pages)
            if h.length % self.page_tokens and holders.setdefault(h.pages[-1], self._holders[h.pages[-1]]) > 1:
                holders[h.pages[-1]] -= 1
                need += 1
        if need > len(self._free):
            raise RuntimeError(f"the cache is full: {need} pages needed, {len(self._free)} of {self.pages} free")
        copies = []
        for h, n in zip(held, tokens):
            if h.length % self.page_tokens and self._holders[h.pages[-1]] > 1:
                source = h.pages[-1]
                h.pages[-1] = self._take()
                self._holders[source] -= 1
                copies.append((source, h.pages[-1]))
            h.length += n
            while len(h.pages) * self.page_tokens < h.length:
                h.pages.append(self._take())
        return copies

    def compact(self) -> list[tuple[int, int]]:
        """Move every held page to the front of the pool; returns the (source, target) page copies due."""
        live = self.pages - len(self._free)
        holes = [page for page in range(live) if not self._holders[page]]
        moves = dict(zip((page for page in range(live, self.pages) if self._holders[page]), holes))
        for h in self._held.values():
            h.pages = [moves.get(page, page) for page in h.pages]
        for source, target in moves.items():
            self._holders[target], self._holders[source] = self._holders[source], 0
        self._free = list(range(live, self.pages))
        return list(moves.items())

    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._holders[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self._holders[page] -= 1
        if self._holders[page] == 0:
            heapq.heappush(self._free, page)


@dataclass(frozen=True)
class KVBatch:
    """The device-side description of one step: what ``PagedKVCache.plan`` returns."""

    slots: torch.Tensor        # int64 [tokens]: where the new tokens go
    table: torch.Tensor        # int32 [seqs, width]: pages
    lengths: torch.Tensor      # int32 [seqs]: tokens, the new ones included
    query_start: torch.Tensor  # int32 [seqs + 1]: rows of the new tokens
    max_length: int
    max_queries: int
    epoch: int


class PagedKVCache:
    """Keys and values of many sequences and layers in MXFP4 pages.

    One step of a decoder: ``batch = cache.plan(seqs, new_tokens)``, then in
    each layer ``cache.append(layer, k, v, batch)`` and ``cache.attend(layer, q,
    batch)``.  ``fork`` shares pages (the first sequence that writes to a shared
    page gets a copy of it, in all layers), ``truncate`` and ``free`` give them
    back, ``compact`` moves what is held to the front of the pool.  All work is
    ordered on the current stream.  A batch ends with the next plan, fork, free,
    truncate or compact: using it later raises.
    """

    def __init__(self, pages: int, *, kv_heads: int, head_dim: int, layers: int = 1, page_tokens: int = 64,
                 device: torch.device | str = "cuda") -> None:
        if page_tokens not in PAGE_TOKENS or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_tokens must be one of {PAGE_TOKENS} and head_dim one of {HEAD_DIMS}, got {page_tokens} and {head_dim}")
        if kv_heads <= 0 or layers <= 0:
            raise ValueError("kv_heads and layers must be positive")
        self.books = PageBooks(pages, page_tokens)
        shape = (layers, pages, 2, kv_heads, page_tokens)
        self.codes = torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device)
        self.scales = torch.zeros((*shape, head_dim // BLOCK_SIZE), dtype=torch.uint8, device=device)
        self.epoch = 0

    def add(self) -> int:
        """A new, empty sequence."""
        return self.books.add()

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens; pages are shared until one of the two writes."""
        new = self.books.fork(seq)
        self.epoch += 1
        return new

    def free(self, seq: int) -> None:
        """Drop a sequence."""
        self.books.free(seq)
        self.epoch += 1

    def truncate(self, seq: int, length: int) -> None:
        """Drop a sequence's tokens from `length` on (rejected drafts)."""
        self.books.truncate(seq, length)
        self.epoch += 1

    def compact(self) -> int:
        """Move the held pages to the front of the pool; returns how many moved."""
        self.epoch += 1
        return self._copy(self.books.compact())

    def plan(self, seqs: Iterable[int], new_tokens: Iterable[int]) -> KVBatch:
        """Make room for each sequence's new tokens and describe the step to the device.

        Raises RuntimeError, and changes nothing, when the pool is full.
        """
        seqs, new_tokens = list(seqs), [index(n) for n in new_tokens]
        if not seqs:
            raise ValueError("a step needs at least one sequence")
        copies = self.books.grow(seqs, new_tokens)
        self.epoch += 1
        self._copy(copies)
        page = self.books.page_tokens
        held = [self.books.pages_of(seq) for seq in seqs]
        lengths = [self.books.length(seq) for seq in seqs]
        width = max(map(len, held))
        table = torch.zeros((len(seqs), width), dtype=torch.int32)
        slots = []
        for i, (pages, length, n) in enumerate(zip(held, lengths, new_tokens)):
            row = torch.tensor(pages, dtype=torch.int32)
            table[i, : len(pages)] = row
            token = torch.arange(length - n, length)
            slots.append(row[token // page].long() * page + token % page)
        start = torch.zeros(len(seqs) + 1, dtype=torch.int32)
        start[1:] = torch.tensor(new_tokens, dtype=torch.int32).cumsum(0)
        device = self.codes.device
        return KVBatch(torch.cat(slots).to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32).to(device), start.to(device),
                       max(lengths), max(new_tokens), self.epoch)

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, batch: KVBatch) -> None:
        """Write the new tokens' keys and values [tokens, kv_heads, head_dim] of one layer."""
        self._check(batch)
        append_mxfp4_(self.codes[layer], self.scales[layer], key, value, batch.slots)

    def attend(self, layer: int, query: torch.Tensor, batch: KVBatch, *, softmax_scale: float | None = None, window: int = 0) -> torch.Tensor:
        """Causal attention of the new tokens' queries [tokens, heads, head_dim] over one layer."""
        self._check(batch)
        return paged_attention_mxfp4(query, self.codes[layer], self.scales[layer], batch.table, batch.lengths, batch.query_start,
                                     max_length=batch.max_length, max_queries=batch.max_queries, softmax_scale=softmax_scale, window=window)

    def gather(self, layer: int, seq: int, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """A sequence's keys and values of one layer, each [length, kv_heads, head_dim] of `dtype`."""
        page = self.books.page_tokens
        token = torch.arange(self.books.length(seq))
        slots = torch.tensor(self.books.pages_of(seq), dtype=torch.int64)[token // page] * page + token % page
        return gather_mxfp4(self.codes[layer], self.scales[layer], slots.to(self.codes.device), dtype)

    def _check(self, batch: KVBatch) -> None:
        if batch.epoch != self.epoch:
            raise ValueError("this batch was planned before another plan, fork, free, truncate or compact: plan the step again")

    def _copy(self, copies: list[tuple[int, int]]) -> int:
        if copies:
            # A page may go to several targets, and no target is a source: see grow and compact.
            copy_pages_(self.codes, self.scales, [s for s, _ in copies], [t for _, t in copies])
        return len(copies)


__all__ = ["HEAD_DIMS", "PAGE_TOKENS", "KVBatch", "PageBooks", "PagedKVCache", "append_mxfp4_", "copy_pages_", "gather_mxfp4",
           "paged_attention_mxfp4"]
