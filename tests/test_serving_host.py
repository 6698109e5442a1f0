"""CPU tests of the serving operators' host side: refusals by the public
functions and by the C ABI (no launch happens), schemas and fake shapes."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mxwave_b200 import _lib, kvcache, ops  # noqa: F401  -- registers the operators
from mxwave_b200.linear import linear_mxfp4

BF = torch.bfloat16


def _linear_args(rows: int = 2, outs: int = 4, inner: int = 64):
    return torch.zeros(rows, inner, dtype=BF), torch.zeros(outs, inner // 2, dtype=torch.uint8), torch.zeros(outs, inner // 32, dtype=torch.uint8)


@pytest.mark.parametrize("change, error", [
    (dict(), RuntimeError),  # a CPU tensor: there is no fallback
    (dict(activation="tanh"), ValueError),
    (dict(x=torch.zeros(2, 48, dtype=BF)), ValueError),
    (dict(x=torch.zeros(2, 96, dtype=BF)), ValueError),
    (dict(x=torch.zeros(2, 64)), ValueError),
    (dict(packed=torch.zeros(4, 32, dtype=torch.int8)), ValueError),
    (dict(scales=torch.zeros(4, 3, dtype=torch.uint8)), ValueError),
])
def test_linear_refuses(change: dict, error: type) -> None:
    x, packed, scales = _linear_args()
    kw = dict(x=x, packed=packed, scales=scales)
    kw.update(change)
    with pytest.raises(error):
        linear_mxfp4(**kw)


def _pool(pages: int = 4, heads: int = 2, page: int = 16, dim: int = 64, layers: int | None = None):
    lead = () if layers is None else (layers,)
    shape = (*lead, pages, 2, heads, page)
    return torch.zeros(*shape, dim // 2, dtype=torch.uint8), torch.zeros(*shape, dim // 32, dtype=torch.uint8)


def test_cache_functions_refuse_cpu_tensors() -> None:
    codes, scales = _pool()
    rows = torch.zeros(3, 2, 64, dtype=BF)
    slots = torch.arange(3)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        kvcache.append_mxfp4_(codes, scales, rows, rows, slots)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        kvcache.gather_mxfp4(codes, scales, slots)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        kvcache.copy_pages_(*_pool(layers=2), [0], [1])
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        kvcache.paged_attention_mxfp4(rows, codes, scales, i32[None], i32, torch.zeros(2, dtype=torch.int32), max_length=1, max_queries=1)


@pytest.mark.parametrize("codes, scales", [
    (_pool(page=8)[0], _pool(page=8)[1]),
    (_pool(dim=32)[0], _pool(dim=32)[1]),
    (_pool()[0], _pool(dim=128)[1]),
    (_pool()[0].float(), _pool()[1]),
    (_pool(layers=2)[0], _pool(layers=2)[1]),
])
def test_pool_shapes_are_checked(codes: torch.Tensor, scales: torch.Tensor) -> None:
    with pytest.raises(ValueError):
        kvcache.gather_mxfp4(codes, scales, torch.arange(2))


def test_cache_refuses_odd_pages_and_heads() -> None:
    for kw in (dict(page_tokens=48, head_dim=64, kv_heads=1), dict(page_tokens=64, head_dim=96, kv_heads=1),
               dict(page_tokens=64, head_dim=64, kv_heads=0)):
        with pytest.raises(ValueError):
            kvcache.PagedKVCache(4, device="cpu", **kw)


def test_batches_end_with_the_next_change() -> None:
    cache = kvcache.PagedKVCache(8, kv_heads=1, head_dim=64, page_tokens=16, device="cpu")
    a = cache.add()
    batch = cache.plan([a], [20])
    assert batch.slots.tolist() == list(range(20)) and batch.table.tolist() == [[0, 1]]
    assert batch.lengths.tolist() == [20] and batch.query_start.tolist() == [0, 20]
    assert (batch.max_length, batch.max_queries) == (20, 20)
    q = torch.zeros(20, 1, 64, dtype=BF)
    for change in (lambda: cache.plan([a], [1]), lambda: cache.fork(a), lambda: cache.truncate(a, 16), lambda: cache.compact()):
        batch = cache.plan([a], [12]) if cache.books.length(a) % 16 == 4 else cache.plan([a], [4])
        change()
        with pytest.raises(ValueError, match="plan the step again"):
            cache.attend(0, q, batch)
        for seq in cache.books.sequences:
            if seq != a:
                cache.books.free(seq)
    with pytest.raises(ValueError):
        cache.plan([], [])


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    return _lib.load()


P16 = ctypes.c_void_p(16)


@pytest.mark.parametrize("kw", [
    dict(inner=48), dict(dtype=_lib.MXW_F32), dict(act=9), dict(ldx=32), dict(ldr=2, residual=P16), dict(ws=0), dict(packed=ctypes.c_void_p(24)),
    dict(packed=None), dict(rows=-1),
])
def test_linear_abi_refuses(lib: ctypes.CDLL, kw: dict) -> None:
    rows, inner = kw.get("rows", 40), kw.get("inner", 64)
    need = lib.mxw_linear_workspace_size(40, 64, _lib.MXW_BF16)
    assert need > 0
    status = lib.mxw_linear_mxfp4(P16, kw.get("dtype", _lib.MXW_BF16), rows, inner, kw.get("ldx", inner), kw.get("packed", P16), P16, 4, None,
                                  kw.get("act", 0), kw.get("residual"), kw.get("ldr", 4), P16, P16, kw.get("ws", need), None, None)
    assert status == _lib.MXW_EINVAL


def test_linear_abi_empty_is_a_no_op(lib: ctypes.CDLL) -> None:
    assert lib.mxw_linear_mxfp4(None, 0, 0, 64, 64, None, None, 4, None, 0, None, 0, None, None, 0, None, None) == _lib.MXW_OK
    assert lib.mxw_linear_mxfp4(None, 0, 3, 64, 64, None, None, 0, None, 0, None, 0, None, None, 0, None, None) == _lib.MXW_OK


def _pages(values: list[int]):
    return (ctypes.c_int64 * len(values))(*values)


@pytest.mark.parametrize("source, target", [
    ([0, 1], [2, 2]),  # a target twice
    ([0, 2], [2, 3]),  # a target that is a source
    ([1], [1]),
    ([4], [0]),
    ([0], [4]),
    ([-1], [0]),
])
def test_copy_pages_abi_refuses(lib: ctypes.CDLL, source: list[int], target: list[int]) -> None:
    assert lib.mxw_copy_pages(P16, P16, 2, 4, 1024, 64, _pages(source), _pages(target), len(source), None) == _lib.MXW_EINVAL


def test_copy_pages_abi_checks_sizes(lib: ctypes.CDLL) -> None:
    assert lib.mxw_copy_pages(P16, P16, 2, 4, 1000, 64, _pages([0]), _pages([1]), 1, None) == _lib.MXW_EINVAL
    assert lib.mxw_copy_pages(ctypes.c_void_p(8), P16, 2, 4, 1024, 64, _pages([0]), _pages([1]), 1, None) == _lib.MXW_EINVAL
    assert lib.mxw_copy_pages(P16, P16, 2, 4, 1024, 64, _pages([]), _pages([]), 0, None) == _lib.MXW_OK


@pytest.mark.parametrize("kw", [
    dict(dim=96), dict(page=48), dict(heads=3, kv=2), dict(window=5, causal=0), dict(scale=0.0), dict(scale=float("nan")), dict(ld=1, width=2),
    dict(dtype=_lib.MXW_F32), dict(ws=0), dict(window=-1),
])
def test_attention_abi_refuses(lib: ctypes.CDLL, kw: dict) -> None:
    heads, kv, dim = kw.get("heads", 4), kw.get("kv", 2), kw.get("dim", 64)
    need = lib.mxw_paged_attention_workspace_size(2, 4, 2, 64, 100, 1)
    assert need > 0
    status = lib.mxw_paged_attention(P16, kw.get("dtype", _lib.MXW_BF16), 2, heads, heads * dim, dim, P16, P16, 8, kv, kw.get("page", 16), dim, P16,
                                     kw.get("ld", 8), kw.get("width", 8), P16, P16, 2, 100, 1, kw.get("scale", 0.1), kw.get("causal", 1),
                                     kw.get("window", 0), P16, None, P16, kw.get("ws", need), None, None)
    assert status == _lib.MXW_EINVAL


@pytest.mark.parametrize("kw", [dict(dim=96), dict(page=48), dict(heads=0), dict(dtype=5), dict(stride=-1)])
def test_append_and_gather_abi_refuse(lib: ctypes.CDLL, kw: dict) -> None:
    heads, page, dim, dtype = kw.get("heads", 2), kw.get("page", 16), kw.get("dim", 64), kw.get("dtype", _lib.MXW_BF16)
    stride = kw.get("stride", 128)
    assert lib.mxw_kv_append(P16, P16, 4, heads, page, dim, P16, P16, dtype, stride, 64, 128, 64, P16, 3, None) == _lib.MXW_EINVAL
    if "stride" not in kw:
        assert lib.mxw_kv_gather(P16, P16, 4, heads, page, dim, P16, 3, dtype, P16, P16, None) == _lib.MXW_EINVAL


def test_fake_shapes() -> None:
    with FakeTensorMode():
        x = torch.empty(3, 64, dtype=BF, device="cuda")
        w, s = torch.empty(10, 32, dtype=torch.uint8, device="cuda"), torch.empty(10, 2, dtype=torch.uint8, device="cuda")
        assert torch.ops.mxwave_b200.linear_mxfp4(x, w, s, None, None, 0).shape == (3, 10)
        assert linear_mxfp4(x[None], w, s).shape == (1, 3, 10)
        codes = torch.empty(4, 2, 2, 16, 32, dtype=torch.uint8, device="cuda")
        scales = torch.empty(4, 2, 2, 16, 2, dtype=torch.uint8, device="cuda")
        k, v = kvcache.gather_mxfp4(codes, scales, torch.empty(5, dtype=torch.int64, device="cuda"), torch.float32)
        assert k.shape == v.shape == (5, 2, 64) and k.dtype == torch.float32
        i32 = torch.empty(3, dtype=torch.int32, device="cuda")
        q = torch.empty(6, 4, 64, dtype=torch.float16, device="cuda")
        out, lse = kvcache.paged_attention_mxfp4(q, codes, scales, torch.empty(3, 4, dtype=torch.int32, device="cuda"), i32,
                                                 torch.empty(4, dtype=torch.int32, device="cuda"), max_length=9, max_queries=2, return_lse=True)
        assert out.shape == q.shape and out.dtype == torch.float16 and lse.shape == (6, 4) and lse.dtype == torch.float32
