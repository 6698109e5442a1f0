"""Calls of the serving operators that the ordinary path must not take as they come: recorded, transformed and
unusually bounded ones."""

from __future__ import annotations

import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from mxwave_b200 import _lib, kvcache, ops
from mxwave_b200.core import quantize_mxfp4
from mxwave_b200.linear import linear_mxfp4

BF, HF = torch.bfloat16, torch.float16


def _watchers():
    """Ways to run f(t) under something that records or transforms its operators."""
    return {
        "jit": lambda f, t: torch.jit.trace(f, (t,), check_trace=False),
        "pre-dispatch": lambda f, t: make_fx(f, pre_dispatch=True)(t),
        "dispatch": lambda f, t: make_fx(f)(t),
        "vmap": lambda f, t: torch.vmap(f)(t),
        "functionalize": lambda f, t: torch.func.functionalize(f)(t),
    }


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def _pool(g: torch.Generator, lengths: list[int], heads: int = 2, page: int = 16, dim: int = 64):
    """codes, scales, table, lengths of sequences of random rows."""
    need = [-(-n // page) for n in lengths]
    shape = (sum(need) + 1, 2, heads, page)
    codes = torch.zeros(*shape, dim // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(*shape, dim // 32, dtype=torch.uint8, device="cuda")
    rows = shape[0] * page
    kvcache.append_mxfp4_(codes, scales, _randn(g, rows, heads, dim), _randn(g, rows, heads, dim), torch.arange(rows, device="cuda"))
    table = torch.zeros(len(lengths), max(need), dtype=torch.int32, device="cuda")
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n)
    return codes, scales, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("name", sorted(_watchers()))
def test_what_watches_is_noticed(name: str) -> None:
    found = []

    def f(t: torch.Tensor) -> torch.Tensor:
        found.append(ops.plain_eager(t))
        return t + 1

    assert ops.plain_eager(torch.ones(3))
    with torch.inference_mode():
        assert ops.plain_eager(torch.ones(3))
    with torch.autocast("cpu", dtype=BF):
        assert ops.plain_eager(torch.ones(3))
    _watchers()[name](f, torch.ones(3))
    assert found and not any(found)
    assert ops.plain_eager(torch.ones(3))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["jit", "pre-dispatch", "dispatch"])
def test_recorded_calls_run_the_operators(name: str) -> None:
    g = _gen(1)
    packed, scales = quantize_mxfp4(_randn(g, 96, 64), method="rtn")
    pool = _pool(g, [40, 3])
    start = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")

    def product(x: torch.Tensor) -> torch.Tensor:
        return linear_mxfp4(x, packed, scales, activation="silu", residual=x[:, :1].expand(-1, 96))

    def attention(q: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return kvcache.paged_attention_mxfp4(q, *pool, start, max_length=40, max_queries=2, return_lse=True)

    def rows(r: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        codes, sc = torch.zeros_like(pool[0]), torch.zeros_like(pool[1])
        slots = torch.arange(5, device="cuda")
        kvcache.append_mxfp4_(codes, sc, r, r + 1, slots)
        kvcache.copy_pages_(codes[None], sc[None], torch.tensor([0]), torch.tensor([2]))
        return kvcache.gather_mxfp4(codes, sc, slots + 32, torch.float32)

    for f, shape in ((product, (5, 64)), (attention, (3, 4, 64)), (rows, (5, 2, 64))):
        first, other = _randn(g, *shape).to(BF), _randn(g, *shape).to(BF)
        graph = _watchers()[name](f, first)
        for t in (other, first):
            torch.empty(1 << 20, device="cuda").fill_(float("nan"))  # what an unwritten output would be made of
            got, want = graph(t), f(t)
            for a, b in zip((got,) if torch.is_tensor(got) else got, (want,) if torch.is_tensor(want) else want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_vmap_runs_slice_by_slice() -> None:
    g = _gen(2)
    packed, scales = quantize_mxfp4(_randn(g, 96, 64), method="rtn")
    x = _randn(g, 4, 5, 64).to(BF)
    got = torch.vmap(lambda t: linear_mxfp4(t, packed, scales))(x)
    assert torch.equal(got, torch.stack([linear_mxfp4(t, packed, scales) for t in x]))
    pool = _pool(g, [40, 3])
    start = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    q = _randn(g, 4, 3, 4, 64).to(BF)
    attend = lambda t: kvcache.paged_attention_mxfp4(t, *pool, start, max_length=40, max_queries=2)  # noqa: E731
    assert torch.equal(torch.vmap(attend)(q), torch.stack([attend(t) for t in q]))


@pytest.mark.parametrize("lengths", [100, 5000])
def test_a_bound_of_no_queries_sizes_the_launch_for_one(lengths: int) -> None:
    lib = _lib.load()
    assert lib.mxw_paged_attention_workspace_size(2, 8, 2, 64, lengths, 0) == lib.mxw_paged_attention_workspace_size(2, 8, 2, 64, lengths, 1) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [[1, 1], [3, 0], [90, 40], [0, 0]])
def test_a_bound_of_no_queries_costs_speed_only(queries: list[int], monkeypatch) -> None:
    g = _gen(3)
    codes, scales, table, lengths = _pool(g, [200, 77])
    start = torch.tensor([0, queries[0], sum(queries)], dtype=torch.int32, device="cuda")
    q = _randn(g, sum(queries) + 2, 4, 64).to(BF)
    run = lambda most: kvcache.paged_attention_mxfp4(q, codes, scales, table, lengths, start, max_length=200, max_queries=most,  # noqa: E731
                                                     return_lse=True)
    want = run(1)
    assert (want[0][: sum(queries)] != 0).any() == (sum(queries) > 0)
    for _ in range(2):
        out, lse = run(0)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert (out[sum(queries) :] == 0).all() and (lse[sum(queries) :] == -math.inf).all()
        monkeypatch.setattr(ops, "binding", None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("length, queries", [(40, 1), (3000, 3), (300, 150)])
@pytest.mark.parametrize("wide", [False, True])
def test_an_infinite_query_gives_nan(dtype: torch.dtype, length: int, queries: int, wide: bool) -> None:
    """Also where the infinity makes every score -infinity; rows that no key reaches stay zero."""
    g = _gen(4)
    codes, scales, table, lengths = _pool(g, [length, length], heads=16)
    codes[:, 0, ..., 0] = 0xAA  # the first two channels of every key: -1 times the scale
    if wide:
        scales[:, 1, ..., 3, :] = 20  # values far smaller than the others
    lengths[1] = 0
    start = torch.tensor([0, queries, 2 * queries], dtype=torch.int32, device="cuda")
    q = _randn(g, 2 * queries, 16, 64).to(dtype)
    run = lambda: kvcache.paged_attention_mxfp4(q, codes, scales, table, lengths, start, max_length=length, max_queries=queries,  # noqa: E731
                                                return_lse=True)
    clean, _ = run()
    bad = torch.zeros(2 * queries, 16, dtype=torch.bool, device="cuda")
    for row, head, value in ((0, 0, math.inf), (queries - 1, 3, -math.inf), (queries, 5, math.inf)):
        q[row, head, 0] = value
        bad[row, head] = True
    out, lse = run()
    assert out[:queries][bad[:queries]].isnan().all() and lse[:queries][bad[:queries]].isnan().all()
    assert torch.equal(out[~bad], clean[~bad])
    assert (out[queries:] == 0).all() and (lse[queries:] == -math.inf).all()


@pytest.mark.gpu
def test_forward_mode_gradients_are_refused() -> None:
    import torch.autograd.forward_ad as forward

    g = _gen(5)
    packed, scales = quantize_mxfp4(_randn(g, 32, 64), method="rtn")
    pool = _pool(g, [20])
    start = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    x, bias, q = _randn(g, 2, 64).to(BF), _randn(g, 32).to(BF), _randn(g, 2, 4, 64).to(BF)
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: linear_mxfp4(dual(x), packed, scales), lambda: linear_mxfp4(x, packed, scales, dual(bias)),
                     lambda: linear_mxfp4(x, packed, scales, residual=dual(x[:, :32])),
                     lambda: kvcache.paged_attention_mxfp4(dual(q), *pool, start, max_length=20, max_queries=2)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        assert linear_mxfp4(x, packed, scales, bias).isfinite().all()  # nothing asks for one here


@pytest.mark.parametrize("source, target, error", [
    ([0.5], [1], TypeError), ([0], [1.9], TypeError), (["0"], [1], TypeError), (torch.tensor([0.0]), [1], ValueError),
    ([0], torch.tensor([True]), ValueError),
])
def test_page_numbers_are_whole(source, target, error: type) -> None:
    codes, scales = torch.zeros(2, 4, 2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 4, 2, 1, 16, 2, dtype=torch.uint8)
    with pytest.raises(error):
        kvcache.copy_pages_(codes, scales, source, target)


def test_token_counts_are_whole() -> None:
    cache = kvcache.PagedKVCache(8, kv_heads=1, head_dim=64, page_tokens=16, device="cpu")
    seq = cache.add()
    with pytest.raises(TypeError):
        cache.plan([seq], [1.9])
    with pytest.raises(TypeError):
        cache.books.grow([seq], [1.9])
    with pytest.raises(TypeError):
        cache.truncate(seq, 0.0)
    assert cache.books.length(seq) == 0 and cache.plan([seq], torch.tensor([2])).lengths.tolist() == [2]


def test_the_library_builds_without_the_binding(tmp_path: Path) -> None:
    """Users of the C ABI alone need no torch headers: `make` ends well without the host binding, `make binding` says so."""
    root = Path(__file__).resolve().parents[1]
    shutil.copytree(root / "mxwave_b200" / "csrc", tmp_path / "mxwave_b200" / "csrc")
    shutil.copytree(root / "include", tmp_path / "include")
    make = ["make", "-C", str(tmp_path / "mxwave_b200" / "csrc"), "NVCC=true", "CXX=false", "PYTHON=false"]
    done = subprocess.run(make, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert "built ../_native/libmxwave_b200.so" in done.stdout and "torch's headers" in done.stdout
    assert subprocess.run([*make, "binding"], capture_output=True).returncode != 0
