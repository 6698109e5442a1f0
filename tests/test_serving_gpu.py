"""The serving operators on a B200 against plain 64-bit implementations:
products with MXFP4 weights, the paged MXFP4 cache, and attention over it.

Tolerances are derived, not fitted.  With u(t) = eps(t) / 2 the half step of a
type (bf16 2^-8, f16 2^-11, fp32 2^-24, relative to the value):

* a product's output is the exact sum S = sum x w plus fp32 additions -- one per
  32 inputs and term, each off by at most a step 2^-23 of the running sum (the
  tensor cores may truncate), so (3 K / 32 + 16) (2^-23 sum |x w| + 2^-149) -- plus the part
  of x below E4M3's subnormals, 2^-22 of its block's largest; the activation
  passes an error on by at most 1.2 (the steepest slope of silu and gelu) and
  adds a few fp32 steps; one rounding to the output type at the end;
* attention's probabilities are rounded to f16 (2^-11) and its scores are off by
  d = scale sum |q k| (D + 16) 2^-23 at most, which moves each probability by
  the factor e^d, and the sum of probabilities likewise; values below 2^-27 of
  the largest scale are dropped.
"""

from __future__ import annotations

import math

import pytest
import torch

from mxwave_b200 import kvcache, ops
from mxwave_b200.core import dequant_mxfp4, quantize_mxfp4
from mxwave_b200.linear import linear_mxfp4

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
LUT = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device="cuda")


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def values64(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    lut = torch.tensor(LUT + tuple(-v for v in LUT), dtype=torch.float64, device=codes.device)
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


# ----------------------------------------------------------------------- linear


def act64(y: torch.Tensor, name: str) -> torch.Tensor:
    return {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[name](y)


def check_linear(x, packed, scales, bias, act, residual, got) -> None:
    w, xd = values64(packed, scales), x.double()
    want = xd @ w.T + (0 if bias is None else bias.double())
    k = x.shape[-1]
    mass = xd.abs() @ w.abs().T + (0 if bias is None else bias.double().abs())
    tops = xd.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1) @ w.abs().T
    # An addition's step is 2^-23 of the sum, but never less than fp32's smallest number, 2^-149.
    err = 1.2 * ((3 * k / 32 + 16) * (2.0**-23 * mass + 2.0**-149) + 2.0**-22 * tops)
    want = act64(want, act)
    err = err + 2.0**-21 * want.abs()
    if residual is not None:
        want = want + residual.double()
        err = err + 2.0**-23 * want.abs()
    # A rounding's half step is relative to the value rounded; below the normal range it is that of the smallest normal.
    tol = err + half_step(x.dtype) * (want.abs() + err).clamp_min(torch.finfo(x.dtype).tiny)
    assert got.dtype == x.dtype and got.shape == want.shape
    assert ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())


SHAPES = [(1, 1, 32), (1, 130, 96), (2, 256, 512), (7, 64, 160), (8, 257, 2080), (16, 384, 5120), (17, 100, 544), (33, 129, 256), (64, 200, 1024),
          (65, 500, 224), (128, 128, 128), (129, 300, 640), (333, 1000, 2080), (700, 4100, 192), (1300, 2304, 448)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows, outs, inner", SHAPES)
def test_linear_matches_64_bits(rows: int, outs: int, inner: int, dtype: torch.dtype) -> None:
    g = gen(rows * 7 + outs)
    packed, scales = quantize_mxfp4(randn(g, outs, inner) * 0.02, method="rtn")
    x = (randn(g, rows, inner) * torch.exp(randn(g, inner))).to(dtype)
    bias, residual = randn(g, outs).to(dtype), randn(g, rows, outs).to(dtype)
    check_linear(x, packed, scales, None, "none", None, linear_mxfp4(x, packed, scales))
    for act, b, r in (("silu", None, residual), ("gelu", bias, None), ("relu", bias, residual)):
        check_linear(x, packed, scales, b, act, r, linear_mxfp4(x, packed, scales, b, activation=act, residual=r))


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 24, 100, 300])
@pytest.mark.parametrize("outs, inner", [(9472, 5120), (2048, 17408)])
def test_linear_over_long_rows(rows: int, outs: int, inner: int) -> None:
    """Rows of many stages, more blocks than SMs, weights not in the caches: every ring of stages wraps while loads are slow."""
    g = gen(rows)
    x = randn(g, rows, inner).to(BF)
    weights = [quantize_mxfp4(randn(g, outs, inner) * 0.02, method="rtn") for _ in range(4)]
    got = [linear_mxfp4(x, p, s) for p, s in weights]
    for (p, s), y in zip(weights, got):
        check_linear(x, p, s, None, "none", None, y)


@pytest.mark.parametrize("rows", [4, 20, 50, 200])
@pytest.mark.parametrize("outs, inner", [(100, 96), (100, 640), (4780, 1184), (2310, 1184), (3480, 1184), (100, 1184), (100, 2080), (100, 4064)])
def test_linear_shares_of_the_inputs(rows: int, outs: int, inner: int) -> None:
    """Clusters of one to eight blocks, with shares of the inputs that are not equal and end in the middle of a chunk."""
    g = gen(rows + outs + inner)
    packed, scales = quantize_mxfp4(randn(g, outs, inner) * 0.02, method="rtn")
    x, bias, residual = randn(g, rows, inner).to(HF), randn(g, outs).to(HF), randn(g, rows, outs).to(HF)
    y = linear_mxfp4(x, packed, scales, bias, activation="silu", residual=residual)
    check_linear(x, packed, scales, bias, "silu", residual, y)
    assert torch.equal(y, linear_mxfp4(x, packed, scales, bias, activation="silu", residual=residual))


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_linear_takes_strides_slices_and_leading_dims(rows: int) -> None:
    g = gen(rows)
    outs, inner = 260, 288
    packed, scales = quantize_mxfp4(randn(g, outs + 1, inner), method="rtn")
    packed, scales = packed[1:], scales[1:]  # starts inside a 16-byte line
    wide = randn(g, rows, 2 * inner + 3).to(BF)
    res = randn(g, rows, outs + 5).to(BF)
    for x, r in ((wide[:, 3 : 3 + inner], res[:, 5:]), (wide[:, :inner], res[:, 1 : 1 + outs]), (wide[:, ::2][:, :inner], res[:, :outs])):
        check_linear(x, packed, scales, None, "none", r, linear_mxfp4(x, packed, scales, residual=r))
    x3 = randn(g, rows, 1, inner).to(BF)
    got = linear_mxfp4(x3, packed, scales)
    assert got.shape == (rows, 1, outs)
    check_linear(x3[:, 0], packed, scales, None, "none", None, got[:, 0])
    assert linear_mxfp4(x3[:0], packed, scales).shape == (0, 1, outs)
    vec = linear_mxfp4(x3[0, 0], packed, scales)
    assert vec.shape == (outs,)
    check_linear(x3[:1, 0], packed, scales, None, "none", None, vec[None])


@pytest.mark.parametrize("rows", [2, 50, 400])
def test_linear_over_the_range_of_scales(rows: int) -> None:
    """Scale bytes and inputs far from 1: 2^-60 to 2^60, and inputs that span 2^-14 of a block's largest."""
    g = gen(5)
    outs, inner = 128 * 40, 256
    packed = torch.randint(0, 256, (outs, inner // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(67, 188, (outs, 1), generator=g, device="cuda", dtype=torch.uint8).expand(outs, inner // 32).contiguous()
    x = (randn(g, rows, inner) * torch.exp2(-14 * torch.rand(rows, inner, generator=g, device="cuda"))).to(BF)
    check_linear(x, packed, scales, None, "none", None, linear_mxfp4(x, packed, scales))
    check_linear(x * 2.0**-100, packed, scales, None, "none", None, linear_mxfp4(x * 2.0**-100, packed, scales))


@pytest.mark.parametrize("rows", [4, 40, 600])
def test_linear_non_finite_rows_stay_their_own(rows: int) -> None:
    g = gen(6)
    outs, inner = 1200, 192
    packed, scales = quantize_mxfp4(randn(g, outs, inner), method="rtn")
    x = randn(g, rows, inner).to(BF)
    clean = linear_mxfp4(x, packed, scales)
    x[1, 5], x[3, 100] = float("inf"), float("nan")
    got = linear_mxfp4(x, packed, scales)
    assert got[1].isnan().all() and got[3].isnan().all()
    keep = torch.arange(rows, device="cuda")
    keep = keep[(keep != 1) & (keep != 3)]
    assert torch.equal(got[keep], clean[keep])


def test_linear_zero_and_repeated_calls() -> None:
    g = gen(7)
    packed, scales = quantize_mxfp4(randn(g, 3000, 512), method="rtn")
    for rows in (1, 30, 100, 900):
        x = randn(g, rows, 512).to(BF)
        first = linear_mxfp4(x, packed, scales, activation="silu")
        assert all(torch.equal(first, linear_mxfp4(x, packed, scales, activation="silu")) for _ in range(3))
        assert (linear_mxfp4(torch.zeros_like(x), packed, scales) == 0).all()


def test_linear_refuses_gradients_and_mixed_types() -> None:
    packed, scales = quantize_mxfp4(torch.ones(8, 64, device="cuda"), method="rtn")
    x = torch.ones(2, 64, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_mxfp4(x.requires_grad_(), packed, scales)
    with torch.no_grad():
        linear_mxfp4(x, packed, scales)
    x = x.detach()
    with pytest.raises(ValueError, match="bias"):
        linear_mxfp4(x, packed, scales, torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError, match="residual"):
        linear_mxfp4(x, packed, scales, residual=torch.zeros(2, 9, dtype=BF, device="cuda"))
    with pytest.raises(ValueError, match="is on"):
        linear_mxfp4(x, packed.cpu(), scales)


# ------------------------------------------------------------------------ cache


def pool(pages: int, heads: int, page: int, dim: int, fill: int = 0):
    codes = torch.full((pages, 2, heads, page, dim // 2), fill, dtype=torch.uint8, device="cuda")
    scales = torch.full((pages, 2, heads, page, dim // 32), fill, dtype=torch.uint8, device="cuda")
    return codes, scales


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("tokens, heads, page, dim, strided", [
    (1, 1, 16, 64, False), (5, 3, 16, 128, True), (64, 8, 64, 128, False), (70, 5, 32, 128, True), (33, 17, 128, 64, False), (300, 2, 16, 64, True)])
def test_append_writes_what_quantize_writes(tokens: int, heads: int, page: int, dim: int, strided: bool, dtype: torch.dtype) -> None:
    g = gen(tokens)
    pages = -(-tokens // page) + 2
    codes, scales = pool(pages, heads, page, dim, fill=0xA5)
    both = (randn(g, tokens, 3 * heads, dim + (3 if strided else 0)) * torch.exp(3 * randn(g, tokens, 1, 1))).to(dtype)[..., :dim]
    both[0, :, 0] = 0
    both[0, 0, :32] = 0  # a zero block
    key, value = both[:, :heads], both[:, -heads:]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 3:
        slots[1], slots[2] = -1, pages * page  # padding, and a slot past the pool
    kvcache.append_mxfp4_(codes, scales, key, value, slots)
    kept = (slots >= 0) & (slots < pages * page)
    at, off = slots[kept] // page, slots[kept] % page
    for part, rows in ((0, key), (1, value)):
        p, s = quantize_mxfp4(rows[kept].reshape(-1, dim).contiguous(), method="rtn")
        assert torch.equal(codes[at, part, :, off], p.view(-1, heads, dim // 2))
        assert torch.equal(scales[at, part, :, off], s.view(-1, heads, dim // 32))
    untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    untouched[at, off] = False
    assert (codes.permute(0, 3, 1, 2, 4)[untouched] == 0xA5).all() and (scales.permute(0, 3, 1, 2, 4)[untouched] == 0xA5).all()
    for out in (BF, F32, HF):
        got = kvcache.gather_mxfp4(codes, scales, slots, out)
        for part, rows in enumerate(got):
            want = values64(codes[at, part, :, off], scales[at, part, :, off])
            assert torch.equal(rows[kept], want.to(out)) and (rows[~kept] == 0).all()


def test_append_non_finite_rows_match_quantize() -> None:
    rows = torch.randn(6, 1, 64, device="cuda")
    rows[0, 0, 3], rows[1, 0, 40], rows[2, 0, 0], rows[3, 0, 33] = float("nan"), float("inf"), float("-inf"), -float("nan")
    rows[4] = 3.0e38
    rows[5] = 1.0e-42
    codes, scales = pool(1, 1, 16, 64)
    kvcache.append_mxfp4_(codes, scales, rows, rows, torch.arange(6, device="cuda"))
    p, s = quantize_mxfp4(rows[:, 0], method="rtn")
    for part in (0, 1):
        assert torch.equal(codes[0, part, 0, :6], p) and torch.equal(scales[0, part, 0, :6], s)


def test_gather_agrees_with_dequant() -> None:
    g = gen(11)
    codes, scales = pool(4, 2, 16, 128)
    rows = randn(g, 64, 2, 128)
    kvcache.append_mxfp4_(codes, scales, rows, -rows, torch.arange(64, device="cuda"))
    k, v = kvcache.gather_mxfp4(codes, scales, torch.arange(64, device="cuda"), F32)
    p, s = quantize_mxfp4(rows.reshape(-1, 128), method="rtn")
    assert torch.equal(k.reshape(-1, 128), dequant_mxfp4(p, s, (128, 128)))
    assert torch.equal(v, -k)


@pytest.mark.parametrize("layers, pages, moves, heads, page, dim", [(1, 4, 1, 1, 16, 64), (3, 130, 65, 3, 16, 128), (2, 4500, 2100, 1, 16, 64),
                                                                   (2, 40, 20, 8, 128, 128)])
def test_copy_pages(layers: int, pages: int, moves: int, heads: int, page: int, dim: int) -> None:
    g = gen(pages)
    codes = torch.randint(0, 256, (layers, pages, 2, heads, page, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(0, 256, (layers, pages, 2, heads, page, dim // 32), generator=g, device="cuda", dtype=torch.uint8)
    order = torch.randperm(pages)
    source, target = order[:moves], order[-moves:]
    source[0] = source[-1]  # one page to two targets
    want = codes.clone(), scales.clone()
    for w in want:
        w[:, target.cuda()] = w[:, source.cuda()]
    kvcache.copy_pages_(codes, scales, source, target.tolist())
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    with pytest.raises(ValueError):
        kvcache.copy_pages_(codes, scales, [0, 1], [2, 2])
    with pytest.raises(ValueError):
        kvcache.copy_pages_(codes, scales, [0], [pages])
    assert torch.equal(codes, want[0])


# -------------------------------------------------------------------- attention


class Case:
    """Sequences over a pool of random pages; unwritten rows hold arbitrary bytes."""

    def __init__(self, seed: int, lens: list[int], queries: list[int], heads: int, kv: int, page: int, dim: int, dtype: torch.dtype, behind: int = 0):
        g = gen(seed)
        self.lens, self.queries, self.page, self.kv, self.dim = lens, queries, page, kv, dim
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        shape = (pages, 2, kv, page)
        self.codes = torch.randint(0, 256, (*shape, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
        self.scales = torch.randint(0, 256, (*shape, dim // 32), generator=g, device="cuda", dtype=torch.uint8)  # stale rows: anything
        self.table = torch.full((len(lens), max([1, *need])), 0x7FFFFFF0, dtype=torch.int32, device="cuda")  # unused entries: anything
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        first = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[first : first + n]
            if lens[b]:
                rows = randn(g, lens[b], kv, dim) * (1 + 9 * (torch.rand(kv, dim, generator=g, device="cuda") < 0.05))
                token = torch.arange(lens[b], device="cuda")
                slots = order[first + token // page].long() * page + token % page
                kvcache.append_mxfp4_(self.codes, self.scales, rows, randn(g, lens[b], kv, dim), slots)
            first += n
        total = sum(queries)
        self.query = randn(g, total + behind, heads, dim).to(dtype)
        start = [0]
        for q in queries:
            start.append(start[-1] + q)
        self.start = torch.tensor(start, dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def run(self, query: torch.Tensor | None = None, **kw):
        kw = {"max_length": max(self.lens), "max_queries": max(self.queries), "return_lse": True, **kw}
        return kvcache.paged_attention_mxfp4(self.query if query is None else query, self.codes, self.scales, self.table, self.lengths, self.start, **kw)

    def check(self, out: torch.Tensor, lse: torch.Tensor, *, softmax_scale: float | None = None, causal: bool = True, window: int = 0,
              dead: frozenset = frozenset()) -> None:
        scale = self.dim**-0.5 if softmax_scale is None else softmax_scale
        group = self.query.shape[1] // self.kv
        first = 0
        for b, (n, q) in enumerate(zip(self.lens, self.queries)):
            if q == 0:
                continue
            o, le = out[first : first + q].double(), lse[first : first + q].double()
            query = self.query[first : first + q].double()
            first += q
            pages = self.table[b, : -(-n // self.page)].long()
            bad = [i for i, p in enumerate(pages.tolist()) if not 0 <= p < self.codes.shape[0]] if dead else []
            pages = pages.clamp(0, self.codes.shape[0] - 1)
            dense = values64(self.codes[pages], self.scales[pages])
            k, v = (dense[:, part].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(group, 0) for part in (0, 1))
            i = torch.arange(n - q, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            seen = (j <= i) if causal else torch.ones(q, n, dtype=torch.bool, device="cuda")
            if window:
                seen = seen & (j > i - window)
            for p in bad:
                seen = seen & ((j < p * self.page) | (j >= (p + 1) * self.page))
            s = scale * query.transpose(0, 1) @ k.transpose(1, 2)
            s = s.masked_fill(~seen, -math.inf)
            some = seen.any(-1)
            assert (o[~some] == 0).all() and (le[~some] == -math.inf).all()
            if not some.any():
                continue
            p = torch.softmax(s[:, some], -1)
            want = (p @ v).transpose(0, 1)
            want_lse = torch.logsumexp(s[:, some], -1).T
            mass = (p @ v.abs()).transpose(0, 1)
            reach = (scale * query.transpose(0, 1)[:, some].abs() @ k.abs().transpose(1, 2)).masked_fill(~seen[some], 0).amax(-1).T  # [q, heads]
            d = reach * (self.dim + 16) * 2.0**-23 + 2.0**-20
            err = mass * (2.0**-11 + 2 * d[..., None]) + 2.0**-26 * v.abs().amax()
            tol = err + half_step(self.query.dtype) * (want.abs() + err).clamp_min(torch.finfo(self.query.dtype).tiny)
            assert ((o[some] - want).abs() <= tol).all(), float(((o[some] - want).abs() / tol).max())
            assert ((le[some] - want_lse).abs() <= d + 2.0**-21 * (1 + want_lse.abs())).all()
        assert (out[first:] == 0).all() and (lse[first:] == -math.inf).all()


DECODE = [
    # lens, queries, heads, kv, page, dim
    ([1], [1], 1, 1, 16, 64),
    ([0, 5, 0, 1], [1, 1, 0, 1], 4, 2, 16, 64),
    ([15, 16, 17, 31, 32, 33], [1] * 6, 8, 8, 16, 128),
    ([127, 128, 129, 500, 1], [1] * 5, 10, 2, 64, 128),
    ([700, 3, 64], [1] * 3, 40, 8, 64, 128),
    ([1000, 77], [2, 2], 9, 3, 32, 128),
    ([300, 299], [3, 1], 17, 1, 128, 64),
    ([60, 513, 9], [7, 5, 9], 6, 3, 16, 64),
    ([5000, 4999], [1, 1], 3, 1, 128, 128),
    ([40, 20, 1] * 40, [1] * 120, 4, 4, 16, 64),
    ([260, 90], [33, 20], 5, 1, 64, 128),
]
PROMPT = [
    ([70] * 10, [70] * 10, 8, 4, 16, 64),
    ([300, 1, 129, 0, 64], [300, 1, 129, 0, 64], 16, 8, 64, 128),
    ([513, 900], [200, 511], 20, 4, 32, 128),
    ([1000, 333], [1000, 130], 15, 15, 128, 64),
    ([257, 77, 640], [256, 70, 2], 24, 8, 64, 128),
    ([90, 60], [90, 65], 34, 17, 16, 128),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DECODE + PROMPT)
def test_attention_matches_64_bits(lens, queries, heads, kv, page, dim, dtype) -> None:
    case = Case(len(lens) + heads, lens, queries, heads, kv, page, dim, dtype)
    case.check(*case.run())


SHARED = [
    # Units of more tiles than a block keeps to itself.
    ([1700, 3, 2900], [1] * 3, 40, 8, 64, 128),
    ([2000, 1300], [3, 1], 17, 1, 128, 64),
    ([1500, 0, 1601, 5702], [7, 0, 5, 9], 6, 3, 16, 64),
    ([4097, 1025], [33, 20], 5, 1, 32, 128),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window", [0, 1900])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", SHARED)
def test_attention_over_shared_units(lens, queries, heads, kv, page, dim, window, dtype) -> None:
    case = Case(22, lens, queries, heads, kv, page, dim, dtype)
    out, lse = case.run(window=window)
    case.check(out, lse, window=window)
    again, lse2 = case.run(window=window)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    for bound in (1, 100, 100000):  # what the launch is sized for changes which blocks share, not the result
        case.check(*case.run(window=window, max_length=bound), window=window)


@pytest.mark.parametrize("window", [1, 16, 17, 100, 5000])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[3], DECODE[5], DECODE[8], PROMPT[1], PROMPT[2], PROMPT[3]])
def test_sliding_windows(lens, queries, heads, kv, page, dim, window) -> None:
    case = Case(window, lens, queries, heads, kv, page, dim, BF)
    case.check(*case.run(window=window), window=window)


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[1], DECODE[7], PROMPT[0], PROMPT[4]])
def test_without_a_mask_and_with_another_scale(lens, queries, heads, kv, page, dim) -> None:
    case = Case(3, lens, queries, heads, kv, page, dim, HF)
    case.check(*case.run(causal=False, softmax_scale=0.31), causal=False, softmax_scale=0.31)


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[4], PROMPT[2]])
def test_rows_behind_the_last_sequence_are_zero(lens, queries, heads, kv, page, dim) -> None:
    case = Case(4, lens, queries, heads, kv, page, dim, BF, behind=7)
    case.query[sum(queries):] = float("nan")
    case.check(*case.run())


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[3], DECODE[7], PROMPT[1], PROMPT[2]])
def test_queries_of_any_stride(lens, queries, heads, kv, page, dim) -> None:
    case = Case(5, lens, queries, heads, kv, page, dim, BF)
    out, lse = case.run()
    fused = torch.zeros(case.query.shape[0], heads + 2 * kv, dim, dtype=BF, device="cuda")
    fused[:, :heads] = case.query
    odd = torch.zeros(case.query.shape[0], heads, dim + 3, dtype=BF, device="cuda")
    odd[..., 3:] = case.query
    for q in (fused[:, :heads], odd[..., 3:], case.query.transpose(0, 1).contiguous().transpose(0, 1)):
        o, le = case.run(query=q)
        assert torch.equal(o, out) and torch.equal(le, lse)


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[3], DECODE[5], PROMPT[1], PROMPT[2]])
def test_bad_pages_are_left_out(lens, queries, heads, kv, page, dim) -> None:
    case = Case(6, lens, queries, heads, kv, page, dim, BF)
    b = max(range(len(lens)), key=lambda i: lens[i])
    case.table[b, 0], case.table[b, 1] = -1, case.codes.shape[0]
    case.check(*case.run(), dead=frozenset((b,)))


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[4], DECODE[7], PROMPT[1], PROMPT[4]])
def test_wrong_bounds_cost_speed_only(lens, queries, heads, kv, page, dim) -> None:
    case = Case(7, lens, queries, heads, kv, page, dim, BF)
    for length, most in ((1, 1), (100000, 1), (1, 500), (100000, 500)):
        case.check(*case.run(max_length=length, max_queries=most))


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[3], PROMPT[2]])
@pytest.mark.parametrize("size", [2.0**-60, 1.0e4])
def test_large_and_small_queries(lens, queries, heads, kv, page, dim, size) -> None:
    case = Case(8, lens, queries, heads, kv, page, dim, BF)
    case.query = (case.query.float() * size).to(BF)
    scale = case.dim**-0.5 / max(size, 1.0)
    case.check(*case.run(softmax_scale=scale), softmax_scale=scale)


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[3], PROMPT[2]])
def test_values_of_very_different_size(lens, queries, heads, kv, page, dim) -> None:
    """Values that grow by 2^40 along the sequence, then fall: the reference they are held to has to follow."""
    case = Case(9, lens, queries, heads, kv, page, dim, BF)
    b = max(range(len(lens)), key=lambda i: lens[i])
    n = lens[b]
    token = torch.arange(n, device="cuda")
    pages = case.table[b, : -(-n // page)].long()
    grow = (40 * torch.sin(3.1 * token / n)).round().int()
    s = case.scales[pages, 1].permute(0, 2, 1, 3).reshape(-1, kv, dim // 32)
    s[:n] = (s[:n].int() + grow[:, None, None]).clamp(0, 254).to(torch.uint8)
    case.scales[pages, 1] = s.view(len(pages), page, kv, dim // 32).permute(0, 2, 1, 3)
    case.check(*case.run())


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[5], PROMPT[2]])
def test_non_finite_queries_stay_their_own(lens, queries, heads, kv, page, dim) -> None:
    case = Case(10, lens, queries, heads, kv, page, dim, BF)
    out, _ = case.run()
    case.query[1, 0, 5], case.query[2, 1, 7] = float("nan"), float("inf")
    got, _ = case.run()
    same = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    same[1, 0] = same[2, 1] = False
    assert got[1, 0].isnan().all() and got[2, 1].isnan().all() and torch.equal(got[same], out[same])


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[4], DECODE[9], PROMPT[2]])
def test_equal_calls_give_equal_bits_on_any_stream(lens, queries, heads, kv, page, dim) -> None:
    case = Case(11, lens, queries, heads, kv, page, dim, BF)
    out, lse = case.run()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [case.run() for _ in range(3)]  # three streams at once, each with its own workspaces
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) and torch.equal(le, lse) for o, le in got)


@pytest.mark.parametrize("queries", [1, 600])
def test_pages_past_32_bits(queries: int) -> None:
    """A layer of more than 2^32 bytes: what lies at its end is as good as what lies at its start."""
    g = gen(20)
    kv, page, dim, pages, held = 8, 128, 128, 33000, 5
    big = [torch.zeros(pages, 2, kv, page, n, dtype=torch.uint8, device="cuda") for n in (dim // 2, dim // 32)]
    small = [torch.zeros(held, 2, kv, page, n, dtype=torch.uint8, device="cuda") for n in (dim // 2, dim // 32)]
    assert big[0].numel() > 2**32
    tokens = held * page - 7
    key, value, query = randn(g, tokens, kv, dim), randn(g, tokens, kv, dim), randn(g, queries, 4 * kv, dim).to(BF)
    slots = torch.arange(tokens, device="cuda")
    far = pages - held
    start = torch.tensor([0, queries], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    got = []
    for pool, first in ((small, 0), (big, far)):
        kvcache.append_mxfp4_(*pool, key, value, slots + first * page)
        table = torch.arange(first, first + held, dtype=torch.int32, device="cuda")[None]
        got.append((*kvcache.gather_mxfp4(*pool, slots + first * page),
                    *kvcache.paged_attention_mxfp4(query, *pool, table, lengths, start, max_length=tokens, max_queries=queries, return_lse=True)))
    assert got[0][0].abs().sum() > 0 and got[0][2].abs().sum() > 0
    assert all(torch.equal(a, b) for a, b in zip(*got))
    kvcache.copy_pages_(big[0][None], big[1][None], [far + 1, far + 2], [2, far - 1])
    for part, pool in enumerate(big):
        assert torch.equal(pool[2], small[part][1]) and torch.equal(pool[far - 1], small[part][2])
        assert not pool[0].any() and not pool[far - 2].any()


def test_no_sequences_and_no_queries() -> None:
    case = Case(12, [5, 9], [0, 0], 4, 2, 16, 64, BF, behind=3)
    case.check(*case.run())
    codes, scales = case.codes, case.scales
    i32 = torch.zeros(0, dtype=torch.int32, device="cuda")
    out, lse = kvcache.paged_attention_mxfp4(case.query, codes, scales, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), i32,
                                             torch.zeros(1, dtype=torch.int32, device="cuda"), max_length=0, max_queries=0, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out = kvcache.paged_attention_mxfp4(case.query[:0], codes, scales, case.table, case.lengths, case.start, max_length=9, max_queries=1)
    assert out.shape == (0, 4, 64)


def test_attention_refusals() -> None:
    case = Case(13, [5], [1], 4, 2, 16, 64, BF)
    for kw, error in ((dict(query=case.query.float()), ValueError), (dict(query=case.query[:, :3]), ValueError), (dict(window=4, causal=False), ValueError),
                      (dict(softmax_scale=0.0), ValueError), (dict(max_length=-1), ValueError)):
        with pytest.raises(error):
            case.run(**kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        case.run(query=case.query.clone().requires_grad_())
    with pytest.raises(ValueError):
        kvcache.paged_attention_mxfp4(case.query, case.codes, case.scales, case.table.long(), case.lengths, case.start, max_length=5, max_queries=1)


# ------------------------------------------------------- operators and graphs


def test_opcheck() -> None:
    g = gen(14)
    packed, scales = quantize_mxfp4(randn(g, 40, 64), method="rtn")
    x = randn(g, 20, 64).to(BF)
    op = torch.ops.mxwave_b200
    torch.library.opcheck(op.linear_mxfp4.default, (x, packed, scales, randn(g, 40).to(BF), None, 2))
    case = Case(15, [20, 3], [1, 1], 4, 2, 16, 64, BF)
    rows, slots = randn(g, 3, 2, 64), torch.arange(3, device="cuda")
    torch.library.opcheck(op.kv_append_mxfp4_.default, (case.codes, case.scales, rows, rows, slots))
    torch.library.opcheck(op.kv_gather_mxfp4.default, (case.codes, case.scales, slots, torch.float32))
    torch.library.opcheck(op.paged_attention_mxfp4.default,
                          (case.query, case.codes, case.scales, case.table, case.lengths, case.start, 20, 1, 0.125, True, 0, True))
    layers = case.codes[None].clone(), case.scales[None].clone()
    torch.library.opcheck(op.copy_pages_.default, (*layers, torch.tensor([0]), torch.tensor([1])))


def test_the_two_eager_ways_agree(monkeypatch) -> None:
    """The host binding and the general path: the same results, the same side effects."""
    assert ops.binding is not None
    g = gen(20)
    packed, scales = quantize_mxfp4(randn(g, 200, 128), method="rtn")
    case = Case(21, [300, 20], [2, 2], 8, 2, 32, 64, BF)
    x, bias, residual = randn(g, 5, 128).to(BF), randn(g, 200).to(BF), randn(g, 5, 200).to(BF)
    rows, slots = randn(g, 4, 2, 64).to(BF), torch.tensor([1, 3, -1, 40], device="cuda")
    layers = case.codes[None].repeat(2, 1, 1, 1, 1, 1), case.scales[None].repeat(2, 1, 1, 1, 1, 1)

    def run():
        codes, sc = case.codes.clone(), case.scales.clone()
        versions = codes._version, sc._version
        kvcache.append_mxfp4_(codes, sc, rows, rows, slots)
        assert codes._version > versions[0] and sc._version > versions[1]
        pair = layers[0].clone(), layers[1].clone()
        kvcache.copy_pages_(*pair, torch.tensor([0, 2]), torch.tensor([1, 3]))
        return [linear_mxfp4(x, packed, scales, bias, activation="gelu", residual=residual), linear_mxfp4(x[None], packed, scales), codes, sc, *pair,
                *kvcache.gather_mxfp4(codes, sc, slots, HF), *case.run(window=50), case.run(return_lse=False)]

    first = run()
    monkeypatch.setattr(ops, "binding", None)
    for a, b in zip(first, run()):
        assert a.shape == b.shape and torch.equal(a, b)


def test_captured_steps_replay_with_new_inputs() -> None:
    """Two graphs of one step each (decode and prompt), replayed in turn and on two streams at once."""
    g = gen(16)
    packed, scales = quantize_mxfp4(randn(g, 512, 256), method="rtn")
    graphs = []
    for rows, case in ((3, Case(17, [300, 20, 64], [1] * 3, 8, 2, 64, 128, BF)), (200, Case(18, [513, 900], [200, 511], 20, 4, 32, 128, BF))):
        x = randn(g, rows, 256).to(BF)
        run = lambda case=case, x=x: (case.run(), linear_mxfp4(x, packed, scales))  # noqa: E731
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        graphs.append((case, x, graph, held, run))
    side = torch.cuda.Stream()
    for _ in range(3):
        for case, x, *_rest in graphs:
            case.query.copy_(randn(g, *case.query.shape))
            x.copy_(randn(g, *x.shape))
        torch.cuda.synchronize()
        graphs[0][2].replay()
        with torch.cuda.stream(side):
            graphs[1][2].replay()
        torch.cuda.synchronize()
        for case, _x, _graph, ((out, lse), y), run in graphs:
            (o, le), y2 = run()
            assert torch.equal(o, out) and torch.equal(le, lse) and torch.equal(y, y2)
            case.check(out, lse)


def test_a_decoder_runs_on_the_set() -> None:
    """Prompts, decoding steps, a fork, rejected drafts and a compaction, through two layers: every step's attention against
    the cache read back and multiplied out in 64 bits."""
    g = gen(19)
    hidden, heads, kv, dim, layers = 256, 6, 2, 64, 2
    proj = [[quantize_mxfp4(randn(g, o, i) * i**-0.5) for o, i in (((heads + 2 * kv) * dim, hidden), (hidden, heads * dim))] for _ in range(layers)]
    cache = kvcache.PagedKVCache(48, kv_heads=kv, head_dim=dim, layers=layers, page_tokens=16)

    def step(seqs: list[int], tokens: list[int]) -> None:
        batch = cache.plan(seqs, tokens)
        h = randn(g, sum(tokens), hidden).to(BF)
        for layer, (qkv_w, o_w) in enumerate(proj):
            qkv = linear_mxfp4(h, *qkv_w).unflatten(-1, (-1, dim))
            q, k, v = qkv.split((heads, kv, kv), 1)
            cache.append(layer, k, v, batch)
            out = cache.attend(layer, q, batch)
            first = 0
            for seq, n in zip(seqs, tokens):
                kd, vd = (t.double().repeat_interleave(heads // kv, 1).transpose(0, 1) for t in cache.gather(layer, seq))
                length = kd.shape[1]
                assert length == cache.books.length(seq)
                s = q[first : first + n].double().transpose(0, 1) @ kd.transpose(1, 2) * dim**-0.5
                at = torch.arange(length - n, length, device="cuda")[:, None]
                s = s.masked_fill(torch.arange(length, device="cuda")[None] > at, -math.inf)
                p = torch.softmax(s, -1)
                want, mass = (p @ vd).transpose(0, 1), (p @ vd.abs()).transpose(0, 1)
                tol = mass * (2.0**-11 + 2.0**-12) + half_step(BF) * want.abs() + 1e-30
                assert ((out[first : first + n].double() - want).abs() <= tol).all()
                first += n
            h = linear_mxfp4(out.flatten(1), *o_w, residual=h)
        assert h.isfinite().all()

    a, b = cache.add(), cache.add()
    step([a, b], [37, 90])
    step([a, b], [1, 1])
    kept = [cache.gather(layer, b) for layer in range(layers)]
    c = cache.fork(b)
    step([c, a, b], [5, 1, 2])
    cache.truncate(c, 92)
    step([c], [3])
    for layer in range(layers):
        for seq in (b, c):
            assert all(torch.equal(now[:91], then) for now, then in zip(cache.gather(layer, seq), kept[layer]))
    cache.free(a)
    before = [cache.gather(layer, seq, F32) for layer in range(layers) for seq in (b, c)]
    cache.compact()
    after = [cache.gather(layer, seq, F32) for layer in range(layers) for seq in (b, c)]
    assert all(torch.equal(x, y) for pair, other in zip(before, after) for x, y in zip(pair, other))
    step([b, c, cache.add()], [1, 4, 65])
    with pytest.raises(RuntimeError, match="full"):
        cache.plan([b], [48 * 16])
