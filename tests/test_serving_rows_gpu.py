"""What one row of an attention call may not do to another, and what a row that sees a key gives, on a B200.

The tolerance is that of the row alone.  Probabilities are held as f16 (a half step of 2^-11, and 2^-25 below its normal
range, where a row's largest is at least 2^7: 2^-32 of it), values exactly, scores are off by d = scale sum |q k| (D +
16) 2^-23 + 2^-20 at most (each probability by the factor e^d, their sum likewise), and n keys are added in fp32, 16 at a
time, each addition off by a step 2^-23 at most:

    |out - want| <= sum p |v| (2^-11 + 2 d + (n / 16 + 64) 2^-23) + 2^-32 sum |v| + half a step of the type

with both sums over the keys that the row sees.
"""

from __future__ import annotations

import math

import pytest
import torch

from mxwave_b200 import kvcache
from tests.test_serving_gpu import BF, DECODE, HF, PROMPT, Case, gen, half_step, randn, values64

pytestmark = pytest.mark.gpu

# lens, queries, heads, kv, page, dim: several queries a sequence, on each of the kernels.
DRAFTS = [([60, 513, 9], [7, 5, 9], 6, 3, 16, 64), ([700, 41], [3, 4], 4, 2, 64, 128), ([2600, 90], [6, 2], 8, 8, 32, 128)]
PROMPTS = [([300, 129, 64], [300, 129, 64], 16, 8, 64, 128), ([513, 900], [200, 511], 20, 4, 32, 128), ([400, 333], [400, 130], 15, 15, 128, 64)]


class RowCase(Case):
    def slots(self, b: int) -> torch.Tensor:
        token = torch.arange(self.lens[b], device="cuda")
        return self.table[b].long()[token // self.page] * self.page + token % self.page

    def raise_values(self, b: int, keys: list[int], by: int) -> None:
        """The values of these keys times 2^by."""
        slots = self.slots(b)[keys]
        page, off = slots // self.page, slots % self.page
        self.scales[page, 1, :, off] = (self.scales[page, 1, :, off].int() + by).clamp(1, 254).to(torch.uint8)

    def check_rows(self, out: torch.Tensor, lse: torch.Tensor, *, window: int = 0, causal: bool = True) -> None:
        scale = self.dim**-0.5
        group = self.query.shape[1] // self.kv
        first = 0
        for b, (n, q) in enumerate(zip(self.lens, self.queries)):
            if q == 0 or n == 0:
                first += q
                continue
            o, le, query = (t[first : first + q].double() for t in (out, lse, self.query))
            first += q
            pages = self.table[b, : -(-n // self.page)].long()
            dense = values64(self.codes[pages], self.scales[pages])
            k, v = (dense[:, part].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(group, 0) for part in (0, 1))
            i, j = torch.arange(n - q, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            seen = ((j <= i) if causal else (j >= 0)).expand(q, n) & ((j > i - window) if window else (j >= 0))
            s = (scale * query.transpose(0, 1) @ k.transpose(1, 2)).masked_fill(~seen, -math.inf)
            some = seen.any(-1)  # a query before the sequence's first key sees none
            assert (o[~some] == 0).all() and (le[~some] == -math.inf).all()
            o, le, query, s, seen = o[some], le[some], query[some], s[:, some], seen[some]
            p = torch.softmax(s, -1)
            want, mass = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
            whole = (seen.double() @ v.abs()).transpose(0, 1)
            reach = (scale * query.transpose(0, 1).abs() @ k.abs().transpose(1, 2)).masked_fill(~seen, 0).amax(-1).T
            d = reach * (self.dim + 16) * 2.0**-23 + 2.0**-20
            err = mass * (2.0**-11 + 2 * d[..., None] + (n / 16 + 64) * 2.0**-23) + 2.0**-32 * whole
            tol = err + half_step(self.query.dtype) * (want.abs() + err).clamp_min(torch.finfo(self.query.dtype).tiny)
            fits = want.abs() + tol <= torch.finfo(self.query.dtype).max
            off = ((o - want).abs() / tol)[fits]
            assert (off <= 1).all(), (b, float(off.max()))
            assert (o[~fits].abs() >= 0.98 * torch.finfo(self.query.dtype).max).all()
            assert ((le - torch.logsumexp(s, -1).T).abs() <= d + 2.0**-21 * (1 + le.abs())).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DECODE + PROMPT)
def test_ordinary_rows_keep_their_own_tolerance(lens, queries, heads, kv, page, dim, dtype) -> None:
    case = RowCase(len(lens) + heads, lens, queries, heads, kv, page, dim, dtype)
    case.check_rows(*case.run())


@pytest.mark.parametrize("by", [24, 30, 60])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DRAFTS + PROMPTS)
def test_values_of_later_tokens_stay_out_of_earlier_rows(lens, queries, heads, kv, page, dim, by) -> None:
    """The last token's value is far larger than all others, which every earlier query of the call has to be blind to."""
    case = RowCase(31, lens, queries, heads, kv, page, dim, BF)
    for b, n in enumerate(lens):
        case.raise_values(b, [n - 1], by)
    case.check_rows(*case.run())


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DRAFTS + PROMPTS)
def test_overflowed_values_stay_out_of_earlier_rows(lens, queries, heads, kv, page, dim) -> None:
    case = RowCase(32, lens, queries, heads, kv, page, dim, BF)
    for b, n in enumerate(lens):
        row = torch.full((1, kv, dim), math.inf, device="cuda")
        key, _ = kvcache.gather_mxfp4(case.codes, case.scales, case.slots(b)[-1:], torch.float32)
        kvcache.append_mxfp4_(case.codes, case.scales, key, row, case.slots(b)[-1:])
    out, lse = case.run()
    case.check_rows(out, lse)
    # A value of 6 x 2^127: the row that sees it overflows unless its probability is under a third.
    assert not out[case.start[1:].long() - 1].isnan().any()


@pytest.mark.parametrize("window", [5, 33, 100])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DRAFTS + PROMPTS)
def test_values_before_the_window_have_no_say(lens, queries, heads, kv, page, dim, window) -> None:
    case = RowCase(33, lens, queries, heads, kv, page, dim, BF)
    for b, (n, q) in enumerate(zip(lens, queries)):
        keys = [max(0, n - q - window), max(0, n - q - window + 1), max(0, n - window - 1), n - 1 - min(n - 1, window)]
        case.raise_values(b, sorted(set(keys)), 40)
    case.check_rows(*case.run(window=window), window=window)


@pytest.mark.parametrize("queries", [1, 150])
@pytest.mark.parametrize("size, by", [(4.0, 40), (4.0, 28), (1.6, 25), (1.0, 18)])
@pytest.mark.parametrize("n", [333, 3000])
def test_improbable_keys_count_by_their_probability(queries, size, by, n) -> None:
    """A key whose value is 2^by times the others and whose score is far below them."""
    heads, page, dim = 40, 64, 128
    case = RowCase(34, [n], [queries], heads, heads, page, dim, BF)
    case.query[:] = case.query[:1]  # (every row finds the key improbable)
    at = n - queries - 7
    key, value = kvcache.gather_mxfp4(case.codes, case.scales, case.slots(0)[at : at + 1], torch.float32)
    kvcache.append_mxfp4_(case.codes, case.scales, -size * case.query[:1].float(), value, case.slots(0)[at : at + 1])
    case.raise_values(0, [at], by)
    case.check_rows(*case.run())


@pytest.mark.parametrize("dtype, by", [(BF, -60), (BF, 50), (BF, -24), (BF, 22), (HF, -14), (HF, 30)])
@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DRAFTS[:2] + PROMPTS[1:])
def test_channel_blocks_of_different_size(lens, queries, heads, kv, page, dim, dtype, by) -> None:
    """The first 32 channels of every value are 2^by times the others."""
    case = RowCase(35, lens, queries, heads, kv, page, dim, dtype)
    if dtype == HF:  # both sizes within f16's range
        case.scales[:, 1] = (case.scales[:, 1].int() - (15 if by > 0 else 0)).clamp(0, 254).to(torch.uint8)
    case.scales[:, 1, ..., 0] = (case.scales[:, 1, ..., 0].int() + by).clamp(0, 254).to(torch.uint8)
    case.check_rows(*case.run())


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", [DECODE[1], DECODE[3], DECODE[8], PROMPT[2], PROMPT[3]])
def test_values_of_very_different_size_by_rows(lens, queries, heads, kv, page, dim) -> None:
    """Values that grow by 2^40 along the sequence, then fall."""
    case = RowCase(9, lens, queries, heads, kv, page, dim, BF)
    for b, n in enumerate(lens):
        for key in range(n):
            by = round(40 * math.sin(3.1 * key / n))
            if key % 64 == 0 or by != round(40 * math.sin(3.1 * (key - 1) / n)):
                end = next((k for k in range(key + 1, n) if round(40 * math.sin(3.1 * k / n)) != by or k % 64 == 0), n)
                case.raise_values(b, list(range(key, end)), by)
    case.check_rows(*case.run())


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DRAFTS + PROMPTS)
def test_bad_pages_and_wide_values(lens, queries, heads, kv, page, dim) -> None:
    """Pages outside the pool are left out of rows whose values differ widely in size too."""
    case = RowCase(36, lens, queries, heads, kv, page, dim, BF)
    b = max(range(len(lens)), key=lambda i: lens[i])
    case.raise_values(b, [lens[b] - 1], 50)
    case.raise_values(b, [lens[b] // 2], -50)
    case.table[b, 1] = case.codes.shape[0]
    got = case.run()
    want = RowCase.__new__(RowCase)
    want.__dict__ = {**case.__dict__, "lens": [lens[b] - page], "queries": [queries[b]]}
    first = sum(queries[:b])
    want.query = case.query[first : first + queries[b]]
    want.table = torch.cat((case.table[b : b + 1, :1], case.table[b : b + 1, 2:]), 1)
    if lens[b] - queries[b] >= 2 * page:  # the sequence without that page: the same keys at other places
        want.check_rows(*(t[first : first + queries[b]] for t in got))
    assert not got[0].isnan().any()


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DRAFTS + PROMPTS)
def test_wide_values_without_a_mask(lens, queries, heads, kv, page, dim) -> None:
    case = RowCase(38, lens, queries, heads, kv, page, dim, HF)
    for b, n in enumerate(lens):
        case.raise_values(b, [n // 3], 13)
        case.raise_values(b, [n // 2], -13)
    case.check_rows(*case.run(causal=False), causal=False)


def test_wide_values_give_equal_bits() -> None:
    case = RowCase(37, [2600, 900], [6, 300], 8, 8, 32, 128, BF)
    case.raise_values(0, [2599], 60)
    case.raise_values(1, [899, 20], 60)
    first = case.run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, case.run()))
    fused = torch.zeros(306, 8, 131, dtype=BF, device="cuda")
    fused[..., 3:] = case.query
    assert all(torch.equal(a, b) for a, b in zip(first, case.run(query=fused[..., 3:])))


@pytest.mark.parametrize("lens, queries, heads, kv, page, dim", DECODE[:10] + PROMPTS)
@pytest.mark.parametrize("by", [118, -112])
def test_values_near_the_ends_of_the_range(lens, queries, heads, kv, page, dim, by) -> None:
    """Sums in the units of the probabilities would overflow where the values themselves do not."""
    case = RowCase(39, lens, queries, heads, kv, page, dim, BF)
    for b, n in enumerate(lens):
        if n:
            case.raise_values(b, list(range(n)), by)
    case.check_rows(*case.run())


@pytest.mark.parametrize("queries", [1, 6])
def test_an_overflowed_value_in_a_share_of_little_weight(queries) -> None:
    """A value past fp32's range, in a block's share of the keys that next to nothing of the probability falls on."""
    heads, n, page, dim = 2, 30000, 64, 128
    case = RowCase(40, [n], [queries], heads, heads, page, dim, BF)
    case.query[:] = case.query[:1]
    far = torch.arange(0, 20000, device="cuda")
    key = (-20.0 * case.query[:1].float()).expand(len(far), -1, -1).contiguous()
    value = randn(gen(41), len(far), heads, dim)
    value[7777] = math.inf
    kvcache.append_mxfp4_(case.codes, case.scales, key, value, case.slots(0)[far])
    case.check_rows(*case.run())
