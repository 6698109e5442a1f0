// K10: softmax attention over a paged key/value cache held in MXFP4.
//
//   out[i, h] = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j + mask)
//
// for packed queries of many sequences, grouped-query heads, causal masks and
// sliding windows.  Keys and values are decoded on the way into the matrix
// instructions; nothing is written back.
//
// Decoding kernel (attention_kernel): few query rows per key/value head, so
// the time is that of reading 2 x 4.25 bits per cached element, if the decoding
// keeps up.  Every choice below serves that:
//   * Matrix instructions m16n8k16 with the cached tensor as the 16-row operand:
//     S^T = K Q^T (16 keys x 8 query rows) and O^T = V^T P^T (16 channels x 8
//     rows).  Eight rows is the least a matrix instruction takes; grouped heads
//     share one, so each code is decoded once per group of up to 8 NT rows.
//   * The contraction's order is free, so lanes take bytes that lie together.
//     Four lanes share a key row, each a word of eight codes of every block: no
//     product of 16 elements mixes two scales, and the block's scale is applied
//     to the fp32 sum.  Eight lanes share a value row, eight bytes each, and
//     key pairs are interleaved nibble by nibble.  The 16-byte pieces of the
//     rows are placed so that none of these loads meets a bank conflict.
//   * A byte of two codes becomes an f16 pair in one conversion.  Codes are
//     exact in f16; queries are scaled by a power of two per row (bf16) and are
//     exact down to 2^-31 of the row's largest.  The values' scales run across
//     the contraction, so they are multiplied into the codes, relative to the
//     largest scale seen so far (times 2^13, below f16's maximum): exact down to
//     2^-27 of it, and rows with smaller ones are done again (kAttSpan).
//   * Probabilities are rounded to f16 as 2^(x - m + 7): 11 bits down to 2^-21
//     of the largest, nothing lost above 2^-31.  Their sum is taken in fp32
//     before the rounding.  m is raised only when a score passes it by 8
//     (binary), which spares most tiles the reduction and the rescaling.
//   * Four warps of a block take steps of 32 keys in turn, each with its own
//     running maximum and sum, its own ring of asynchronous copies and no
//     synchronisation with the others until the end of a segment.
// Work split: the (sequence, head, row group) units are cut into tiles of 128
// keys, all tiles are laid end to end (each unit's behind the cost of starting
// it), and each block takes an equal share, whatever the lengths (units of few
// tiles stay whole, see kAttWhole).  A unit that
// several blocks share leaves partial results (normalised rows and their
// log-sum-exp) in the workspace, two slots per block, and attention_join_kernel
// adds them in block order.
// Measured: 32 sequences of 1 to 65,536 keys, 40 heads over 8 of 128, one query
// each: 192 us, 4.2 TB/s of cache and rows, 65% of the copy rate; bound by its
// instructions (some 340 a warp per 16 keys, half of them conversions and matrix
// instructions; 61% of the issue slots with 16 warps an SM).  One sequence of 517 keys: 13.2 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "attention.cuh"
#include "blockscale.cuh"
#include "common.cuh"
#include "runtime.h"

namespace mxw {

constexpr int kAttWarps = 4;
constexpr int kAttThreads = kAttWarps * 32;
constexpr int kAttHalf = 16;                      // keys per matrix instruction
constexpr int kAttKeys = 2 * kAttHalf;            // keys per warp step
constexpr int kAttTile = kAttWarps * kAttKeys;    // keys per block step
constexpr int kAttStages = 3;
constexpr int kAttJoinThreads = 256;
// What starting a unit costs a block, in tiles: with units of a tile or two
// counted by their tiles alone, blocks that got a run of short sequences
// finished last (393 us against 212 on 32 sequences of 1 to 65,536 keys; 325,
// 253, 212 and 217 us with 1, 2, 4 and 8 here).
constexpr int kAttStart = 4;
// Short units are not shared between blocks, and nothing is joined: up to 12
// tiles when there is a unit for every block that fits the GPU, up to 6 when
// there are few (40 heads over 8, one query, whole against shared: 1 sequence of
// 300, 516, 1000 keys 9.8, 12.2, 15.0 and 12.7, 12.4, 12.6 us; 64 sequences of 300,
// 700, 1100 keys 17, 23, 30 and 25, 32, 39 us).
constexpr int kAttWhole = 12, kAttWholeFew = 6;
// Scales of values up to this many powers of two below the largest so far are not
// looked at one by one: tracking the smallest in every step took 197 us where this
// takes 192 (32 sequences of 1 to 65,536 keys; 187 without a look at the range).
// So the range is looked at closer when the largest rises by more than kAttSpan
// - kAttQuiet.
constexpr int kAttQuiet = 16;
// Partial results are this much of themselves: 6 x 2^127, an overflowed value, is finite, and nothing where its share weighs nothing.
constexpr float kAttPartial = 0.0625f;

// One sequence's share of the work.
struct AttSeq {
  int q0, queries;  // its rows of the packed queries
  int length;       // cached tokens
  int lo;           // first key that some query sees, rounded down to 32 (a step stays in a page)
  int tiles;        // tiles of 128 keys from lo on, at least one
  int row_groups;   // groups of 8 NT rows per key/value head
};

template <int ROWS>
__device__ __forceinline__ AttSeq att_seq(const AttParams& P, int b) {
  AttSeq s;
  const int64_t first = P.start[b], last = P.start[b + 1];
  s.q0 = static_cast<int>(max(static_cast<int64_t>(0), min(first, P.tokens)));
  s.queries = static_cast<int>(max(static_cast<int64_t>(0), min(last, P.tokens) - s.q0));
  const int64_t held = P.table_width << P.page_shift;
  s.length = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(P.lengths[b]), held)));
  s.lo = P.window > 0 ? max(0, s.length - s.queries - P.window + 1) / kAttKeys * kAttKeys : 0;
  s.tiles = max(1, (s.length - s.lo + kAttTile - 1) / kAttTile);
  s.row_groups = (s.queries * P.group + ROWS - 1) / ROWS;
  return s;
}

__device__ __forceinline__ int64_t att_work(const AttParams& P, const AttSeq& s) {
  return static_cast<int64_t>(P.whole ? 1 : s.tiles + kAttStart) * s.row_groups * P.kv_heads;
}

// Sum over the block (all threads get it); `red` holds one word per warp.
template <int THREADS>
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) sum += red[w];
  return sum;
}

// All tiles, and the tiles of the sequences before `upto`.
template <int ROWS, int THREADS>
__device__ __forceinline__ void att_totals(const AttParams& P, int upto, int64_t* red, int64_t& total, int64_t& before) {
  int64_t all = 0, part = 0;
  for (int b = threadIdx.x; b < P.seqs; b += THREADS) {
    const int64_t w = att_work(P, att_seq<ROWS>(P, b));
    all += w;
    if (b < upto) part += w;
  }
  total = block_sum<THREADS>(all, red);
  before = upto > 0 ? block_sum<THREADS>(part, red) : 0;
}

// Equal shares of `total` tiles: the first total % blocks of them are one larger.
struct AttShares {
  int64_t each, more;
  __device__ __forceinline__ AttShares(int64_t total, int64_t blocks) : each(total / blocks), more(total % blocks) {}
  __device__ __forceinline__ int64_t first(int64_t block) const { return each * block + min(block, more); }
  __device__ __forceinline__ int64_t block_of(int64_t tile) const {
    const int64_t large = (each + 1) * more;
    return tile < large ? tile / (each + 1) : more + (tile - large) / each;
  }
};

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void cp_async16_if(bool on, uint32_t saddr, const void* src, uint32_t src_bytes) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16, %2;\n\t}" ::"r"(saddr),
      "l"(src), "r"(src_bytes), "r"(static_cast<uint32_t>(on))
      : "memory");
}
// Shared-memory loads by 32-bit address and a constant offset: the kernel's
// lanes keep their places and add only the stage.
template <int OFF>
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1+%2];" : "=r"(v) : "r"(a), "n"(OFF));
  return v;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1+%2];" : "=h"(v) : "r"(a), "n"(OFF));
  return v;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1+%2];" : "=r"(v) : "r"(a), "n"(OFF));
  return v;
}
// WORDS (1 or 2) consecutive words.
template <int WORDS, int OFF>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[WORDS]) {
  if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2+%3];" : "=r"(v[0]), "=r"(v[1]) : "r"(a), "n"(OFF));
  else
    v[0] = lds32<OFF>(a);
}
// The low nibbles of `a` and the high nibbles of `b`: one three-input operation.
__device__ __forceinline__ uint32_t nibbles(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xCA;" : "=r"(d) : "r"(0x0f0f0f0fu), "r"(a), "r"(b));
  return d;
}
// 2^(byte - 127) of byte `b` of a word (0 for a zero byte: 2^-127 is nothing next to a score).
template <int B>
__device__ __forceinline__ float scale_of(uint32_t word) {
  return bits_f32((B == 3 ? word >> 1 : word << (23 - 8 * B)) & 0x7f800000u);
}

template <int D, int NT>
struct AttShape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kCodes = kAttHalf * D / 2;    // bytes of 16 rows
  static constexpr int kScales = kAttHalf * D / 32;
  static constexpr int kHalf = 2 * (kCodes + kScales);  // 16 keys and values: [K codes][V codes][K scales][V scales]
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kRing = kAttStages * kStage;
  static constexpr int kJoin = kAttWarps * kRows * D * 4;  // fp32 rows of each warp, in the drained rings
  static constexpr int kSmem = kAttWarps * kRing > kJoin ? kAttWarps * kRing : kJoin;
  static constexpr int kBlocks = NT == 1 ? 4 : 3;  // per SM: 128 and 168 registers a thread
  static constexpr int kSlot = kRows * D + kRows;  // floats of a partial result
};

// What odd data needs, as calls: their registers are not the kernel's (inline, the
// ragged batch took 196 us instead of 192).
template <bool BF16, int D>
__device__ __noinline__ float row_wide(const AttParams& P, int b, int head, const uint16_t* q, int from, int to, float (&o)[D / 32]) {
  return att_row_wide<BF16, D>(P, b, head, q, from, to, o);
}

template <int D>
__device__ __noinline__ uint64_t segment_range(const AttParams& P, int b, int head, int from, int to, int warp) {
  AttRange<D> range;
  range.look(P, b, head, from, to, warp, kAttWarps);
  return static_cast<uint64_t>(range.top) << 32 | range.low;
}

template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, AttShape<D, NT>::kBlocks) attention_kernel(const __grid_constant__ AttParams P) {
  using Shape = AttShape<D, NT>;
  constexpr int ROWS = Shape::kRows;
  constexpr int QREGS = D / 8;       // f16 pairs of a query row per lane
  constexpr int STEPS = D / 16;      // k16 steps of S, and 16-channel groups of O
  constexpr int BLOCKS = D / 32;     // scales per row
  extern __shared__ __align__(128) uint8_t att_smem[];
  __shared__ int64_t red[kAttWarps];
  __shared__ float row_m[kAttWarps][ROWS], row_l[kAttWarps][ROWS];
  __shared__ int warp_first[kAttWarps];     // ref at its first value; 0 once a scale below kAttQuiet has been met
  __shared__ int warp_ref[kAttWarps];       // ref below, and 256 where the range may be wide
  grid_dependents_launch();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* join = reinterpret_cast<float*>(att_smem);  // [warp][row][D]
  const uint32_t ring_s = smem_u32(att_smem) + warp * Shape::kRing;

  att_clear_rest<BF16>(P, D, blockIdx.x, gridDim.x);
  int64_t total, ignored;
  att_totals<ROWS, kAttThreads>(P, 0, red, total, ignored);
  const AttShares shares(total, gridDim.x);
  int64_t at = shares.first(blockIdx.x);
  const int64_t end = shares.first(blockIdx.x + 1ll);
  if (at >= end) return;

  // The sequence that holds the first tile: 32 at a time, every warp the same.
  int b = 0;
  int64_t rem = at;
  for (; b < P.seqs; b += 32) {
    const int64_t w = b + lane < P.seqs ? att_work(P, att_seq<ROWS>(P, b + lane)) : 0;
    int64_t sum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, sum > rem);
    if (past) {
      const int k = __ffs(past) - 1;
      rem -= __shfl_sync(0xffffffffu, sum - w, k);
      b += k;
      break;
    }
    rem -= __shfl_sync(0xffffffffu, sum, 31);
  }
  AttSeq seq = att_seq<ROWS>(P, b);

  const int tok_a = g ^ ((g >> 1) & 1);  // key of row g of S^T (row g + 8: 8 further on)
  const int v_a = (2 * t) ^ (t & 1), v_b = (2 * t + 1) ^ (t & 1);  // keys of the contraction's slots 2t, 2t + 1
  // Where this lane's 16-byte pieces of a copy go, and where it reads (bytes of half a stage).  Pieces of
  // key rows rotate over pairs of rows (D = 128) or fours; value rows four apart have their halves swapped.
  const uint32_t key_put = 16u * (D == 128 ? lane ^ ((lane >> 3) & 3) : lane ^ ((lane >> 3) & 1));
  const uint32_t value_put = 16u * (D == 128 ? lane ^ (((lane >> 4) & 1) << 1) : lane);
  const uint32_t key_get = tok_a * (D / 2) + t * 4 + 16u * (D == 128 ? (tok_a >> 1) & 3 : (tok_a >> 2) & 1);
  const uint32_t value_a = Shape::kCodes + v_a * (D / 2) + (D == 128 ? (g * 8) ^ ((t & 2) << 4) : g * 4);
  const uint32_t value_b = value_a + (v_b - v_a) * (D / 2);
  const uint32_t key_scale = 2 * Shape::kCodes + tok_a * BLOCKS;
  const uint32_t scale_a = 2 * Shape::kCodes + Shape::kScales + v_a * BLOCKS + g * BLOCKS / 8;
  const uint32_t scale_b = scale_a + (v_b - v_a) * BLOCKS;
  bool first_segment = true;
  while (at < end) {
    while (rem >= att_work(P, seq)) {
      rem -= att_work(P, seq);
      seq = att_seq<ROWS>(P, ++b);
    }
    const int cost = P.whole ? 1 : seq.tiles + kAttStart;
    const int64_t unit = rem / cost;
    const int c0 = static_cast<int>(rem % cost);
    const int c1 = static_cast<int>(min(static_cast<int64_t>(cost), c0 + (end - at)));
    const int tile0 = P.whole ? 0 : max(0, c0 - kAttStart), tile1 = P.whole ? seq.tiles : c1 - kAttStart;
    const bool opens = first_segment;
    at += c1 - c0;
    rem += c1 - c0;
    first_segment = false;
    if (tile1 <= tile0) continue;  // the share ends before the unit's first tile
    const int head = static_cast<int>(unit / seq.row_groups);  // key/value head
    const int row0 = static_cast<int>(unit % seq.row_groups) * ROWS;
    const int n_rows = min(ROWS, seq.queries * P.group - row0);

    // Bounds over the rows of the unit: a query's position grows with its row.
    const int pos0 = seq.length - seq.queries + row0 / P.group;
    const int pos1 = seq.length - seq.queries + (row0 + n_rows - 1) / P.group;
    const int lo_min = P.window > 0 ? max(0, pos0 - P.window + 1) : 0;
    const int lo_max = P.window > 0 ? max(0, pos1 - P.window + 1) : 0;
    const int hi_max = P.causal ? max(0, min(pos1 + 1, seq.length)) : seq.length;
    const int hi_min = P.causal ? max(0, pos0 + 1) : seq.length;  // rows past n_rows are never stored: any mask will do

    // ---- this warp's steps: 32 keys, every fourth of the segment
    const int key0 = seq.lo + tile0 * kAttTile + warp * kAttKeys;
    const int key_end = min(seq.lo + tile1 * kAttTile, hi_max);
    const int skip = lo_min > key0 ? (lo_min - key0) / kAttTile : 0;  // steps that end before the window
    const int steps = key_end > key0 ? (key_end - key0 + kAttTile - 1) / kAttTile : 0;
    // A page's size divides a tile's, so a step's place in its page is that of
    // the first step.  This lane's places in a page, and the step from page to page:
    const bool apart = P.page_shift == 4;  // each half of a step has a page of its own
    const int offset = key0 & ((1 << P.page_shift) - 1);
    const int head_codes = (D / 2) << P.page_shift, head_scales = BLOCKS << P.page_shift;
    const uint32_t page_codes = 2u * P.kv_heads * head_codes, page_scales = 2u * P.kv_heads * head_scales;
    constexpr int SC = Shape::kScales / 16;  // 16-byte pieces of 16 rows' scales: lanes 0.. keys, SC.. values
    const uint8_t* codes = P.codes + static_cast<int64_t>(head) * head_codes + offset * (D / 2) + lane * 16;
    const int64_t to_values = static_cast<int64_t>(P.kv_heads) * head_codes;
    const uint8_t* scales = P.scales + static_cast<int64_t>(head) * head_scales + offset * BLOCKS +
                            (lane < SC ? lane * 16 : static_cast<int64_t>(P.kv_heads) * head_scales + (lane - SC) * 16);
    const int32_t* table = P.table + static_cast<int64_t>(b) * P.table_ld + (key0 >> P.page_shift);
    const int table_step = kAttTile >> P.page_shift;

    // Copies 16 rows of a page into half a stage, zeros for a page outside the
    // pool (no branch, and no read: the copies' source size is zero).
    auto copy_half = [&](uint32_t st, int page, uint32_t in_page) -> uint32_t {
      const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(P.pages);
      const uint32_t at = ok ? page : 0, bytes = ok ? 16u : 0u;
      const uint8_t* kc = codes + static_cast<uint64_t>(at) * page_codes + in_page * (D / 2);
      const uint8_t* vc = kc + to_values;
      const uint8_t* sc = scales + static_cast<uint64_t>(at) * page_scales + in_page * BLOCKS;
#pragma unroll
      for (int k = 0; k < Shape::kCodes / 512; ++k) {
        cp_async16(st + key_put + (k * 512), kc + k * 512, bytes);
        cp_async16(st + value_put + (Shape::kCodes + k * 512), vc + k * 512, bytes);
      }
      cp_async16_if(lane < 2 * SC, st + lane * 16 + 2 * Shape::kCodes, sc, bytes);
      return ok ? 1u : 0u;
    };
    // Pages of a step's halves (-1 past the end), read one step before they are needed.
    int next0 = -1, next1 = -1;
    auto look_up = [&](int step) {
      next0 = step < steps ? table[step * table_step] : -1;
      if (apart) next1 = key0 + step * kAttTile + kAttHalf < key_end ? table[step * table_step + 1] : -1;
    };
    uint32_t valid = 0;  // two bits per stage: its halves hold rows of pages of the pool
    auto issue = [&](int step, int stage) {
      const int page0 = next0, page1 = apart ? next1 : next0;
      look_up(step + 1);
      const uint32_t st = ring_s + stage * Shape::kStage;
      uint32_t ok = copy_half(st, page0, 0);
      ok |= copy_half(st + Shape::kHalf, page1, apart ? 0 : kAttHalf) << 1;
      valid = (valid & ~(3u << (2 * stage))) | (ok << (2 * stage));
      cp_async_commit();
    };
    look_up(skip);
#pragma unroll
    for (int k = 0; k < kAttStages - 1; ++k) issue(skip + k, k);

    // ---- queries: row n = 8 nt + g of this lane, elements [8t, 8t + 8) of each block
    uint32_t q[NT][QREGS];
    float fq[NT][2];        // score factors of rows 2t and 2t + 1
    int key_lo[NT][2], key_hi[NT][2];  // and the keys they see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 8 * nt + g;
      const bool on = r < n_rows;
      const int i = on ? (row0 + r) / P.group : 0;
      const int h = head * P.group + (on ? (row0 + r) - i * P.group : 0);
      const int64_t base = static_cast<int64_t>(seq.q0 + i) * P.q_token + static_cast<int64_t>(h) * P.q_head + t * 8;
      const uint16_t* src = static_cast<const uint16_t*>(P.query) + base;
      uint16_t raw[D / 4];
      if (P.q_vec) {
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k)
          reinterpret_cast<uint4*>(raw)[k] = on ? reinterpret_cast<const uint4*>(src)[4 * k] : make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int k = 0; k < D / 4; ++k) raw[k] = on ? src[k / 8 * 32 + k % 8] : static_cast<uint16_t>(0);
      }
      float f = P.scale_log2;
      if constexpr (BF16) {
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < D / 4; ++k) amax = max(amax, static_cast<uint32_t>(raw[k]) & 0x7fffu);
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // The row's largest magnitude to [2^14, 2^15): exact in f16 down to 2^-31 of it.
        const int e = min(127 + 14 - max(static_cast<int>(amax >> 7), 1), 127);
        const float up = exp2i(e);
        f = __fmul_rn(f, exp2i(-e));
#pragma unroll
        for (int k = 0; k < QREGS; ++k)
          q[nt][k] = pack_f16x2(__fmul_rn(bits_f32(static_cast<uint32_t>(raw[2 * k]) << 16), up),
                                __fmul_rn(bits_f32(static_cast<uint32_t>(raw[2 * k + 1]) << 16), up));
      } else {
#pragma unroll
        for (int k = 0; k < QREGS; ++k) q[nt][k] = raw[2 * k] | (static_cast<uint32_t>(raw[2 * k + 1]) << 16);
      }
      f = fmaxf(f, 1e-37f);  // a masked score times it has to stay -infinity
      fq[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);      // lane of row 2t
      fq[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);  // lane of row 2t + 1
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int rr = 8 * nt + 2 * t + c;
        const int pos = seq.length - seq.queries + (row0 + rr) / P.group;
        key_hi[nt][c] = P.causal && rr < n_rows ? max(pos + 1, 0) : seq.length;
        key_lo[nt][c] = P.window > 0 ? max(0, pos - P.window + 1) : 0;
      }
    }

    float o[NT][STEPS][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < STEPS; ++k)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][k][c] = 0.0f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
    }
    int ref = 0;  // exponent byte that the values are relative to
    if (lane == 0) warp_first[warp] = 0;

    int stage = 0;
    for (int step = skip; step < steps; ++step) {
      issue(step + kAttStages - 1, stage == 0 ? kAttStages - 1 : stage - 1);
      cp_async_wait<kAttStages - 1>();
      __syncwarp();
      const int key = key0 + step * kAttTile;
      const uint32_t st = ring_s + stage * Shape::kStage;
      const uint32_t held = (valid >> (2 * stage)) & 3u;

      // ---- scores
      float s[2][NT][4];
      auto score_half = [&](auto which) {
        constexpr int H = decltype(which)::value, OFF = H * Shape::kHalf;
        uint32_t wa[BLOCKS], wb[BLOCKS];  // eight codes of each block, of two keys
#pragma unroll
        for (int w = 0; w < BLOCKS; ++w) {
          const uint32_t a = st + (key_get ^ (16u * w));
          wa[w] = lds32<OFF>(a);
          wb[w] = lds32<OFF + 8 * D / 2>(a);
        }
        uint32_t sa, sb;
        if constexpr (D == 128) {
          sa = lds32<OFF>(st + key_scale);
          sb = lds32<OFF + 8 * BLOCKS>(st + key_scale);
        } else {
          sa = lds16<OFF>(st + key_scale);
          sb = lds16<OFF + 8 * BLOCKS>(st + key_scale);
        }
        auto block = [&](auto index) {
          constexpr int B = decltype(index)::value;
          uint32_t ha[4], hb[4];
          e2m1x8_to_f16x2(wa[B], ha);
          e2m1x8_to_f16x2(wb[B], hb);
          const float fa = scale_of<B>(sa), fb = scale_of<B>(sb);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float acc[4];
            mma_f16_first(acc, ha[0], hb[0], ha[1], hb[1], q[nt][4 * B], q[nt][4 * B + 1]);
            mma_f16(acc, ha[2], hb[2], ha[3], hb[3], q[nt][4 * B + 2], q[nt][4 * B + 3]);
            s[H][nt][0] = B == 0 ? __fmul_rn(acc[0], fa) : __fmaf_rn(acc[0], fa, s[H][nt][0]);
            s[H][nt][1] = B == 0 ? __fmul_rn(acc[1], fa) : __fmaf_rn(acc[1], fa, s[H][nt][1]);
            s[H][nt][2] = B == 0 ? __fmul_rn(acc[2], fb) : __fmaf_rn(acc[2], fb, s[H][nt][2]);
            s[H][nt][3] = B == 0 ? __fmul_rn(acc[3], fb) : __fmaf_rn(acc[3], fb, s[H][nt][3]);
          }
        };
        block(std::integral_constant<int, 0>{});
        block(std::integral_constant<int, 1>{});
        if constexpr (BLOCKS == 4) {
          block(std::integral_constant<int, 2>{});
          block(std::integral_constant<int, 3>{});
        }
      };
      score_half(std::integral_constant<int, 0>{});
      score_half(std::integral_constant<int, 1>{});
      const bool edge = key < lo_max || key + kAttKeys > hi_min || held != 3u;
      if (edge) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bool in = (held >> half) & 1u;
          const int key_a = key + half * kAttHalf + tok_a, key_b = key_a + 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (!in || key_a < key_lo[nt][c] || key_a >= key_hi[nt][c]) s[half][nt][c] = -INFINITY;
              if (!in || key_b < key_lo[nt][c] || key_b >= key_hi[nt][c]) s[half][nt][2 + c] = -INFINITY;
            }
        }
      }
      // ---- scales of the values
      uint32_t sv[2][2];  // halfwords: (v_a, v_b), (v_a + 8, v_b + 8)
      sv[0][0] = lds8<0>(st + scale_a) | (lds8<0>(st + scale_b) << 16);
      sv[0][1] = lds8<8 * BLOCKS>(st + scale_a) | (lds8<8 * BLOCKS>(st + scale_b) << 16);
      sv[1][0] = lds8<Shape::kHalf>(st + scale_a) | (lds8<Shape::kHalf>(st + scale_b) << 16);
      sv[1][1] = lds8<Shape::kHalf + 8 * BLOCKS>(st + scale_a) | (lds8<Shape::kHalf + 8 * BLOCKS>(st + scale_b) << 16);
      if (edge) {
        // Keys that no row sees (stale rows of the page) have no say in the reference.
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int k = key + half * kAttHalf + 8 * c;
            const bool in = (held >> half) & 1u;
            if (!in || k + v_a < lo_min || k + v_a >= hi_max) sv[half][c] &= 0xffff0000u;
            if (!in || k + v_b < lo_min || k + v_b >= hi_max) sv[half][c] &= 0x0000ffffu;
          }
      }
      // Scales outside [ref - kAttQuiet, ref] (zeros too) are looked at below; most steps have none.
      const uint32_t base2 = (static_cast<uint32_t>(kAttQuiet - ref) & 0xffffu) * 0x10001u;
      const uint32_t far2 = __vmaxu2(__viaddmax_u16x2(sv[0][1], base2, __vadd2(sv[0][0], base2)),
                                     __viaddmax_u16x2(sv[1][1], base2, __vadd2(sv[1][0], base2)));
      bool raise = max(far2 & 0xffffu, far2 >> 16) > static_cast<uint32_t>(kAttQuiet);
      // (The factors fq are positive: the largest raw score gives the largest.)
      float most[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          most[nt][c] = __fmul_rn(fmaxf(fmaxf(s[0][nt][c], s[0][nt][2 + c]), fmaxf(s[1][nt][c], s[1][nt][2 + c])), fq[nt][c]);
          raise |= most[nt][c] > __fadd_rn(m[nt][c], kAttSlack);
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = most[nt][c];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float up = fmaxf(m[nt][c], x);
            const float f = m[nt][c] == up ? 1.0f : ex2(__fsub_rn(m[nt][c], up));
            m[nt][c] = up;
            l[nt][c] = __fmul_rn(l[nt][c], f);
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
              o[nt][k][c] = __fmul_rn(o[nt][k][c], f);
              o[nt][k][2 + c] = __fmul_rn(o[nt][k][2 + c], f);
            }
          }
        const uint32_t top2 = __vmaxu2(__vmaxu2(sv[0][0], sv[0][1]), __vmaxu2(sv[1][0], sv[1][1]));
        const int top = __reduce_max_sync(0xffffffffu, static_cast<int>(max(top2 & 0xffffu, top2 >> 16)));
        // (A zero byte is a block of zeros, or of values under 6 x 2^-127, which count as zeros next to larger ones.)
        uint32_t low2 = 0xffffffffu;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int c = 0; c < 2; ++c) low2 = __viaddmin_u16x2(sv[half][c], 0xffffffffu, low2);
        if (ref == 0 && lane == 0) warp_first[warp] = top;
        __syncwarp();
        if (static_cast<int>(min(low2 & 0xffffu, low2 >> 16)) + 1 < max(ref, top) - kAttQuiet) warp_first[warp] = 0;
        if (top > ref) {
          const float f = exp2i(max(ref - top, -149));
          ref = top;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[nt][k][c] = __fmul_rn(o[nt][k][c], f);
        }
      }

      // ---- probabilities, transposed into the second product's operand
      uint32_t p0[2][NT], p1[2][NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float base0 = __fsub_rn(kAttLift, m[nt][0] == -INFINITY ? 0.0f : m[nt][0]);
        const float base1 = __fsub_rn(kAttLift, m[nt][1] == -INFINITY ? 0.0f : m[nt][1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float x0 = ex2(__fmaf_rn(s[half][nt][0], fq[nt][0], base0)), x1 = ex2(__fmaf_rn(s[half][nt][1], fq[nt][1], base1));
          const float x2 = ex2(__fmaf_rn(s[half][nt][2], fq[nt][0], base0)), x3 = ex2(__fmaf_rn(s[half][nt][3], fq[nt][1], base1));
          l[nt][0] = __fadd_rn(l[nt][0], __fadd_rn(x0, x2));
          l[nt][1] = __fadd_rn(l[nt][1], __fadd_rn(x1, x3));
          p0[half][nt] = transpose8(pack_f16x2(x0, x1));
          p1[half][nt] = transpose8(pack_f16x2(x2, x3));
        }
      }

      const uint32_t lift2 = (static_cast<uint32_t>(28 - ref) & 0xffffu) * 0x10001u;
      auto value_half = [&](auto which) {
        constexpr int H = decltype(which)::value, OFF = H * Shape::kHalf;
        constexpr int VW = D / 64;  // words of an eighth of a row
        uint32_t wa[VW], wb[VW], wc[VW], wd[VW];
        lds_words<VW, OFF>(st + value_a, wa);
        lds_words<VW, OFF>(st + value_b, wb);
        lds_words<VW, OFF + 8 * D / 2>(st + value_a, wc);
        lds_words<VW, OFF + 8 * D / 2>(st + value_b, wd);
        const uint32_t mlo = f16_factors(sv[H][0], lift2), mhi = f16_factors(sv[H][1], lift2);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          // Bytes of (first key's code, second key's code): even channels, then odd.
          uint32_t el[4], ol[4], eh[4], oh[4];
          e2m1x8_to_f16x2(nibbles(wa[w], wb[w] << 4), el);
          e2m1x8_to_f16x2(nibbles(wa[w] >> 4, wb[w]), ol);
          e2m1x8_to_f16x2(nibbles(wc[w], wd[w] << 4), eh);
          e2m1x8_to_f16x2(nibbles(wc[w] >> 4, wd[w]), oh);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a0 = hmul2(el[k], mlo), a1 = hmul2(ol[k], mlo);
            const uint32_t a2 = hmul2(eh[k], mhi), a3 = hmul2(oh[k], mhi);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * w + k], a0, a1, a2, a3, p0[H][nt], p1[H][nt]);
          }
        }
      };
      value_half(std::integral_constant<int, 0>{});
      value_half(std::integral_constant<int, 1>{});
      __syncwarp();
      stage = stage == kAttStages - 1 ? 0 : stage + 1;
    }
    cp_async_wait<0>();

    // ---- the four warps' results into one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 16));
        if (g == 0) {
          row_m[warp][8 * nt + 2 * t + c] = m[nt][c];
          row_l[warp][8 * nt + 2 * t + c] = x;
        }
      }
    __syncwarp();
    if (lane == 0) warp_ref[warp] = ref + (ref - warp_first[warp] > kAttSpan - kAttQuiet ? 256 : 0);
    __syncthreads();  // (the rings are drained too: `join` takes their place)
    const int ref_all = max(max(warp_ref[0] & 255, warp_ref[1] & 255), max(warp_ref[2] & 255, warp_ref[3] & 255));
    const float back = exp2i(max(ref - ref_all, -149));  // (to the values' own size only when divided: the sums could overflow)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * nt + 2 * t + c;
        float top = row_m[0][r];
#pragma unroll
        for (int w = 1; w < kAttWarps; ++w) top = fmaxf(top, row_m[w][r]);
        const float f = m[nt][c] == -INFINITY ? 0.0f : ex2(__fsub_rn(m[nt][c], top));
        float2* dst = reinterpret_cast<float2*>(join + (warp * ROWS + r) * D + g * (D / 8));
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
          dst[k] = make_float2(__fmul_rn(__fmul_rn(o[nt][k][c], f), back), __fmul_rn(__fmul_rn(o[nt][k][2 + c], f), back));
      }
    // A row without a sum sees no key of the segment, or its infinite query made every score -infinity and it is NaN.
    auto empty = [&](int r) {
      bool none = true;
#pragma unroll
      for (int w = 0; w < kAttWarps; ++w) none &= row_l[w][r] == 0.0f;
      return none;
    };
    const bool again = __syncthreads_or((threadIdx.x < n_rows && empty(threadIdx.x)) || warp_ref[warp] >= 256);
    bool wide = false;
    const bool whole = tile0 == 0 && tile1 == seq.tiles;
    float* slot = P.partial + (2 * static_cast<int64_t>(blockIdx.x) + (opens ? 0 : 1)) * Shape::kSlot;
    if (__builtin_expect(again, 0)) {
      const AttSeq seq = att_seq<ROWS>(P, b);  // (read again: kept over the steps above, it would cost them registers)
      if (((warp_ref[0] | warp_ref[1] | warp_ref[2] | warp_ref[3]) & 256) != 0) {
        const int pos0 = seq.length - seq.queries + row0 / P.group, pos1 = seq.length - seq.queries + (row0 + n_rows - 1) / P.group;
        const int from = max(seq.lo + tile0 * kAttTile, P.window > 0 ? pos0 - P.window + 1 : 0);
        const int to = min(min(seq.lo + tile1 * kAttTile, seq.length), P.causal ? pos1 + 1 : seq.length);
        AttRange<D> range;
        const uint64_t part = segment_range<D>(P, b, head, from, to, warp);
        if (lane == 0) red[warp] = static_cast<int64_t>(part);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) range.add(static_cast<uint32_t>(red[w] >> 32), static_cast<uint32_t>(red[w]));
        wide = range.wide();
      }
      for (int r = warp; r < n_rows; r += kAttWarps) {
        if (!wide && !empty(r)) continue;
        const int i_q = (row0 + r) / P.group, h = head * P.group + (row0 + r) - i_q * P.group;
        const int pos = seq.length - seq.queries + i_q;
        const int from = max(seq.lo + tile0 * kAttTile, P.window > 0 ? pos - P.window + 1 : 0);
        const int to = min(min(seq.lo + tile1 * kAttTile, seq.length), P.causal ? pos + 1 : seq.length);
        float v[D / 32];
        const float lse2 = row_wide<BF16, D>(
            P, b, head, static_cast<const uint16_t*>(P.query) + static_cast<int64_t>(seq.q0 + i_q) * P.q_token + static_cast<int64_t>(h) * P.q_head,
            from, to, v);
        const int64_t row = static_cast<int64_t>(seq.q0 + i_q) * P.heads + h;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const int d = lane * (D / 32) + c;
          if (whole)
            att_store<BF16>(P.out, row * D + d, __fmul_rn(v[c], kAttWideUnit));
          else
            slot[r * D + d] = __fmul_rn(v[c], kAttWideUnit * kAttPartial);
        }
        if (lane == 0) {
          if (!whole)
            slot[ROWS * D + r] = lse2;
          else if (P.lse)
            P.lse[row] = __fmul_rn(lse2, 0.69314718055994531f);
        }
      }
    }
    for (int i = threadIdx.x; i < n_rows * D && !wide; i += kAttThreads) {
      const int r = i / D, d = i % D;
      float top = row_m[0][r];
#pragma unroll
      for (int w = 1; w < kAttWarps; ++w) top = fmaxf(top, row_m[w][r]);
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttWarps; ++w) {
        const float f = row_m[w][r] == -INFINITY ? 0.0f : ex2(__fsub_rn(row_m[w][r], top));
        sum = __fadd_rn(sum, __fmul_rn(row_l[w][r], f));
        acc = __fadd_rn(acc, join[(w * ROWS + r) * D + d]);
      }
      if (empty(r)) continue;  // (done above)
      const float v = __fdiv_rn(acc, sum);
      const int unit = ref_all - 140;  // exponent of the values' unit
      const float lse2 = __fadd_rn(top, __fsub_rn(log2f(sum), kAttLift));
      if (whole) {
        const int i_q = (row0 + r) / P.group;
        const int64_t row = static_cast<int64_t>(seq.q0 + i_q) * P.heads + head * P.group + (row0 + r) - i_q * P.group;
        att_store<BF16>(P.out, row * D + d, __fmul_rn(v, exp2i(unit)));
        if (P.lse && d == 0) P.lse[row] = __fmul_rn(lse2, 0.69314718055994531f);
      } else {
        slot[r * D + d] = __fmul_rn(v, exp2i(unit - 4));  // (kAttPartial)
        if (d == 0) slot[ROWS * D + r] = lse2;
      }
    }
    __syncthreads();
  }
}

// Adds the partial results of a unit that several blocks shared, in block order.
template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(kAttJoinThreads) attention_join_kernel(const AttParams P, int blocks) {
  using Shape = AttShape<D, NT>;
  constexpr int ROWS = Shape::kRows;
  constexpr int CHUNK = 64;  // partial results whose weights are held at a time
  constexpr int QUADS = ROWS * D / 4, EACH = (QUADS + kAttJoinThreads - 1) / kAttJoinThreads;
  __shared__ int64_t red[kAttJoinThreads / 32];
  __shared__ float weight[CHUNK][ROWS];
  __shared__ float row_top[ROWS], row_sum[ROWS];
  const int b = blockIdx.y;
  const AttSeq seq = att_seq<ROWS>(P, b);
  const int64_t units = static_cast<int64_t>(seq.row_groups) * P.kv_heads;
  int64_t total = 0, before = 0;
  if (blockIdx.x < units) att_totals<ROWS, kAttJoinThreads>(P, b, red, total, before);
  // Every block waits, also those without work: what follows this kernel in the
  // stream may then rely on the first kernel's results too.
  grid_dependency_wait();
  // (The grid has a block per unit when the caller's bound on the queries holds.)
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const AttShares shares(total, blocks);
    const int64_t u0 = before + unit * (seq.tiles + kAttStart), u1 = u0 + seq.tiles + kAttStart;
    const int64_t j0 = shares.block_of(u0 + kAttStart), j1 = shares.block_of(u1 - 1) + 1;  // the blocks that share its tiles
    if (j1 - j0 == 1) continue;  // one block had it all
    // A block's partial result is in its first slot when its share starts with this unit.
    const float* first = P.partial + (2 * j0 + (u0 <= shares.first(j0) ? 0 : 1)) * Shape::kSlot;
    auto slot = [&](int64_t j) { return j == j0 ? first : P.partial + 2 * j * Shape::kSlot; };
    const int n = static_cast<int>(j1 - j0);
    const int row0 = static_cast<int>(unit % seq.row_groups) * ROWS, head = static_cast<int>(unit / seq.row_groups);
    const int n_rows = min(ROWS, seq.queries * P.group - row0);
    // Each row's largest log-sum, by 256 / ROWS threads.
    __syncthreads();
    if (threadIdx.x < ROWS * 16) {
      const int r = threadIdx.x >> 4;
      float top = -INFINITY;
      bool bad = false;
      for (int k = threadIdx.x & 15; k < n; k += 16) {
        const float x = slot(j0 + k)[ROWS * D + r];
        bad |= x != x;
        top = fmaxf(top, x);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        bad |= __shfl_xor_sync(0xffffffffu, static_cast<int>(bad), o) != 0;
      }
      if ((threadIdx.x & 15) == 0) {
        row_top[r] = bad ? NAN : top;
        row_sum[r] = 0.0f;
      }
    }
    float4 acc[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = 0; c0 < n; c0 += CHUNK) {
      const int nc = min(CHUNK, n - c0);
      __syncthreads();
      for (int i = threadIdx.x; i < nc * ROWS; i += kAttJoinThreads) {
        const int k = i / ROWS, r = i % ROWS;
        const float x = slot(j0 + c0 + k)[ROWS * D + r];
        weight[k][r] = x == -INFINITY ? 0.0f : ex2(__fsub_rn(x, row_top[r]));
      }
      __syncthreads();
      if (threadIdx.x < ROWS) {
        float sum = row_sum[threadIdx.x];
        for (int k = 0; k < nc; ++k) sum = __fadd_rn(sum, weight[k][threadIdx.x]);
        row_sum[threadIdx.x] = sum;
      }
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = threadIdx.x + e * kAttJoinThreads;
        const int r = i / (D / 4);
        if (i < QUADS && r < n_rows) {
#pragma unroll 8
          for (int k = 0; k < nc; ++k) {
            const float4 v = reinterpret_cast<const float4*>(slot(j0 + c0 + k))[i];
            const float w = weight[k][r];
            acc[e].x = __fmaf_rn(v.x, w, acc[e].x);
            acc[e].y = __fmaf_rn(v.y, w, acc[e].y);
            acc[e].z = __fmaf_rn(v.z, w, acc[e].z);
            acc[e].w = __fmaf_rn(v.w, w, acc[e].w);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = threadIdx.x + e * kAttJoinThreads;
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      if (i < QUADS && r < n_rows) {
        const float sum = row_sum[r];
        const bool seen = !(sum == 0.0f);
        const int i_q = (row0 + r) / P.group;
        const int64_t row = static_cast<int64_t>(seq.q0 + i_q) * P.heads + head * P.group + (row0 + r) - i_q * P.group;
        const float v[4] = {acc[e].x, acc[e].y, acc[e].z, acc[e].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) att_store<BF16>(P.out, row * D + d + k, seen ? __fmul_rn(__fdiv_rn(v[k], sum), 1.0f / kAttPartial) : 0.0f);
        if (P.lse && d == 0) P.lse[row] = seen ? __fmul_rn(__fadd_rn(row_top[r], log2f(sum)), 0.69314718055994531f) : -INFINITY;
      }
    }
  }
}

// -------------------------------------------------------------------- host

struct AttPlan {
  int nt;            // groups of eight rows per unit
  int64_t units;     // at most, per sequence
  unsigned blocks;
  bool whole;        // no unit is shared
  size_t bytes;      // of the workspace
};

// Bounds that the caller states (the longest sequence, the most queries of one)
// fix the launch; the kernels read the true lengths.
static AttPlan att_plan(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_length,
                        int64_t max_queries, int64_t window) {
  AttPlan plan{};
  const int64_t group = heads / kv_heads, rows = max_queries * group;
  plan.nt = rows <= 8 ? 1 : 2;
  const int64_t unit_rows = 8 * plan.nt;
  plan.units = (rows + unit_rows - 1) / unit_rows * kv_heads;
  // (A window's keys start anywhere in a tile.)
  const int64_t reach = window > 0 ? std::min(max_length, window + max_queries + kAttTile) : max_length;
  const int64_t deep = std::max<int64_t>(1, (reach + kAttTile - 1) / kAttTile), units = plan.units * seqs;
  const int64_t slots = static_cast<int64_t>(num_sms()) * (plan.nt == 1 ? 4 : 3);
  plan.whole = deep <= kAttWhole && deep * (slots - std::min(slots, units)) <= kAttWholeFew * slots;
  // At most 64 blocks per unit: joining more partial results costs what the split saves.
  const int64_t tiles = (plan.whole ? 1 : std::min<int64_t>(deep, 64)) * units;
  plan.blocks = static_cast<unsigned>(std::min<int64_t>(tiles, slots));
  plan.bytes = plan.whole ? 16 : static_cast<size_t>(plan.blocks) * 2 * static_cast<size_t>(unit_rows * dim + unit_rows) * sizeof(float);
  return plan;
}

template <bool BF16, int D, int NT>
static int launch_attention(const AttParams& P, const AttPlan& plan, cudaStream_t s) {
  auto kernel = attention_kernel<BF16, D, NT>;
  static std::atomic<uint64_t> done{0};
  int status = set_max_smem_once(reinterpret_cast<const void*>(kernel), AttShape<D, NT>::kSmem, done);
  if (status != MXW_OK) return status;
  kernel<<<plan.blocks, kAttThreads, AttShape<D, NT>::kSmem, s>>>(P);
  status = check_launch();
  if (status != MXW_OK || plan.whole) return status;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.units), static_cast<unsigned>(P.seqs));
  cfg.blockDim = dim3(kAttJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, attention_join_kernel<BF16, D, NT>, P, static_cast<int>(plan.blocks));
  return err == cudaSuccess ? MXW_OK : record_cuda_error(err);
}

template <bool BF16, int D>
static int launch_attention_rows(const AttParams& P, const AttPlan& plan, cudaStream_t s) {
  return plan.nt == 1 ? launch_attention<BF16, D, 1>(P, plan, s) : launch_attention<BF16, D, 2>(P, plan, s);
}

static bool att_shape_ok(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_length,
                         int64_t max_queries) {
  if (dim != 64 && dim != 128) return false;
  if (kv_heads < 1 || kv_heads > 1024 || heads < kv_heads || heads % kv_heads != 0 || heads > 65536) return false;
  return seqs >= 0 && max_length >= 0 && max_length <= 0x7fffff00 && max_queries >= 0 && max_queries <= 0x7fffffff / heads;
}

}  // namespace mxw

using namespace mxw;

extern "C" size_t mxw_paged_attention_workspace_size(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t dim,
                                                     int64_t max_length, int64_t max_queries) {
  if (!att_shape_ok(seqs, heads, kv_heads, dim, max_length, max_queries) || seqs == 0) return 0;
  max_queries = std::max<int64_t>(max_queries, 1);  // (0 may be wrong too: the starts decide)
  if (attention_prompt_fits(seqs, heads, kv_heads, max_queries)) return 16;  // nothing is shared between blocks
  return att_plan(seqs, heads, kv_heads, dim, max_length, max_queries, 0).bytes;  // (a window needs no more)
}

extern "C" int mxw_paged_attention(const void* query, int dtype, int64_t tokens, int64_t heads, int64_t q_token,
                                   int64_t q_head, const uint8_t* codes, const uint8_t* scales, int64_t pages,
                                   int64_t kv_heads, int64_t page_tokens, int64_t dim, const int32_t* table,
                                   int64_t table_ld, int64_t table_width, const int32_t* lengths, const int32_t* start,
                                   int64_t seqs, int64_t max_length, int64_t max_queries, double softmax_scale,
                                   int causal, int64_t window, void* out, float* lse, void* workspace,
                                   size_t workspace_bytes, uint32_t* flags, void* stream) {
  if (!att_shape_ok(seqs, heads, kv_heads, dim, max_length, max_queries) || tokens < 0) return MXW_EINVAL;
  if (dtype != MXW_BF16 && dtype != MXW_F16) return MXW_EINVAL;
  if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128) return MXW_EINVAL;
  if (pages < 0 || pages > 0x7fffffff || table_width < 0 || (seqs > 1 && table_ld < table_width)) return MXW_EINVAL;
  if (q_token < 0 || q_head < 0 || window < 0 || (window > 0 && !causal)) return MXW_EINVAL;
  if (!(softmax_scale > 0.0) || !std::isfinite(softmax_scale)) return MXW_EINVAL;
  if (tokens == 0) return MXW_OK;
  if (!query || !out || reinterpret_cast<uintptr_t>(out) % 16 != 0) return MXW_EINVAL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (seqs == 0) {
    // Every row is one that no key reaches.
    return lse ? MXW_EUNSUPPORTED
               : (cudaMemsetAsync(out, 0, static_cast<size_t>(tokens * heads * dim) * 2, s) == cudaSuccess
                      ? MXW_OK
                      : record_cuda_error(cudaGetLastError()));
  }
  max_queries = std::max<int64_t>(max_queries, 1);
  if (!codes || !scales || !lengths || !start || (table_width > 0 && !table)) return MXW_EINVAL;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return MXW_EINVAL;
  const AttPlan plan = att_plan(seqs, heads, kv_heads, dim, max_length, max_queries, std::min<int64_t>(window, 0x3fffffff));
  const bool prompt = attention_prompt_fits(seqs, heads, kv_heads, max_queries);
  if (!prompt && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < plan.bytes)) return MXW_EINVAL;
  if (seqs > 65535 || plan.units > 0x7fffffff || tokens > 0x7fffffff) return MXW_EUNSUPPORTED;
  AttParams P{};
  P.query = query;
  P.q_token = q_token;
  P.q_head = q_head;
  P.codes = codes;
  P.scales = scales;
  P.pages = pages;
  P.table = table;
  P.table_ld = table_ld;
  P.table_width = std::min<int64_t>(table_width, 0x7fffff00 / page_tokens);
  P.lengths = lengths;
  P.start = start;
  P.tokens = tokens;
  P.q_vec = q_token % 8 == 0 && q_head % 8 == 0 && reinterpret_cast<uintptr_t>(query) % 16 == 0;
  P.seqs = static_cast<int>(seqs);
  P.heads = static_cast<int>(heads);
  P.kv_heads = static_cast<int>(kv_heads);
  P.group = static_cast<int>(heads / kv_heads);
  P.page_shift = page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
  P.scale_log2 = std::max(static_cast<float>(softmax_scale * 1.4426950408889634), 1e-37f);  // positive: it meets -infinity
  P.causal = causal ? 1 : 0;
  P.window = static_cast<int>(std::min<int64_t>(window, 0x3fffffff));
  P.out = out;
  P.lse = lse;
  P.partial = static_cast<float*>(workspace);
  P.whole = plan.whole;
  P.flags = flags;
  if (prompt) return launch_attention_prompt(P, dtype == MXW_BF16, static_cast<int>(dim), max_queries, s);
  if (dtype == MXW_BF16)
    return dim == 128 ? launch_attention_rows<true, 128>(P, plan, s) : launch_attention_rows<true, 64>(P, plan, s);
  return dim == 128 ? launch_attention_rows<false, 128>(P, plan, s) : launch_attention_rows<false, 64>(P, plan, s);
}
