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
//   * The contraction's order is free, so each lane takes the bytes that lie
//     together in a cached row: for K four lanes share a row (a quarter of it
//     each), for V eight lanes do, and token pairs are interleaved nibble by
//     nibble.  Every shared-memory load is 8 or 16 bytes without conflicts.
//   * A byte of two codes becomes an f16 pair in one conversion, and one f16x2
//     product applies the scale.  f16 has 11 significant bits where a code has
//     two; what it lacks is range, so scales are taken relative to a running
//     reference: the largest of the row's blocks for a key, the largest seen so
//     far for the values (times 2^13, below f16's maximum).  A block whose scale
//     is 2^-36 of the reference or more is exact; smaller ones lose bits that
//     are 2^-37 of the reference.  Queries are exact in the same sense (scaled
//     by a power of two per row for bf16).
//   * Probabilities are rounded to f16 as 2^(x - m + 7): 11 bits down to 2^-21
//     of the largest, nothing lost above 2^-31.  Their sum is taken in fp32
//     before the rounding.  m is raised only when a score passes it by 8
//     (binary), which spares most tiles the reduction and the rescaling.
//   * Four warps of a block take tiles of 16 keys in turn, each with its own
//     running maximum and sum, its own ring of asynchronous copies and no
//     synchronisation with the others until the end of a segment.
// Work split: the (sequence, head, row group) units are cut into tiles of 64
// keys, all tiles are laid end to end, and each block takes an equal share of
// them, whatever the lengths.  A unit that several blocks share leaves partial
// results (normalised rows and their log-sum-exp) in the workspace, two slots
// per block, and attention_join_kernel adds them in block order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "blockscale.cuh"
#include "common.cuh"
#include "runtime.h"

namespace mxw {

constexpr int kAttWarps = 4;
constexpr int kAttThreads = kAttWarps * 32;
constexpr int kAttKeys = 16;                      // keys per warp step
constexpr int kAttTile = kAttWarps * kAttKeys;    // keys per block step
constexpr int kAttStages = 4;
constexpr float kAttLift = 7.0f;    // probabilities are held as 2^(x - m + 7)
constexpr float kAttSlack = 8.0f;   // and x may pass m by 8 before m is raised: at most 2^15

struct AttParams {
  const void* query;
  int64_t q_token, q_head;  // strides in elements
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t pages;
  const int32_t* table;
  int64_t table_ld, table_width;
  const int32_t* lengths;
  const int32_t* start;
  int64_t tokens;
  int seqs, heads, kv_heads, group, page_shift;
  float scale_log2;  // softmax scale times log2(e)
  int causal, window;
  void* out;   // [tokens][heads][dim]
  float* lse;  // [tokens][heads] or null
  float* partial;
};

// One sequence's share of the work.
struct AttSeq {
  int q0, queries;  // its rows of the packed queries
  int length;       // cached tokens
  int lo;           // first key that some query sees, rounded down to a tile step
  int tiles;        // tiles of 64 keys from lo on, at least one
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
  return static_cast<int64_t>(s.tiles) * s.row_groups * P.kv_heads;
}

// Sum over the block (all threads get it); `red` holds one word per warp.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t sum = 0;
#pragma unroll
  for (int w = 0; w < kAttWarps; ++w) sum += red[w];
  return sum;
}

// All tiles, and the tiles of the sequences before `upto`.
template <int ROWS>
__device__ __forceinline__ void att_totals(const AttParams& P, int upto, int64_t* red, int64_t& total, int64_t& before) {
  int64_t all = 0, part = 0;
  for (int b = threadIdx.x; b < P.seqs; b += kAttThreads) {
    const int64_t w = att_work(P, att_seq<ROWS>(P, b));
    all += w;
    if (b < upto) part += w;
  }
  total = block_sum(all, red);
  before = block_sum(part, red);
}

__device__ __forceinline__ int64_t att_first_tile(int64_t total, int64_t block, int64_t blocks) {
  return total / blocks * block + total % blocks * block / blocks;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
  return h;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 2^(13 - n) as f16 bits for n >= 0: normal down to 2^-14, subnormal to 2^-24, then 0.
__device__ __forceinline__ uint32_t f16_pow2_13_minus(int n) {
  return n <= 27 ? static_cast<uint32_t>(28 - n) << 10 : 0x400u >> min(n - 27, 31);
}

// The f16 pair of byte q of a word.
#define MXW_PAIR(word, q) e2m1x2_to_f16x2((word) >> (8 * (q)))

template <int D, int NT>
struct AttShape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kCodes = kAttKeys * D / 2;    // bytes of 16 rows
  static constexpr int kScales = kAttKeys * D / 32;
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kRing = kAttStages * kStage;
  static constexpr int kJoin = kAttWarps * kRows * D * 4;  // fp32 rows of each warp
  static constexpr int kSmem = kAttWarps * kRing + kJoin;
  static constexpr int kBlocks = NT == 1 ? 4 : 3;  // per SM: 128 and 168 registers a thread
  static constexpr int kSlot = kRows * D + kRows;  // floats of a partial result
};

template <bool BF16>
__device__ __forceinline__ float att_load_q(const void* q, int64_t i) {
  const uint16_t b = static_cast<const uint16_t*>(q)[i];
  return BF16 ? bits_f32(static_cast<uint32_t>(b) << 16) : __half2float(*reinterpret_cast<const __half*>(&b));
}
template <bool BF16>
__device__ __forceinline__ void att_store(void* p, int64_t i, float v) {
  if constexpr (BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Rows of `out` that no sequence covers: zeros.
template <bool BF16>
__device__ __forceinline__ void att_clear_rest(const AttParams& P, int dim) {
  const int64_t first = max(static_cast<int64_t>(0), min(static_cast<int64_t>(P.start[0]), P.tokens));
  const int64_t last = max(first, min(static_cast<int64_t>(P.start[P.seqs]), P.tokens));
  const int64_t width = static_cast<int64_t>(P.heads) * dim, rest = P.tokens - (last - first);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kAttThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kAttThreads + threadIdx.x; i < rest * width; i += step) {
    const int64_t r = i / width, token = r < first ? r : last + r - first;
    att_store<BF16>(P.out, token * width + i % width, 0.0f);
    if (P.lse && i % width < P.heads) P.lse[token * P.heads + i % width] = -INFINITY;
  }
}

template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, AttShape<D, NT>::kBlocks) attention_kernel(const AttParams P) {
  using Shape = AttShape<D, NT>;
  constexpr int ROWS = Shape::kRows;
  constexpr int QREGS = D / 8;       // f16 pairs of a query row per lane
  constexpr int STEPS = D / 16;      // k16 steps of S, and 16-channel groups of O
  extern __shared__ __align__(128) uint8_t att_smem[];
  __shared__ int64_t red[kAttWarps];
  __shared__ float row_m[kAttWarps][ROWS], row_l[kAttWarps][ROWS];
  grid_dependents_launch();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = att_smem + warp * Shape::kRing;
  float* join = reinterpret_cast<float*>(att_smem + kAttWarps * Shape::kRing);  // [warp][row][D]
  const uint32_t ring_s = smem_u32(ring);

  att_clear_rest<BF16>(P, D);
  int64_t total, ignored;
  att_totals<ROWS>(P, 0, red, total, ignored);
  int64_t at = att_first_tile(total, blockIdx.x, gridDim.x);
  const int64_t end = att_first_tile(total, blockIdx.x + 1ll, gridDim.x);
  if (at >= end) return;

  // The sequence that holds the first tile.
  int b = 0;
  int64_t rem = at;
  AttSeq seq = att_seq<ROWS>(P, 0);
  {
    // Skip 32 sequences at a time: every warp does the same.
    for (; b < P.seqs; b += 32) {
      int64_t w = b + lane < P.seqs ? att_work(P, att_seq<ROWS>(P, b + lane)) : 0;
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
    seq = att_seq<ROWS>(P, b);
  }

  bool first_segment = true;
  while (at < end) {
    while (rem >= att_work(P, seq)) {
      rem -= att_work(P, seq);
      seq = att_seq<ROWS>(P, ++b);
    }
    const int64_t unit = rem / seq.tiles;
    const int tile0 = static_cast<int>(rem % seq.tiles);
    const int tile1 = static_cast<int>(min(static_cast<int64_t>(seq.tiles), tile0 + (end - at)));
    const int head = static_cast<int>(unit / seq.row_groups);  // key/value head
    const int row0 = static_cast<int>(unit % seq.row_groups) * ROWS;
    const int n_rows = min(ROWS, seq.queries * P.group - row0);

    // ---- queries: row n = 8 nt + g of this lane, elements [t D/4, (t + 1) D/4)
    uint32_t q[NT][QREGS];
    float fq[NT][2];        // score factors of rows 2t and 2t + 1
    int key_lo[NT][2], key_hi[NT][2];  // and the keys they see
    int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 8 * nt + g;
      const bool on = r < n_rows;
      const int i = on ? (row0 + r) / P.group : 0;
      const int h = head * P.group + (on ? (row0 + r) % P.group : 0);
      const int64_t base = static_cast<int64_t>(seq.q0 + i) * P.q_token + static_cast<int64_t>(h) * P.q_head + t * (D / 4);
      float v[D / 4];
      uint32_t amax = 0;
#pragma unroll
      for (int k = 0; k < D / 4; ++k) {
        v[k] = on ? att_load_q<BF16>(P.query, base + k) : 0.0f;
        amax = max(amax, f32_bits(v[k]) & 0x7fffffffu);
      }
      float f = P.scale_log2;
      float up = 1.0f;
      if constexpr (BF16) {
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // The row's largest magnitude to [2^14, 2^15): exact in f16 down to 2^-31 of it.
        const int e = max(static_cast<int>(amax >> 23), 1) - 127 - 14;
        up = exp2i(min(-e, 127));
        f = __fmul_rn(f, exp2i(-min(-e, 127)));
      }
#pragma unroll
      for (int k = 0; k < QREGS; ++k) q[nt][k] = pack_f16x2(__fmul_rn(v[2 * k], up), __fmul_rn(v[2 * k + 1], up));
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
    {
      // Bounds over the rows of the unit: a query's position grows with its row.
      const int pos0 = seq.length - seq.queries + row0 / P.group;
      const int pos1 = seq.length - seq.queries + (row0 + n_rows - 1) / P.group;
      lo_min = P.window > 0 ? max(0, pos0 - P.window + 1) : 0;
      lo_max = P.window > 0 ? max(0, pos1 - P.window + 1) : 0;
      hi_max = P.causal ? max(0, min(pos1 + 1, seq.length)) : seq.length;
      hi_min = P.causal ? max(0, pos0 + 1) : seq.length;  // rows past n_rows are never stored: any mask will do
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

    // ---- this warp's steps: tiles of 16 keys, every fourth of the segment
    const int key0 = seq.lo + tile0 * kAttTile + warp * kAttKeys;
    const int key_end = min(seq.lo + tile1 * kAttTile, hi_max);
    int skip = 0;
    if (lo_min > key0) skip = (lo_min - key0) / kAttTile;  // steps that end before the window
    const int steps = key_end > key0 ? (key_end - key0 + kAttTile - 1) / kAttTile : 0;
    const int32_t* table = P.table + static_cast<int64_t>(b) * P.table_ld;
    const int page_mask = (1 << P.page_shift) - 1;

    auto page_of = [&](int step) -> int {
      const int key = key0 + step * kAttTile;
      return step < steps ? table[key >> P.page_shift] : -1;
    };
    // Copies the 16 rows of a step into its stage; false when its page is not one of the pool's.
    auto issue = [&](int step, int page) -> bool {
      const bool ok = step < steps && static_cast<uint32_t>(page) < static_cast<uint64_t>(P.pages);
      if (ok) {
        const int key = key0 + step * kAttTile;
        const int64_t row = ((static_cast<int64_t>(page) * 2 * P.kv_heads + head) << P.page_shift) + (key & page_mask);
        const int64_t value = static_cast<int64_t>(P.kv_heads) << P.page_shift;  // rows from a key to its value
        const uint32_t st = ring_s + (step % kAttStages) * Shape::kStage;
        const uint8_t* kc = P.codes + row * (D / 2);
        const uint8_t* vc = kc + value * (D / 2);
#pragma unroll
        for (int k = 0; k < Shape::kCodes / 512; ++k) {
          const int c = k * 32 + lane;
          cp_async<16>(st + c * 16, kc + c * 16, 16);
          // Value rows four apart would meet in the same banks: swap the halves of every other four rows.
          const int vd = D == 128 ? (c ^ (((c >> 4) & 1) << 1)) : c;
          cp_async<16>(st + Shape::kCodes + vd * 16, vc + c * 16, 16);
        }
        constexpr int SC = Shape::kScales / 16;
        if (lane < 2 * SC) {
          const bool is_v = lane >= SC;
          const uint8_t* sc = P.scales + (row + (is_v ? value : 0)) * (D / 32) + (lane - (is_v ? SC : 0)) * 16;
          cp_async<16>(st + 2 * Shape::kCodes + lane * 16, sc, 16);
        }
      }
      cp_async_commit();
      return ok;
    };

    uint32_t valid = 0;  // one bit per stage
    int next_page = page_of(skip);
#pragma unroll
    for (int k = 0; k < kAttStages - 1; ++k) {
      const int page = next_page;
      next_page = page_of(skip + k + 1);
      const bool ok = issue(skip + k, page);
      const uint32_t bit = 1u << ((skip + k) % kAttStages);
      valid = ok ? valid | bit : valid & ~bit;
    }

    const int tok_a = g ^ ((g >> 1) & 1);  // key of row g of S^T (row g + 8: 8 further on)
    const int v_a = (2 * t) ^ (t & 1), v_b = (2 * t + 1) ^ (t & 1);  // keys of the contraction's slots 2t, 2t + 1

    for (int step = skip; step < steps; ++step) {
      {
        const int page = next_page;
        next_page = page_of(step + kAttStages);
        const bool ok = issue(step + kAttStages - 1, page);
        const uint32_t bit = 1u << ((step + kAttStages - 1) % kAttStages);
        valid = ok ? valid | bit : valid & ~bit;
      }
      cp_async_wait<kAttStages - 1>();
      __syncwarp();
      const int stage = step % kAttStages;
      const int key = key0 + step * kAttTile;
      if ((valid >> stage) & 1) {
        const uint8_t* st = ring + stage * Shape::kStage;
        const uint8_t* kc = st;
        const uint8_t* vc = st + Shape::kCodes;
        const uint8_t* ks = st + 2 * Shape::kCodes;
        const uint8_t* vs = ks + Shape::kScales;

        // ---- scores
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[nt][c] = 0.0f;
        constexpr int KW = D / 32;  // words of a row's quarter
        uint32_t wa[KW], wb[KW];
        if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(wa) = *reinterpret_cast<const uint4*>(kc + tok_a * 64 + t * 16);
          *reinterpret_cast<uint4*>(wb) = *reinterpret_cast<const uint4*>(kc + (tok_a + 8) * 64 + t * 16);
        } else {
          *reinterpret_cast<uint2*>(wa) = *reinterpret_cast<const uint2*>(kc + tok_a * 32 + t * 8);
          *reinterpret_cast<uint2*>(wb) = *reinterpret_cast<const uint2*>(kc + (tok_a + 8) * 32 + t * 8);
        }
        constexpr int BLOCKS = D / 32;
        const int sa = ks[tok_a * BLOCKS + t * BLOCKS / 4], sb = ks[(tok_a + 8) * BLOCKS + t * BLOCKS / 4];
        int ra = max(sa, __shfl_xor_sync(0xffffffffu, sa, 1));
        int rb = max(sb, __shfl_xor_sync(0xffffffffu, sb, 1));
        ra = max(ra, __shfl_xor_sync(0xffffffffu, ra, 2));
        rb = max(rb, __shfl_xor_sync(0xffffffffu, rb, 2));
        const uint32_t ma = f16_pow2_13_minus(ra - sa) * 0x10001u, mb = f16_pow2_13_minus(rb - sb) * 0x10001u;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = hmul2(MXW_PAIR(wa[w], 2 * h), ma), a1 = hmul2(MXW_PAIR(wb[w], 2 * h), mb);
            const uint32_t a2 = hmul2(MXW_PAIR(wa[w], 2 * h + 1), ma), a3 = hmul2(MXW_PAIR(wb[w], 2 * h + 1), mb);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(s[nt], a0, a1, a2, a3, q[nt][4 * w + 2 * h], q[nt][4 * w + 2 * h + 1]);
          }
        const float fa = exp2i(ra - 140), fb = exp2i(rb - 140);
        const int key_a = key + tok_a, key_b = key_a + 8;
        bool raise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[nt][0] = __fmul_rn(__fmul_rn(s[nt][0], fa), fq[nt][0]);
          s[nt][1] = __fmul_rn(__fmul_rn(s[nt][1], fa), fq[nt][1]);
          s[nt][2] = __fmul_rn(__fmul_rn(s[nt][2], fb), fq[nt][0]);
          s[nt][3] = __fmul_rn(__fmul_rn(s[nt][3], fb), fq[nt][1]);
        }
        const bool edge = key < lo_max || key + kAttKeys > hi_min;
        if (edge) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              if (key_a < key_lo[nt][c] || key_a >= key_hi[nt][c]) s[nt][c] = -INFINITY;
              if (key_b < key_lo[nt][c] || key_b >= key_hi[nt][c]) s[nt][2 + c] = -INFINITY;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) raise |= fmaxf(s[nt][c], s[nt][2 + c]) > __fadd_rn(m[nt][c], kAttSlack);
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = fmaxf(s[nt][c], s[nt][2 + c]);
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
        }

        // ---- probabilities, transposed into the second product's operand
        uint32_t p0[NT], p1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float base = __fsub_rn(kAttLift, m[nt][c] == -INFINITY ? 0.0f : m[nt][c]);
            p[c] = ex2(__fadd_rn(s[nt][c], base));
            p[2 + c] = ex2(__fadd_rn(s[nt][2 + c], base));
            l[nt][c] = __fadd_rn(l[nt][c], __fadd_rn(p[c], p[2 + c]));
          }
          p0[nt] = transpose8(pack_f16x2(p[0], p[1]));
          p1[nt] = transpose8(pack_f16x2(p[2], p[3]));
        }

        // ---- values
        constexpr int VW = D / 64;  // words of an eighth of a row
        uint32_t va[VW], vb[VW], vc2[VW], vd[VW];
        if constexpr (D == 128) {
          const int sw = (t & 2) << 4;  // rows 4..7 and 12..15 of the stage have their halves swapped
          const int ch = (g * 8) ^ sw;
          *reinterpret_cast<uint2*>(va) = *reinterpret_cast<const uint2*>(vc + v_a * 64 + ch);
          *reinterpret_cast<uint2*>(vb) = *reinterpret_cast<const uint2*>(vc + v_b * 64 + ch);
          *reinterpret_cast<uint2*>(vc2) = *reinterpret_cast<const uint2*>(vc + (v_a + 8) * 64 + ch);
          *reinterpret_cast<uint2*>(vd) = *reinterpret_cast<const uint2*>(vc + (v_b + 8) * 64 + ch);
        } else {
          va[0] = *reinterpret_cast<const uint32_t*>(vc + v_a * 32 + g * 4);
          vb[0] = *reinterpret_cast<const uint32_t*>(vc + v_b * 32 + g * 4);
          vc2[0] = *reinterpret_cast<const uint32_t*>(vc + (v_a + 8) * 32 + g * 4);
          vd[0] = *reinterpret_cast<const uint32_t*>(vc + (v_b + 8) * 32 + g * 4);
        }
        const int blk = g * BLOCKS / 8;
        int s0 = vs[v_a * BLOCKS + blk], s1 = vs[v_b * BLOCKS + blk];
        int s2 = vs[(v_a + 8) * BLOCKS + blk], s3 = vs[(v_b + 8) * BLOCKS + blk];
        if (edge) {
          // Keys that no row sees (stale rows of the page) have no say in the reference.
          if (key + v_a < lo_min || key + v_a >= hi_max) s0 = 0;
          if (key + v_b < lo_min || key + v_b >= hi_max) s1 = 0;
          if (key + v_a + 8 < lo_min || key + v_a + 8 >= hi_max) s2 = 0;
          if (key + v_b + 8 < lo_min || key + v_b + 8 >= hi_max) s3 = 0;
        }
        const int top = __reduce_max_sync(0xffffffffu, max(max(s0, s1), max(s2, s3)));
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
        const uint32_t mlo = f16_pow2_13_minus(ref - s0) | (f16_pow2_13_minus(ref - s1) << 16);
        const uint32_t mhi = f16_pow2_13_minus(ref - s2) | (f16_pow2_13_minus(ref - s3) << 16);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t el = (va[w] & 0x0f0f0f0fu) | ((vb[w] << 4) & 0xf0f0f0f0u);
          const uint32_t ol = ((va[w] >> 4) & 0x0f0f0f0fu) | (vb[w] & 0xf0f0f0f0u);
          const uint32_t eh = (vc2[w] & 0x0f0f0f0fu) | ((vd[w] << 4) & 0xf0f0f0f0u);
          const uint32_t oh = ((vc2[w] >> 4) & 0x0f0f0f0fu) | (vd[w] & 0xf0f0f0f0u);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a0 = hmul2(MXW_PAIR(el, k), mlo), a1 = hmul2(MXW_PAIR(ol, k), mlo);
            const uint32_t a2 = hmul2(MXW_PAIR(eh, k), mhi), a3 = hmul2(MXW_PAIR(oh, k), mhi);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * w + k], a0, a1, a2, a3, p0[nt], p1[nt]);
          }
        }
      }
      __syncwarp();
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
    __syncthreads();
    const float back = exp2i(max(ref - 140, -149));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = 8 * nt + 2 * t + c;
        float top = row_m[0][r];
#pragma unroll
        for (int w = 1; w < kAttWarps; ++w) top = fmaxf(top, row_m[w][r]);
        const float f = m[nt][c] == -INFINITY ? 0.0f : ex2(__fsub_rn(m[nt][c], top));
        float* dst = join + (warp * ROWS + r) * D + g * (D / 8);
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
          dst[2 * k] = __fmul_rn(__fmul_rn(o[nt][k][c], f), back);
          dst[2 * k + 1] = __fmul_rn(__fmul_rn(o[nt][k][2 + c], f), back);
        }
      }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == seq.tiles;
    float* slot = P.partial + (2 * static_cast<int64_t>(blockIdx.x) + (first_segment ? 0 : 1)) * Shape::kSlot;
    for (int i = threadIdx.x; i < ROWS * D; i += kAttThreads) {
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
      const bool seen = !(sum == 0.0f);  // NaN counts as seen
      const float v = seen ? __fdiv_rn(acc, sum) : 0.0f;
      const float lse2 = seen ? __fadd_rn(top, __fsub_rn(log2f(sum), kAttLift)) : -INFINITY;
      if (whole) {
        if (r < n_rows) {
          const int64_t row = static_cast<int64_t>(seq.q0 + (row0 + r) / P.group) * P.heads + head * P.group + (row0 + r) % P.group;
          att_store<BF16>(P.out, row * D + d, v);
          if (P.lse && d == 0) P.lse[row] = __fmul_rn(lse2, 0.69314718055994531f);
        }
      } else {
        slot[r * D + d] = v;
        if (d == 0) slot[ROWS * D + r] = lse2;
      }
    }
    __syncthreads();
    const int64_t taken = tile1 - tile0;
    at += taken;
    rem += taken;
    first_segment = false;
  }
}

// Adds the partial results of a unit that several blocks shared, in block order.
template <bool BF16, int D, int NT>
__global__ void __launch_bounds__(kAttThreads) attention_join_kernel(const AttParams P, int blocks) {
  using Shape = AttShape<D, NT>;
  constexpr int ROWS = Shape::kRows;
  __shared__ int64_t red[kAttWarps];
  const int b = blockIdx.y;
  const AttSeq seq = att_seq<ROWS>(P, b);
  const int64_t units = static_cast<int64_t>(seq.row_groups) * P.kv_heads;
  int64_t total = 0, before = 0;
  if (blockIdx.x < units) att_totals<ROWS>(P, b, red, total, before);
  // Every block waits, also those without work: what follows this kernel in the
  // stream may then rely on the first kernel's results too.
  grid_dependency_wait();
  // (The grid has a block per unit when the caller's bound on the queries holds.)
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
  const int64_t u0 = before + unit * seq.tiles, u1 = u0 + seq.tiles;  // its tiles
  // The block whose share holds tile u0.
  int64_t j = static_cast<int64_t>(static_cast<double>(u0) / static_cast<double>(total) * blocks);
  j = max(static_cast<int64_t>(0), min(j, static_cast<int64_t>(blocks) - 1));
  while (j > 0 && att_first_tile(total, j, blocks) > u0) --j;
  while (j + 1 < blocks && att_first_tile(total, j + 1, blocks) <= u0) ++j;
  if (att_first_tile(total, j + 1, blocks) >= u1) continue;  // one block had it all
  const int head = static_cast<int>(unit / seq.row_groups), row0 = static_cast<int>(unit % seq.row_groups) * ROWS;
  const int n_rows = min(ROWS, seq.queries * P.group - row0);
  for (int i = threadIdx.x; i < n_rows * D; i += kAttThreads) {
    const int r = i / D, d = i % D;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (int64_t k = j; k < blocks; ++k) {
      const int64_t first = att_first_tile(total, k, blocks);
      if (first >= u1) break;
      if (att_first_tile(total, k + 1, blocks) == first) continue;  // a block without work
      const float* slot = P.partial + (2 * k + (u0 <= first ? 0 : 1)) * Shape::kSlot;
      const float x = slot[ROWS * D + r];
      if (x == -INFINITY) continue;
      const float up = fmaxf(top, x);
      const float keep = top == up ? 1.0f : ex2(__fsub_rn(top, up));
      const float w = ex2(__fsub_rn(x, up));
      sum = __fadd_rn(__fmul_rn(sum, keep), w);
      acc = __fmaf_rn(slot[r * D + d], w, __fmul_rn(acc, keep));
      top = up;
    }
    const bool seen = !(sum == 0.0f);
    const int64_t row = static_cast<int64_t>(seq.q0 + (row0 + r) / P.group) * P.heads + head * P.group + (row0 + r) % P.group;
    att_store<BF16>(P.out, row * D + d, seen ? __fdiv_rn(acc, sum) : 0.0f);
    if (P.lse && d == 0) P.lse[row] = seen ? __fmul_rn(__fadd_rn(top, log2f(sum)), 0.69314718055994531f) : -INFINITY;
  }
  }
}

// -------------------------------------------------------------------- host

struct AttPlan {
  int nt;            // groups of eight rows per unit
  int64_t units;     // at most, per sequence
  unsigned blocks;
  size_t bytes;      // of the workspace
};

// Bounds that the caller states (the longest sequence, the most queries of one)
// fix the launch; the kernels read the true lengths.
static AttPlan att_plan(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_length,
                        int64_t max_queries) {
  AttPlan plan{};
  const int64_t group = heads / kv_heads, rows = max_queries * group;
  plan.nt = rows <= 8 ? 1 : 2;
  const int64_t unit_rows = 8 * plan.nt;
  plan.units = (rows + unit_rows - 1) / unit_rows * kv_heads;
  const int64_t tiles = std::max<int64_t>(1, (max_length + kAttTile) / kAttTile) * plan.units * seqs;
  plan.blocks = static_cast<unsigned>(std::min<int64_t>(tiles, static_cast<int64_t>(num_sms()) * (plan.nt == 1 ? 4 : 3)));
  plan.bytes = static_cast<size_t>(plan.blocks) * 2 * static_cast<size_t>(unit_rows * dim + unit_rows) * sizeof(float);
  return plan;
}

template <bool BF16, int D, int NT>
static int launch_attention(const AttParams& P, const AttPlan& plan, cudaStream_t s) {
  auto kernel = attention_kernel<BF16, D, NT>;
  int status = set_max_smem(reinterpret_cast<const void*>(kernel), AttShape<D, NT>::kSmem);
  if (status != MXW_OK) return status;
  kernel<<<plan.blocks, kAttThreads, AttShape<D, NT>::kSmem, s>>>(P);
  status = check_launch();
  if (status != MXW_OK) return status;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.units), static_cast<unsigned>(P.seqs));
  cfg.blockDim = dim3(kAttThreads);
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
  if (!att_shape_ok(seqs, heads, kv_heads, dim, max_length, max_queries) || seqs == 0 || max_queries == 0) return 0;
  return att_plan(seqs, heads, kv_heads, dim, max_length, max_queries).bytes;
}

extern "C" int mxw_paged_attention(const void* query, int dtype, int64_t tokens, int64_t heads, int64_t q_token,
                                   int64_t q_head, const uint8_t* codes, const uint8_t* scales, int64_t pages,
                                   int64_t kv_heads, int64_t page_tokens, int64_t dim, const int32_t* table,
                                   int64_t table_ld, int64_t table_width, const int32_t* lengths, const int32_t* start,
                                   int64_t seqs, int64_t max_length, int64_t max_queries, double softmax_scale,
                                   int causal, int64_t window, void* out, float* lse, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!att_shape_ok(seqs, heads, kv_heads, dim, max_length, max_queries) || tokens < 0) return MXW_EINVAL;
  if (dtype != MXW_BF16 && dtype != MXW_F16) return MXW_EINVAL;
  if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128) return MXW_EINVAL;
  if (pages < 0 || pages > 0x7fffffff || table_width < 0 || (seqs > 1 && table_ld < table_width)) return MXW_EINVAL;
  if (q_token < 0 || q_head < 0 || window < 0 || (window > 0 && !causal)) return MXW_EINVAL;
  if (!(softmax_scale > 0.0) || !std::isfinite(softmax_scale)) return MXW_EINVAL;
  if (tokens == 0) return MXW_OK;
  if (!query || !out) return MXW_EINVAL;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (seqs == 0 || max_queries == 0) {
    // No sequence has a query: every row is one that no key reaches.
    return lse ? MXW_EUNSUPPORTED
               : (cudaMemsetAsync(out, 0, static_cast<size_t>(tokens * heads * dim) * 2, s) == cudaSuccess
                      ? MXW_OK
                      : record_cuda_error(cudaGetLastError()));
  }
  if (!codes || !scales || !lengths || !start || (table_width > 0 && !table)) return MXW_EINVAL;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return MXW_EINVAL;
  const AttPlan plan = att_plan(seqs, heads, kv_heads, dim, max_length, max_queries);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < plan.bytes) return MXW_EINVAL;
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
  P.seqs = static_cast<int>(seqs);
  P.heads = static_cast<int>(heads);
  P.kv_heads = static_cast<int>(kv_heads);
  P.group = static_cast<int>(heads / kv_heads);
  P.page_shift = page_tokens == 16 ? 4 : page_tokens == 32 ? 5 : page_tokens == 64 ? 6 : 7;
  P.scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  P.causal = causal ? 1 : 0;
  P.window = static_cast<int>(std::min<int64_t>(window, 0x3fffffff));
  P.out = out;
  P.lse = lse;
  P.partial = static_cast<float*>(workspace);
  if (dtype == MXW_BF16)
    return dim == 128 ? launch_attention_rows<true, 128>(P, plan, s) : launch_attention_rows<true, 64>(P, plan, s);
  return dim == 128 ? launch_attention_rows<false, 128>(P, plan, s) : launch_attention_rows<false, 64>(P, plan, s);
}
