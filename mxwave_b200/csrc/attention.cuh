// What the attention kernels over the MXFP4 cache share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "f16mma.cuh"
#include "terms.cuh"

namespace mxw {

constexpr float kAttLift = 7.0f;    // probabilities are held as 2^(x - m + 7)
constexpr float kAttSlack = 8.0f;   // and x may pass m by 8 before m is raised: at most 2^15
// Both kernels hold values and probabilities in f16, relative to the largest of
// each.  A value is exact down to 2^-27 of the largest scale, and a probability
// keeps 2^-32 of its row's largest: good for any rows whose values' scales lie
// within kAttExact powers of two of one another, and those of the same 32
// channels within kAttSpan (the probability's part is then 2^-12 of the smallest
// scale).  Rows with a wider range are done again by att_row_wide, so that a key
// counts by its probability alone, and one that a row does not see not at all.
// That is a path for odd data (an overflowed value, say): it takes 11 ms where 32
// sequences of 1 to 65,536 keys take 0.19, and 137 where four prompts of up to
// 3001 tokens take 0.59.  The kernels only watch whether the range over all
// channels may exceed kAttSpan; AttRange then looks closer.
constexpr int kAttSpan = 20, kAttExact = 27;

// The bits of infinity in the queries' type; what has more is NaN.
template <bool BF16>
constexpr uint32_t kAttInf = BF16 ? 0x7f80u : 0x7c00u;

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
  int q_vec;  // 16-byte loads of the queries are aligned
  int seqs, heads, kv_heads, group, page_shift;
  float scale_log2;  // softmax scale times log2(e)
  int causal, window;
  int whole;   // units are not shared between blocks
  void* out;   // [tokens][heads][dim]
  float* lse;  // [tokens][heads] or null
  float* partial;
  uint32_t* flags;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
__device__ __forceinline__ void att_clear_rest(const AttParams& P, int dim, int64_t block, int64_t blocks) {
  const int64_t first = max(static_cast<int64_t>(0), min(static_cast<int64_t>(P.start[0]), P.tokens));
  const int64_t last = max(first, min(static_cast<int64_t>(P.start[P.seqs]), P.tokens));
  const int64_t width = static_cast<int64_t>(P.heads) * dim, rest = P.tokens - (last - first);
  const int64_t step = blocks * blockDim.x;
  for (int64_t i = block * blockDim.x + threadIdx.x; i < rest * width; i += step) {
    const int64_t r = i / width, token = r < first ? r : last + r - first;
    att_store<BF16>(P.out, token * width + i % width, 0.0f);
    if (P.lse && i % width < P.heads) P.lse[token * P.heads + i % width] = -INFINITY;
  }
}

// The range of the values' scales over keys, by blocks of 32 channels: a byte for
// each of the D / 32 blocks.
template <int D>
struct AttRange {
  uint32_t top = 0, low = 0xffffffffu;  // the largest, and the smallest but zero, less one
  // This warp's part of the keys in [from, to): 32 of every 32 `warps`, from the `warp`-th 32 on.
  __device__ __forceinline__ void look(const AttParams& P, int b, int head, int from, int to, int warp, int warps) {
    const int32_t* table = P.table + static_cast<int64_t>(b) * P.table_ld;
#pragma unroll 4
    for (int key = from + 32 * warp + static_cast<int>(threadIdx.x & 31); key < to; key += 32 * warps) {
      const int32_t page = table[key >> P.page_shift];
      if (static_cast<uint32_t>(page) >= static_cast<uint64_t>(P.pages)) continue;
      const int64_t row = (((static_cast<int64_t>(page) * 2 + 1) * P.kv_heads + head) << P.page_shift) + (key & ((1 << P.page_shift) - 1));
      const uint32_t word = D == 128 ? reinterpret_cast<const uint32_t*>(P.scales)[row] : reinterpret_cast<const uint16_t*>(P.scales)[row];
      add(word, __vsub4(word, 0x01010101u));
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) add(__shfl_xor_sync(0xffffffffu, top, s), __shfl_xor_sync(0xffffffffu, low, s));
  }
  __device__ __forceinline__ void add(uint32_t more_top, uint32_t more_low) {
    top = __vmaxu4(top, more_top);
    low = __vminu4(low, more_low);
  }
  __device__ __forceinline__ bool wide() const {
    int all_top = 0, all_low = 256;
    bool wide = false;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      const int t = (top >> (8 * k)) & 255, least = static_cast<int>(((low >> (8 * k)) + 1u) & 255u);  // both 0: none
      wide |= t - least > kAttSpan;
      all_top = max(all_top, t);
      if (least > 0) all_low = min(all_low, least);
    }
    return wide || all_top - all_low > kAttExact;
  }
};

// One row in fp32 throughout, for rows whose values differ widely in size: every
// key in [from, to) counts (pages outside the pool do not).  `q`: the row's D
// elements; `o`: the lane's D / 32 channels of the result, from lane D / 32 on;
// returns the log2 of the sum of exponentials.  The whole warp calls.  A lane
// takes a key of 32 for the scores, then all take the keys' values in turn.
// Values, and the result, are 2^-22 of themselves: sums of 2^22 of the largest,
// 6 x 2^127, do not overflow.
constexpr float kAttWideUnit = 4194304.0f;
template <bool BF16, int D>
__device__ __forceinline__ float att_row_wide(const AttParams& P, int b, int head, const uint16_t* q, int from, int to, float (&o)[D / 32]) {
  constexpr int VPL = D / 32, BLOCKS = D / 32;
  const int lane = threadIdx.x & 31;
  const int32_t* table = P.table + static_cast<int64_t>(b) * P.table_ld;
  const int64_t values = static_cast<int64_t>(P.kv_heads) << P.page_shift;  // rows from a key to its value
  float m = -INFINITY, l = 0.0f;
  bool odd = false;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    o[c] = 0.0f;
    odd |= (q[lane * VPL + c] & 0x7fffu) >= kAttInf<BF16>;
  }
  odd = __any_sync(0xffffffffu, odd);  // the row is NaN if it sees a key
  for (int k0 = from; k0 < to; k0 += 32) {
    const int key = k0 + lane;
    int64_t row = -1;
    if (key < to) {
      const int32_t page = table[key >> P.page_shift];
      if (static_cast<uint32_t>(page) < static_cast<uint64_t>(P.pages))
        row = ((static_cast<int64_t>(page) * 2 * P.kv_heads + head) << P.page_shift) + (key & ((1 << P.page_shift) - 1));
    }
    float x = -INFINITY;
    if (row >= 0) {
      x = 0.0f;
#pragma unroll 1
      for (int k = 0; k < BLOCKS; ++k) {
        const uint4 codes = reinterpret_cast<const uint4*>(P.codes + row * (D / 2))[k];
        const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
        float acc = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint4 qw = load_x8(q + 32 * k + 8 * w, true, P.q_vec);
          const uint32_t qs[4] = {qw.x, qw.y, qw.z, qw.w};
          uint32_t h[4];
          e2m1x8_to_f16x2(words[w], h);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            float2 e;
            if constexpr (BF16)
              e = make_float2(bits_f32(qs[i] << 16), bits_f32(qs[i] & 0xffff0000u));
            else
              e = __half22float2(*reinterpret_cast<const __half2*>(&qs[i]));
            acc = __fmaf_rn(e.x, c.x, acc);
            acc = __fmaf_rn(e.y, c.y, acc);
          }
        }
        x = __fmaf_rn(acc, exp2i(static_cast<int>(P.scales[row * BLOCKS + k]) - 127), x);
      }
      x = odd ? NAN : __fmul_rn(x, P.scale_log2);
    }
    float up = fmaxf(m, x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, s));
    const float f = m == up ? 1.0f : ex2(__fsub_rn(m, up));
    m = up;
    const float p = x == -INFINITY ? 0.0f : ex2(__fsub_rn(x, m));
    l = __fmaf_rn(l, f, p);
#pragma unroll
    for (int c = 0; c < VPL; ++c) o[c] = __fmul_rn(o[c], f);
    const int n = min(32, to - k0);
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const int64_t at = __shfl_sync(0xffffffffu, row, j);
      if (at < 0) continue;  // (the same for all lanes)
      // (A whole word: of a narrower load the compiler's conversion took other bytes.)
      const uint32_t word = reinterpret_cast<const uint32_t*>(P.codes + (at + values) * (D / 2))[lane * VPL / 8] >> (lane * VPL % 8 * 4);
      const float scale = exp2i(static_cast<int>(P.scales[(at + values) * BLOCKS + lane * VPL / 32]) - 149);
      uint32_t h[4];
      e2m1x8_to_f16x2(word, h);
#pragma unroll
      for (int c = 0; c < VPL; c += 2) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[c / 2]));
        o[c] = __fmaf_rn(pj, __fmul_rn(v.x, scale), o[c]);
        o[c + 1] = __fmaf_rn(pj, __fmul_rn(v.y, scale), o[c + 1]);
      }
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, s));
  const bool seen = !(l == 0.0f);  // NaN counts as seen
#pragma unroll
  for (int c = 0; c < VPL; ++c) o[c] = seen ? __fdiv_rn(o[c], l) : 0.0f;
  return seen ? __fadd_rn(m, log2f(l)) : -INFINITY;
}

// Prompts (attention_prompt.cu): whether the call takes that kernel, and its launch.
bool attention_prompt_fits(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t max_queries);
int launch_attention_prompt(const AttParams& P, int bf16, int dim, int64_t max_queries, cudaStream_t stream);

}  // namespace mxw
