// What the attention kernels over the MXFP4 cache share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "f16mma.cuh"

namespace mxw {

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

// Prompts (attention_prompt.cu): whether the call takes that kernel, and its launch.
bool attention_prompt_fits(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t max_queries);
int launch_attention_prompt(const AttParams& P, int bf16, int dim, int64_t max_queries, cudaStream_t stream);

}  // namespace mxw
