// bf16 and f16 rows as sums of E4M3 terms with E8M0 block scales: the operand
// that meets MXFP4 in a block-scaled product.  E4M3 carries 4 significant bits,
// so two terms hold bf16's 8 and three hold f16's 11:
//   s = 2^(floor(log2 amax) - 7) of the block of 32,  t0 = e4m3(x / s),
//   t1 = e4m3((x / s - t0) 2^5),  t2 = e4m3(((x / s - t0) 2^5 - t1) 2^5)
// with scales s, s 2^-5, s 2^-10.  x / s and the remainders are held in f16: below
// 2^8 their last place is at least as fine as the last term's (2^-14, 2^-19),
// and f16's own steps (2^-24) only touch inputs under 2^-24 (bf16) or 2^-20
// (f16) of the block's largest.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "blockscale.cuh"
#include "common.cuh"
#include "f16mma.cuh"

namespace mxw {

constexpr int kLinM = 128;        // outputs per tile
constexpr int kLinK = 128;        // inputs per stage
constexpr int kLinSpread = 128;   // threads that spread a stage of W
constexpr int kLinGroups = 2;     // groups of them, which take every other stage
constexpr int kLinSpreadWarps = kLinGroups * kLinSpread / 32;  // the epilogue's warps too
constexpr int kLinThreads = 64 + 32 * kLinSpreadWarps;  // copies, products, spreading (and four warps that make terms)
constexpr int kLinRawBytes = kLinM * kLinK / 2;    // packed codes of a stage
constexpr int kLinWBytes = kLinM * kLinK;          // spread: 16 bytes per 16 codes
constexpr int kLinSfBytes = 512;                   // scales of 128 rows x 4 blocks

template <int NT, int TERMS>
struct LinearTile {
  static constexpr bool kFused = NT == 16;  // terms made in the product's kernel
  // Small tiles take the terms as rows of one operand (and add up their columns
  // at the end): a half or a third of the products' instructions, which are issued
  // one after the other.
  static constexpr bool kMerged = NT < 128;
  static constexpr int kTermBytes = NT * kLinK;
  static constexpr int kN = kMerged ? TERMS * NT : NT;               // columns of the accumulator
  static constexpr int kOperands = kMerged ? 1 : TERMS;
  static constexpr int kSfTiles = (kMerged ? (TERMS * NT + 127) / 128 : TERMS * ((NT + 127) / 128));
  static constexpr int kXBytes = TERMS * kTermBytes + kSfTiles * kLinSfBytes;  // one chunk of x: terms, then their scales
  // Where the scale of term t of row r lies: 128 operand rows to 512 bytes, [row % 32][row / 32][block].
  __host__ __device__ static constexpr int sf_place(int t, int r) {
    const int n = kMerged ? t * NT + r : r;
    return (kMerged ? 0 : t * kLinSfBytes) + (n >> 7) * kLinSfBytes + (n & 31) * 16 + ((n >> 5) & 3) * 4;
  }
  // A stage of copies: [x terms][x scales][packed W]; a spread buffer: [W][W
  // scales]; and where the terms are made, a ring of those.
  static constexpr int kStage = (kFused ? 0 : kXBytes) + kLinRawBytes;
  static constexpr int kStageStride = (kStage + 1023) / 1024 * 1024;
  static constexpr int kSpreadStride = (kLinWBytes + kLinSfBytes + 1023) / 1024 * 1024;
  static constexpr int kXStages = kFused ? 4 : 0;
  static constexpr int kXStride = (kXBytes + 1023) / 1024 * 1024;
  static constexpr int kThreads = kLinThreads + 32 * kXStages;
  static constexpr int kBuffers = kLinGroups;  // one spread buffer per group
  static constexpr int kBudget = NT <= 32 ? 111 * 1024 : 222 * 1024;  // two CTAs per SM for small tiles
  static constexpr int kFit = (kBudget - kBuffers * kSpreadStride - kXStages * kXStride) / kStageStride;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static_assert(kStages >= 2, "a stage must fit twice");
  static constexpr int kSmem = kBuffers * kSpreadStride + kXStages * kXStride + kStages * kStageStride + 1024 + 256;
  // TMEM: the accumulator, then the scales of two chunks.
  static constexpr uint32_t kSfCols = 4 * (1 + kSfTiles);
  static constexpr uint32_t kCols = kN + 2 * kSfCols;
  static constexpr uint32_t kTmemCols = kCols <= 32 ? 32 : kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
};

__device__ __forceinline__ uint32_t f16x2_to_e4m3x2(uint32_t v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(v)));
  return h;
}

// Eight inputs of a row; zeros outside x.
__device__ __forceinline__ uint4 load_x8(const uint16_t* src, bool in, bool vec) {
  if (!in) return make_uint4(0, 0, 0, 0);
  if (vec) return *reinterpret_cast<const uint4*>(src);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = src[2 * i] | (static_cast<uint32_t>(src[2 * i + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The terms of eight inputs: part `part` (of PARTS) of row `r` of a tile whose
// image starts at `terms` and whose scales start at `sf`.  Four neighbouring
// lanes share a block; all lanes of the warp take part in the shuffles.
template <bool BF16, int NT, int PARTS = 16>
__device__ __forceinline__ void split_x8(const uint4& raw, int r, int part, uint8_t* terms, uint8_t* sf, bool store) {
  constexpr int TERMS = BF16 ? 2 : 3;
  using Tile = LinearTile<NT, TERMS>;
  uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t pair = 0;  // magnitudes as bits: ordered, NaN above infinity
#pragma unroll
  for (int i = 0; i < 4; ++i) pair = __vmaxu2(pair, v[i] & 0x7fff7fffu);
  pair = __vmaxu2(pair, __shfl_xor_sync(0xffffffffu, pair, 1));
  pair = __vmaxu2(pair, __shfl_xor_sync(0xffffffffu, pair, 2));
  const uint32_t amax = max(pair & 0xffffu, pair >> 16);
  // byte = 127 + floor(log2 amax) - 7, at least 0; 255 (NaN) for a non-finite block.
  const int ebits = static_cast<int>(BF16 ? amax >> 7 : f32_bits(__half2float(__ushort_as_half(static_cast<unsigned short>(amax)))) >> 23);
  int byte = max(ebits - 7, 0);
  if (ebits == 255) byte = 255;
  // x / s in f16.
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const uint32_t mult = static_cast<uint32_t>(254 - byte) << 7;  // 2^(127 - byte)
      const __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&v[i]);
      const __nv_bfloat16 f = __ushort_as_bfloat16(static_cast<unsigned short>(mult));
      const __nv_bfloat162 scaled = __hmul2(m, __halves2bfloat162(f, f));
      const uint32_t w = *reinterpret_cast<const uint32_t*>(&scaled);
      v[i] = pack_f16x2(bits_f32(w << 16), bits_f32(w & 0xffff0000u));
    } else {
      const float mult = exp2i(127 - min(byte, 254));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      v[i] = pack_f16x2(__fmul_rn(f.x, mult), __fmul_rn(f.y, mult));
    }
    if (ebits == 255) v[i] = 0;
  }
  // The row's scales, one per block of its 8 PARTS inputs, as a word.
  uint32_t word = static_cast<uint32_t>(byte) << (8 * (part >> 2));
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  if constexpr (PARTS == 16) word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if (!store) return;
  // 16-byte slot part / 2 of the row's 128 bytes, swizzled over eight rows.
  terms += r * 128 + (((part >> 1) ^ (r & 7)) << 4) + ((part & 1) << 3);
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f16x2_to_e4m3x2(v[i]);
    *reinterpret_cast<uint2*>(terms + t * Tile::kTermBytes) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    if (part == 0) *reinterpret_cast<uint32_t*>(sf + Tile::sf_place(t, r)) = word;
    if (t + 1 < TERMS) {
      const int step = byte == 255 ? 0 : min(byte, 5);  // scales do not go below 2^-127
      const __half2 up = __float2half2_rn(static_cast<float>(1 << step));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t q = e4m3x2_to_f16x2(w[i]);
        const __half2 rest = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&v[i]), *reinterpret_cast<const __half2*>(&q)), up);
        v[i] = *reinterpret_cast<const uint32_t*>(&rest);
      }
      byte -= step;
      const uint32_t nan = __vcmpeq4(word, 0xffffffffu);
      word = (__vsubus4(word, 0x05050505u) & ~nan) | (word & nan);
    }
  }
}

}  // namespace mxw
