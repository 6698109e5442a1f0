// K8: matrix product with MXFP4 weights, y = act(x W^T + bias) + residual.
//
// W [N, K] is what the quantizer wrote: E2M1 codes and one E8M0 exponent per
// 32 inputs.  That is an operand format of the tensor cores (kind::mxf8f6f4),
// so the codes go to them as they are and nothing is dequantized.  The other
// operand has to be 8 bits wide, so x is split exactly into a sum of E4M3
// terms with E8M0 block scales (E4M3 carries 4 significant bits: two terms for
// bf16's 8, three for f16's 11):
//   s = 2^(floor(log2 amax) - 7) of the block of 32,  t0 = e4m3(x / s),
//   t1 = e4m3((x / s - t0) 2^5),  t2 = e4m3(((x / s - t0) 2^5 - t1) 2^5)
// with scales s, s 2^-5, s 2^-10.  The remainders are exact (terms.cuh).  An
// element at least 2^-13 of its block's largest is represented exactly; a
// smaller one to within 2^-22 of the block's largest (E4M3's subnormals).
// Products and sums are fp32 in TMEM.  A block that holds a NaN or an infinity
// gets the NaN scale: every output of that row of x is NaN.
//
// CTA tile: 128 outputs (M, W's rows) x NT rows of x (N), 128 inputs a stage.
// One thread copies W's packed bytes (TMA) and the terms of x (bulk copies of
// what linear_terms_kernel laid out) into a ring; four warps spread the codes
// into the 16-byte slots that E2M1 operands take in shared memory (8 bytes of
// codes, 8 of padding) and put the scales into the tensor cores' layout; one
// warp issues the products.  Up to four rows of x four more warps make the
// terms in the same launch.  When there are too few tiles for
// the SMs the CTAs of a cluster split K and add their fp32 partial tiles over
// distributed shared memory in rank order, so results do not change from run
// to run.
//
// Measured: one row, 5120 x 5120: 10 us (1.4 TB/s); 24 rows, 17408 x 5120: 21 us
// (2.3 TB/s); both bound by shared memory, through which W passes three times
// (copied, spread to twice its size, read by the products), and by 6 us of launch,
// set-up, cluster sum and epilogue.  8192 rows, 5120 x 17408: 1.19 ms, 1.23
// PFLOP/s of the product (twice that of the terms').
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cooperative_groups.h>

#include "blockscale.cuh"
#include "common.cuh"
#include "runtime.h"
#include "terms.cuh"

namespace cg = cooperative_groups;

namespace mxw {

struct LinearParams {
  const uint8_t* scales;
  const void* x;
  int64_t ldx;
  int x_vec;  // 16-byte loads of x are aligned
  const uint8_t* terms;  // [token tiles][chunks][kXBytes]
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* y;
  int64_t rows, outs, inner;
  int chunks;
  int act;
  int words;  // the scales of a row start on a 4-byte boundary
  int pairs;  // rows of y and of the residual start on 4-byte boundaries
  uint32_t* flags;
};

// ------------------------------------------------------------- terms of x

struct TermsParams {
  const void* x;
  int64_t ldx, rows, inner;
  int chunks;
  int x_vec;
  uint8_t* terms;  // [token tiles][chunks][kXBytes]
};

// Sixteen threads take the 128 inputs of one (row, chunk), eight each; for a
// prompt, four rows of them with their loads in flight together.  Reads 2 bytes
// an input and writes 2 (bf16) or 3; bound by the conversions and the integer
// work around them (84% of that pipe): 38 us at 8192 x 5120 bf16 under the
// profiler, where HBM would take 26.
constexpr int terms_rows(int nt) { return nt == 128 ? 4 : 1; }

template <bool BF16, int NT>
__global__ void __launch_bounds__(256) linear_terms_kernel(const TermsParams P) {
  constexpr int TERMS = BF16 ? 2 : 3, AHEAD = terms_rows(NT);
  using Tile = LinearTile<NT, TERMS>;
  grid_dependents_launch();
  const uint32_t unit = blockIdx.x * 16u + (threadIdx.x >> 4);
  const int part = threadIdx.x & 15;
  const int64_t padded = (P.rows + NT - 1) / NT * NT;
  const bool in_grid = unit < static_cast<uint32_t>(padded / AHEAD) * static_cast<uint32_t>(P.chunks);
  const uint32_t group = unit / static_cast<uint32_t>(P.chunks);
  const int64_t row = in_grid ? static_cast<int64_t>(group) * AHEAD : 0;
  const int chunk = in_grid ? static_cast<int>(unit - group * static_cast<uint32_t>(P.chunks)) : 0;
  const int64_t k0 = static_cast<int64_t>(chunk) * kLinK + part * 8;
  // inner % 32 == 0: eight inputs are in or out together
  uint4 v[AHEAD];
#pragma unroll
  for (int r = 0; r < AHEAD; ++r)
    v[r] = load_x8(static_cast<const uint16_t*>(P.x) + (row + r) * P.ldx + k0, in_grid && row + r < P.rows && k0 < P.inner, P.x_vec);
  uint8_t* base = P.terms + ((row / NT) * P.chunks + chunk) * static_cast<int64_t>(Tile::kXBytes);
#pragma unroll
  for (int r = 0; r < AHEAD; ++r)
    split_x8<BF16, NT>(v[r], static_cast<int>(row % NT) + r, part, base, base + TERMS * Tile::kTermBytes, in_grid);
}

// ---------------------------------------------------------------- epilogue

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case MXW_ACT_RELU:
      return v > 0.0f ? v : (v != v ? v : 0.0f);
    case MXW_ACT_SILU:
      // __expf is off by 2 + 1.2 |v| steps of fp32 at most, under 2^-16 of the result: far below the output's 2^-8 or 2^-11.
      return v / (1.0f + __expf(-v));
    case MXW_ACT_GELU:
      return 0.5f * v * erfcf(-0.70710678118654752f * v);
    default:
      return v;
  }
}

template <bool BF16>
__device__ __forceinline__ float load16(const void* p, int64_t i) {
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  return BF16 ? bits_f32(static_cast<uint32_t>(b) << 16) : __half2float(*reinterpret_cast<const __half*>(&b));
}
template <bool BF16>
__device__ __forceinline__ void store16(void* p, int64_t i, float v) {
  if constexpr (BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Sixteen columns of the accumulator, the terms' columns added up; NaN for a `bad` one.
template <int NT, int TERMS>
__device__ __forceinline__ void load_sums(uint32_t taddr, bool bad, float (&v)[16]) {
  tmem_ld_32x32b_x16(taddr, v);
  if constexpr (LinearTile<NT, TERMS>::kMerged) {
#pragma unroll
    for (int t = 1; t < TERMS; ++t) {
      float w[16];
      tmem_ld_32x32b_x16(taddr + t * NT, w);
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = __fadd_rn(v[u], w[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < 16; ++u) v[u] = bad ? NAN : v[u];
}

// Two neighbours from a word.
template <bool BF16>
__device__ __forceinline__ float2 pair_values(uint32_t w) {
  if constexpr (BF16) return make_float2(bits_f32(w << 16), bits_f32(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// Brings 128 bytes of a row of the residual towards the epilogue that reads them when the products are done.
__device__ __forceinline__ void prefetch_residual(const LinearParams& P, int64_t row, int64_t n) {
  if (row >= P.rows || n >= P.outs) return;
  const uint16_t* at = static_cast<const uint16_t*>(P.residual) + row * P.ldr + n;
  prefetch_l2(at);
  prefetch_l2(at + min(static_cast<int64_t>(63), P.outs - 1 - n));
}
template <bool BF16>
__device__ __forceinline__ void store16x2(void* p, int64_t i, float a, float b) {
  if constexpr (BF16)
    *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p) + i) = __floats2bfloat162_rn(a, b);
  else
    *reinterpret_cast<__half2*>(static_cast<__half*>(p) + i) = __floats2half2_rn(a, b);
}

// ----------------------------------------------------------------- product

template <bool BF16, int NT>
__global__ void __launch_bounds__((LinearTile<NT, BF16 ? 2 : 3>::kThreads))
    linear_kernel(const __grid_constant__ CUtensorMap map, const LinearParams P) {
  constexpr int TERMS = BF16 ? 2 : 3;
  using Tile = LinearTile<NT, TERMS>;
  constexpr int ST = Tile::kStages, WB = Tile::kBuffers;
  constexpr bool FUSED = Tile::kFused;
  constexpr int kXPart = FUSED ? 0 : Tile::kXBytes;  // x's part of a stage of copies
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  constexpr int XS = FUSED ? Tile::kXStages : 1;
  uint8_t* xring = smem + WB * Tile::kSpreadStride;
  uint8_t* ring = xring + Tile::kXStages * Tile::kXStride;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(ring + ST * Tile::kStageStride);
  uint64_t* raw_empty = raw_full + ST;
  uint64_t* w_full = raw_empty + ST;
  uint64_t* w_empty = w_full + WB;
  uint64_t* x_full = w_empty + WB;
  uint64_t* x_empty = x_full + XS;
  uint64_t* done = x_empty + XS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* fail = reinterpret_cast<int*>(tmem_slot + 1);

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = static_cast<int64_t>(blockIdx.y) * kLinM;
  const int64_t tile = blockIdx.z;
  const int c_begin = static_cast<int>(static_cast<int64_t>(P.chunks) * rank / ranks);
  const int n_chunks = static_cast<int>(static_cast<int64_t>(P.chunks) * (rank + 1) / ranks) - c_begin;

  // The copying thread makes the barriers and sends off the first stages of W
  // before the others are ready to take them.
  auto copy_w = [&](int i) {
    const int s = i % ST;
    mbar_arrive_expect_tx(&raw_full[s], kXPart + kLinRawBytes);
    tma_load_2d(ring + s * Tile::kStageStride + kXPart, &map, &raw_full[s], (c_begin + i) * (kLinK / 2), static_cast<int32_t>(n0));
  };
  const int ahead = n_chunks < ST ? n_chunks : ST;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], FUSED ? 4 : 1);  // freed by the spreading warps, or by the products that read x there
    }
    for (int b = 0; b < WB; ++b) {
      mbar_init(&w_full[b], 4);
      mbar_init(&w_empty[b], 1);
    }
    for (int x = 0; x < XS; ++x) {
      mbar_init(&x_full[x], 1);
      mbar_init(&x_empty[x], 1);
    }
    mbar_init(done, 1);
    *fail = 0;
    fence_mbar_init();
    for (int i = 0; i < ahead; ++i) copy_w(i);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Tile::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // --------------------------------------------------------------- copies
    if (lane == 0) {
      bool ok = true;
      const uint8_t* xsrc = P.terms + (tile * P.chunks + c_begin) * static_cast<int64_t>(Tile::kXBytes);
      auto copy_x = [&](int i) {
        const int s = i % ST;
        bulk_load(ring + s * Tile::kStageStride, xsrc + static_cast<int64_t>(i) * Tile::kXBytes, Tile::kXBytes, &raw_full[s]);
      };
      if constexpr (!FUSED) {
        grid_dependency_wait();  // W does not depend on the launch that makes the terms: its first stages went ahead
        for (int i = 0; i < ahead; ++i) copy_x(i);
      }
      int i = ahead;
      for (; i < n_chunks; ++i) {
        if (!mbar_wait_cycles(&raw_empty[i % ST], static_cast<uint32_t>((i / ST - 1) & 1))) {
          ok = false;
          break;
        }
        copy_w(i);
        if constexpr (!FUSED) copy_x(i);
      }
      // Copies in flight have to land before the CTA may end.
      for (int j = i > ST ? i - ST : 0; j < i; ++j)
        if (!mbar_wait_cycles(&raw_full[j % ST], static_cast<uint32_t>((j / ST) & 1))) ok = false;
      if (!ok) atomicOr(fail, 1);
    }
  } else if (warp >= 2 && warp < 2 + kLinSpreadWarps) {
    // ------------------------------------------------------------ spreading
    const int group = (warp - 2) / (kLinSpread / 32);
    const int e = (threadIdx.x - 64) % kLinSpread;  // and the row of W whose scales this thread brings
    const int64_t nb = P.inner / 32;
    const bool row_in = n0 + e < P.outs;
    const uint8_t* srow = P.scales + (row_in ? (n0 + e) * nb : 0) + static_cast<int64_t>(c_begin) * 4;
    if (P.residual)
      for (int i = threadIdx.x - 64; i < 2 * NT; i += 32 * kLinSpreadWarps)
        if ((i >> 1) % ranks == rank) prefetch_residual(P, tile * NT + (i >> 1), n0 + 64 * (i & 1));
    // Scales of four of the group's chunks at a time, loaded that far ahead.
    uint32_t sf[4], sf_next[4];
    auto load_scales = [&](int i, uint32_t (&w)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = i + kLinGroups * q;
        w[q] = 0;
        if (row_in && c < n_chunks) {
          if (P.words) {
            w[q] = *reinterpret_cast<const uint32_t*>(srow + 4 * c);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (static_cast<int64_t>(c_begin + c) * 4 + k < nb) w[q] |= static_cast<uint32_t>(srow[4 * c + k]) << (8 * k);
          }
        }
      }
    };
    load_scales(group, sf_next);
    bool ok = true;
    uint8_t* w = smem + group * Tile::kSpreadStride;
    for (int i = group, turn = 0; i < n_chunks; i += kLinGroups, ++turn) {
      const int s = i % ST;
      if ((turn & 3) == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sf[q] = sf_next[q];
        load_scales(i + 4 * kLinGroups, sf_next);
      }
      if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait_cycles(&w_empty[group], static_cast<uint32_t>((turn - 1) & 1)))) ok = false;
      if (ok) {
        const uint32_t word = (turn & 2) ? ((turn & 1) ? sf[3] : sf[2]) : ((turn & 1) ? sf[1] : sf[0]);
        *reinterpret_cast<uint32_t*>(w + kLinWBytes + (e & 31) * 16 + (e >> 5) * 4) = word;
        if (!__all_sync(0xffffffffu, mbar_wait_cycles(&raw_full[s], static_cast<uint32_t>((i / ST) & 1)))) ok = false;
      }
      if (!ok) break;
      const uint8_t* raw = ring + s * Tile::kStageStride + kXPart;
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = reinterpret_cast<const uint4*>(raw)[e + j * kLinSpread];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // 32 codes of row r: slots 2p and 2p + 1 of its 128 bytes, swizzled over eight rows.
        const int u = e + j * kLinSpread, r = u >> 2, p = u & 3;
        uint8_t* row = w + r * 128;
        *reinterpret_cast<uint2*>(row + (((2 * p) ^ (r & 7)) << 4)) = make_uint2(v[j].x, v[j].y);
        *reinterpret_cast<uint2*>(row + (((2 * p + 1) ^ (r & 7)) << 4)) = make_uint2(v[j].z, v[j].w);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&w_full[group]);
        // Only here, with the loaded words used: a stage given back with its
        // loads still under way was refilled under them.
        if constexpr (FUSED) mbar_arrive(&raw_empty[s]);
      }
    }
    if (!ok) atomicOr(fail, 1);
  } else if (warp == 1) {
    // ------------------------------------------------------------- products
    constexpr uint32_t idesc = make_idesc_e2m1_e4m3(kLinM, Tile::kN);
    const bool leader = elect_one();
    bool ok = true;
    for (int i = 0; i < n_chunks; ++i) {
      const int s = i % ST, b = i % WB, xs = i % XS;
      // (The spreading warps have seen the copies' barrier: theirs covers x too.)
      ok = mbar_wait_cycles(&w_full[b], static_cast<uint32_t>((i / WB) & 1)) &&
           (!FUSED || mbar_wait_cycles(&x_full[xs], static_cast<uint32_t>((i / XS) & 1)));
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sw = smem_u32(smem) + b * Tile::kSpreadStride;
      const uint32_t sx = FUSED ? smem_u32(xring) + xs * Tile::kXStride : smem_u32(ring) + s * Tile::kStageStride;
      const uint32_t sfa = tmem + Tile::kN + (i & 1) * Tile::kSfCols;
      const uint32_t sfb = sfa + 4;
      const uint32_t a_lo = desc_k_sw128_lo(sw), b_lo = desc_k_sw128_lo(sx);
      if (leader) {
        tmem_cp_scales(sfa, sw + kLinWBytes);
#pragma unroll
        for (int t = 0; t < Tile::kSfTiles; ++t) tmem_cp_scales(sfb + 4 * t, sx + TERMS * Tile::kTermBytes + t * kLinSfBytes);
#pragma unroll
        for (int t = 0; t < Tile::kOperands; ++t)
#pragma unroll
          for (int kk = 0; kk < kLinK / 32; ++kk)  // 32 inputs are 32 bytes of a swizzled 128-byte row
            mma_mxf8f6f4(tmem, desc_of(kDescKSw128Hi, a_lo + 2 * kk), desc_of(kDescKSw128Hi, b_lo + t * (Tile::kTermBytes >> 4) + 2 * kk),
                         mx_idesc_scale_byte(idesc, kk), sfa, sfb + 4 * t, (i > 0 || t > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&w_empty[b]);
        mma_commit(FUSED ? &x_empty[xs] : &raw_empty[s]);
      }
      __syncwarp();
    }
    if (leader) {
      if (!ok) atomicOr(fail, 1);
      mma_commit(done);
    }
  } else if constexpr (FUSED) {
    // --------------------------------------------------------- terms of x
    // A warp takes a chunk whole, every fourth chunk: two rows at a time, 16 lanes each.
    const int part = lane & 15, sub = lane >> 4;
    const int n_rows = static_cast<int>(min(static_cast<int64_t>(NT), P.rows - tile * NT));
    const uint16_t* x = static_cast<const uint16_t*>(P.x) + tile * NT * P.ldx + part * 8;
    const int in_left = static_cast<int>(min(P.inner - static_cast<int64_t>(c_begin) * kLinK, static_cast<int64_t>(n_chunks) * kLinK)) - part * 8;
    bool ok = true;
    for (int i = warp - 2 - kLinSpreadWarps; i < n_chunks; i += XS) {
      const int xs = i % XS;
      uint8_t* xt = xring + xs * Tile::kXStride;
      const uint16_t* src = x + (static_cast<int64_t>(c_begin) + i) * kLinK;
      const bool in = i * kLinK < in_left;  // inner % 32 == 0: eight inputs are in or out together
      uint4 v = load_x8(src + sub * P.ldx, in && sub < n_rows, P.x_vec);
      if (i >= XS && !__all_sync(0xffffffffu, mbar_wait_cycles(&x_empty[xs], static_cast<uint32_t>((i / XS - 1) & 1)))) {
        ok = false;
        break;
      }
      for (int r = 0; r < n_rows; r += 2) {
        const uint4 now = v;
        v = load_x8(src + (r + 2 + sub) * P.ldx, in && r + 2 + sub < n_rows, P.x_vec);
        split_x8<BF16, NT>(now, r + sub, part, xt, xt + TERMS * Tile::kTermBytes, true);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&x_full[xs]);
    }
    if (!ok) atomicOr(fail, 1);
  }

  // ---------------------------------------------------------------- epilogue
  __syncwarp();
  const bool epilogue = warp >= 2 && warp < 2 + kLinSpreadWarps;
  const int half = (warp - 2) >> 2;  // and every other group of columns
  const int quarter = warp & 3, tid = 32 * quarter + lane;  // a warp reads its own quarter of the TMEM lanes
  bool bad = false;  // a wait gave up: NaN, whether or not anybody reads the flags
  if (epilogue) {
    bad = !__all_sync(0xffffffffu, mbar_wait_cycles(done, 0));
    if (bad) atomicOr(fail, 1);
    bad |= *static_cast<volatile int*>(fail) != 0;
  }
  tc_fence_after();
  const int64_t n = n0 + tid;  // this thread's output
  const int64_t t0 = tile * NT;
  float bias = 0.0f;
  if (epilogue && P.bias && n < P.outs) bias = load16<BF16>(P.bias, n);
  if (ranks == 1) {
    if (epilogue) {
#pragma unroll 1
      for (int c = 16 * half; c < NT; c += 32) {
        if (t0 + c >= P.rows) break;
        float v[16];
        load_sums<NT, TERMS>(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + c, bad, v);
        if (n < P.outs) {
          float res[16];
#pragma unroll
          for (int u = 0; u < 16; ++u)
            res[u] = P.residual && t0 + c + u < P.rows ? load16<BF16>(P.residual, (t0 + c + u) * P.ldr + n) : 0.0f;
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const int64_t t = t0 + c + u;
            if (t < P.rows) {
              float o = activate(__fadd_rn(v[u], bias), P.act);
              if (P.residual) o = __fadd_rn(o, res[u]);
              store16<BF16>(P.y, t * P.outs + n, o);
            }
          }
        }
      }
    }
  } else {
    float* part = reinterpret_cast<float*>(smem);  // [NT][128], in the drained stages
    if (epilogue) {
#pragma unroll 1
      for (int c = 16 * half; c < NT && t0 + c < P.rows; c += 32) {
        float v[16];
        load_sums<NT, TERMS>(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + c, bad, v);
#pragma unroll
        for (int u = 0; u < 16; ++u) part[(c + u) * 128 + tid] = v[u];
      }
    }
    cluster_sync_all();
    if (epilogue && n < P.outs) {
      // Columns rank, rank + ranks, ..., every other one: two at a time, all
      // ranks' parts in flight, added in rank order.
      for (int c = rank + half * ranks; c < NT && t0 + c < P.rows; c += 4 * ranks) {
        float v[2][8], res[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = c + 2 * h * ranks;
          const bool in = col < NT && t0 + col < P.rows;
#pragma unroll
          for (int k = 0; k < 8; ++k) v[h][k] = in && k < ranks ? cluster.map_shared_rank(part, k)[col * 128 + tid] : 0.0f;
          res[h] = in && P.residual ? load16<BF16>(P.residual, (t0 + col) * P.ldr + n) : 0.0f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t t = t0 + c + 2 * h * ranks;
          if (c + 2 * h * ranks >= NT || t >= P.rows) break;
          float sum = v[h][0];
#pragma unroll
          for (int k = 1; k < 8; ++k)
            if (k < ranks) sum = __fadd_rn(sum, v[h][k]);
          float o = activate(__fadd_rn(sum, bias), P.act);
          if (P.residual) o = __fadd_rn(o, res[h]);
          store16<BF16>(P.y, t * P.outs + n, o);
        }
      }
    }
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Tile::kTmemCols);
  }
  if (threadIdx.x == 0 && *fail && P.flags) atomicOr(P.flags, MXW_FLAG_TIMEOUT);
}

// ---------------------------------------------------- product of many rows
//
// Tiles of 128 rows of x (M) x 256 outputs (N) for prompts: the terms of x are
// the A operand, W's codes the B operand.  A chunk of 128 inputs brings 33 KB
// of terms and 17 KB of W for 1024 cycles of products (the orientation above
// would bring 75 KB), so three stages of copies cover their latency.  What
// bounds it is shared memory: a chunk's products read 96 KB of it, copies write
// 50, and spreading reads 16 and writes 32, which is 1,500 cycles at 128 bytes a
// cycle (8192 x 5120 x 17408 takes some 1,800 a chunk).

constexpr int kWideN = 256;
constexpr int kWideSpread = 256;  // threads that spread a stage of W
constexpr int kWideGroups = 2;    // groups of them, which take every other stage
constexpr int kWideSpreadWarps = kWideGroups * kWideSpread / 32;  // the epilogue's warps too
constexpr int kWideThreads = 64 + 32 * kWideSpreadWarps;

template <int TERMS>
struct WideTile {
  using X = LinearTile<128, TERMS>;  // the terms' images are those of 128-row tiles
  static constexpr int kRawBytes = kWideN * kLinK / 2;
  static constexpr int kStageStride = (X::kXBytes + kRawBytes + 1023) / 1024 * 1024;  // [x terms][x scales][packed W]
  static constexpr int kSpreadStride = kWideN * kLinK + 2 * kLinSfBytes;              // [W][W scales]
  static constexpr int kBuffers = kWideGroups;
  static constexpr int kStages = (222 * 1024 - kBuffers * kSpreadStride) / kStageStride;
  static_assert(kStages >= 2, "a stage must fit twice");
  static constexpr int kSmem = kBuffers * kSpreadStride + kStages * kStageStride + 1024 + 256;
  static constexpr uint32_t kSfCols = 4 * TERMS + 8;
  static constexpr uint32_t kTmemCols = 512;  // 256 + 2 kSfCols, rounded up
};

template <bool BF16>
__global__ void __launch_bounds__(kWideThreads, 1)
    linear_wide_kernel(const __grid_constant__ CUtensorMap map, const LinearParams P) {
  constexpr int TERMS = BF16 ? 2 : 3;
  using Tile = WideTile<TERMS>;
  using X = typename Tile::X;
  constexpr int ST = Tile::kStages, WB = Tile::kBuffers;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  uint8_t* ring = smem + WB * Tile::kSpreadStride;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(ring + ST * Tile::kStageStride);
  uint64_t* raw_empty = raw_full + ST;
  uint64_t* w_full = raw_empty + ST;
  uint64_t* w_empty = w_full + WB;
  uint64_t* done = w_empty + WB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* fail = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kWideN;
  const int64_t tile = blockIdx.y;
  const int n_chunks = P.chunks;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 1);
    }
    for (int b = 0; b < WB; ++b) {
      mbar_init(&w_full[b], kWideSpread / 32);
      mbar_init(&w_empty[b], 1);
    }
    mbar_init(done, 1);
    *fail = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, Tile::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // --------------------------------------------------------------- copies
    if (lane == 0) {
      bool ok = true;
      const uint8_t* xsrc = P.terms + tile * P.chunks * static_cast<int64_t>(X::kXBytes);
      grid_dependency_wait();
      int i = 0;
      for (; i < n_chunks; ++i) {
        const int s = i % ST;
        if (i >= ST && !mbar_wait_cycles(&raw_empty[s], static_cast<uint32_t>((i / ST - 1) & 1))) {
          ok = false;
          break;
        }
        uint8_t* st = ring + s * Tile::kStageStride;
        mbar_arrive_expect_tx(&raw_full[s], X::kXBytes + Tile::kRawBytes);
        tma_load_2d(st + X::kXBytes, &map, &raw_full[s], i * (kLinK / 2), static_cast<int32_t>(n0));
        bulk_load(st, xsrc + static_cast<int64_t>(i) * X::kXBytes, X::kXBytes, &raw_full[s]);
      }
      // Copies in flight have to land before the CTA may end.
      for (int j = i > ST ? i - ST : 0; j < i; ++j)
        if (!mbar_wait_cycles(&raw_full[j % ST], static_cast<uint32_t>((j / ST) & 1))) ok = false;
      if (!ok) atomicOr(fail, 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- products
    constexpr uint32_t idesc = make_idesc_e4m3_e2m1(128, kWideN);
    const bool leader = elect_one();
    bool ok = true;
    for (int i = 0; i < n_chunks; ++i) {
      const int s = i % ST, b = i % WB;
      // (The spreading warps have seen the copies' barrier: theirs covers x too.)
      ok = mbar_wait_cycles(&w_full[b], static_cast<uint32_t>((i / WB) & 1));
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sw = smem_u32(smem) + b * Tile::kSpreadStride;
      const uint32_t sx = smem_u32(ring) + s * Tile::kStageStride;
      const uint32_t sfa = tmem + kWideN + (i & 1) * Tile::kSfCols;
      const uint32_t sfb = sfa + 4 * TERMS;
      const uint32_t a_lo = desc_k_sw128_lo(sx), b_lo = desc_k_sw128_lo(sw);
      if (leader) {
#pragma unroll
        for (int t = 0; t < TERMS; ++t) tmem_cp_scales(sfa + 4 * t, sx + TERMS * X::kTermBytes + t * kLinSfBytes);
#pragma unroll
        for (int h = 0; h < 2; ++h) tmem_cp_scales(sfb + 4 * h, sw + kWideN * kLinK + h * kLinSfBytes);
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
          for (int kk = 0; kk < kLinK / 32; ++kk)
            mma_mxf8f6f4(tmem, desc_of(kDescKSw128Hi, a_lo + t * (X::kTermBytes >> 4) + 2 * kk), desc_of(kDescKSw128Hi, b_lo + 2 * kk),
                         mx_idesc_scale_byte(idesc, kk), sfa + 4 * t, sfb, (i > 0 || t > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&w_empty[b]);
        mma_commit(&raw_empty[s]);
      }
      __syncwarp();
    }
    if (leader) {
      if (!ok) atomicOr(fail, 1);
      mma_commit(done);
    }
  } else {
    // ------------------------------------------------------------ spreading
    const int group = (warp - 2) / (kWideSpread / 32);
    const int e = (threadIdx.x - 64) % kWideSpread;  // and the row of W whose scales this thread brings
    const int64_t nb = P.inner / 32;
    const bool row_in = n0 + e < P.outs;
    const uint8_t* srow = P.scales + (row_in ? (n0 + e) * nb : 0);
    if (P.residual) prefetch_residual(P, tile * 128 + 32 * (warp & 3) + lane, n0 + 64 * ((warp - 2) >> 2));
    uint32_t sf[4], sf_next[4];
    auto load_scales = [&](int i, uint32_t (&w)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = i + kWideGroups * q;
        w[q] = 0;
        if (row_in && c < n_chunks) {
          if (P.words) {
            w[q] = *reinterpret_cast<const uint32_t*>(srow + 4 * c);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (static_cast<int64_t>(c) * 4 + k < nb) w[q] |= static_cast<uint32_t>(srow[4 * c + k]) << (8 * k);
          }
        }
      }
    };
    load_scales(group, sf_next);
    bool ok = true;
    uint8_t* w = smem + group * Tile::kSpreadStride;
    for (int i = group, turn = 0; i < n_chunks; i += kWideGroups, ++turn) {
      const int s = i % ST;
      if ((turn & 3) == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sf[q] = sf_next[q];
        load_scales(i + 4 * kWideGroups, sf_next);
      }
      if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait_cycles(&w_empty[group], static_cast<uint32_t>((turn - 1) & 1)))) ok = false;
      if (ok) {
        const uint32_t word = (turn & 2) ? ((turn & 1) ? sf[3] : sf[2]) : ((turn & 1) ? sf[1] : sf[0]);
        *reinterpret_cast<uint32_t*>(w + kWideN * kLinK + (e >> 7) * kLinSfBytes + (e & 31) * 16 + ((e >> 5) & 3) * 4) = word;
        if (!__all_sync(0xffffffffu, mbar_wait_cycles(&raw_full[s], static_cast<uint32_t>((i / ST) & 1)))) ok = false;
      }
      if (!ok) break;
      const uint8_t* raw = ring + s * Tile::kStageStride + X::kXBytes;
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = reinterpret_cast<const uint4*>(raw)[e + j * kWideSpread];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int u = e + j * kWideSpread, r = u >> 2, p = u & 3;
        uint8_t* row = w + r * 128;
        *reinterpret_cast<uint2*>(row + (((2 * p) ^ (r & 7)) << 4)) = make_uint2(v[j].x, v[j].y);
        *reinterpret_cast<uint2*>(row + (((2 * p + 1) ^ (r & 7)) << 4)) = make_uint2(v[j].z, v[j].w);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&w_full[group]);
    }
    if (!ok) atomicOr(fail, 1);
  }

  // ---------------------------------------------------------------- epilogue
  // A warp reads its quarter of the rows and 64 of the columns and turns them
  // over in shared memory so that a row's 64 outputs are read (residual) and
  // written together.  The residual's first 16 rows are read before the products
  // are waited for, the others before the first are written.
  __syncwarp();
  if (warp >= 2) {
    const int quarter = warp & 3, c = 64 * ((warp - 2) >> 2);
    const int64_t t0 = tile * 128 + 32 * quarter, n = n0 + c + 2 * lane;
    const int rows = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(32), P.rows - t0)));
    const bool pairs = P.pairs;  // two outputs per load and store
    const bool in0 = n < P.outs, in1 = n + 1 < P.outs;
    uint32_t res[2][16];
    auto load_residual = [&](int half, uint32_t (&w)[16]) {
      const int live = P.residual && in0 ? rows - 16 * half : 0;
      const uint16_t* at = static_cast<const uint16_t*>(P.residual) + (t0 + 16 * half) * P.ldr + n;
      if (pairs) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          w[r] = 0;
          if (r < live) w[r] = in1 ? *reinterpret_cast<const uint32_t*>(at + r * P.ldr) : at[r * P.ldr];
        }
      } else {
        uint16_t lo[16], hi[16];  // put together when all are on their way
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          lo[r] = hi[r] = 0;
          if (r < live) lo[r] = at[r * P.ldr];
          if (r < live && in1) hi[r] = at[r * P.ldr + 1];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = lo[r] | (static_cast<uint32_t>(hi[r]) << 16);
      }
    };
    load_residual(0, res[0]);
    bool bad = !__all_sync(0xffffffffu, mbar_wait_cycles(done, 0));
    if (bad) atomicOr(fail, 1);
    bad |= *static_cast<volatile int*>(fail) != 0;  // a wait gave up: NaN, whether or not anybody reads the flags
    tc_fence_after();
    float* turn = reinterpret_cast<float*>(smem) + (warp - 2) * (32 * 66);  // [32 rows][64 + 2]
    if (n0 + c < P.outs && rows > 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(32 * quarter) << 16) + c + 32 * h, v);
#pragma unroll
        for (int u = 0; u < 16; ++u) *reinterpret_cast<float2*>(turn + lane * 66 + 32 * h + 2 * u) = make_float2(bad ? NAN : v[2 * u], bad ? NAN : v[2 * u + 1]);
      }
      __syncwarp();
      load_residual(1, res[1]);
      const float bias0 = P.bias && in0 ? load16<BF16>(P.bias, n) : 0.0f;
      const float bias1 = P.bias && in1 ? load16<BF16>(P.bias, n + 1) : 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = 16 * half + r;
          if (row >= rows) break;
          const float2 v = *reinterpret_cast<const float2*>(turn + row * 66 + 2 * lane);
          float o0 = activate(__fadd_rn(v.x, bias0), P.act), o1 = activate(__fadd_rn(v.y, bias1), P.act);
          if (P.residual) {
            const float2 add = pair_values<BF16>(res[half][r]);
            o0 = __fadd_rn(o0, add.x);
            o1 = __fadd_rn(o1, add.y);
          }
          const int64_t at = (t0 + row) * P.outs + n;
          if (pairs && in1) {
            store16x2<BF16>(P.y, at, o0, o1);
          } else {
            if (in0) store16<BF16>(P.y, at, o0);
            if (in1) store16<BF16>(P.y, at + 1, o1);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Tile::kTmemCols);
  }
  if (threadIdx.x == 0 && *fail && P.flags) atomicOr(P.flags, MXW_FLAG_TIMEOUT);
}

// -------------------------------------------------------------------- host

// Rows of x per tile: the smallest tile that takes them all, so that W is read
// once.  Up to four rows the terms are made in the product's kernel (tiles of
// 16), which saves a launch; its four warps do not keep up with more rows
// (5120 x 5120 bf16 in clusters of four, one launch against two: 11.0 and 11.6
// us with one row, 11.6 and 11.8 with four, 13.9 and 12.0 with eight, 17.7 and
// 12.4 with sixteen).
static int linear_tile(int64_t rows) { return rows <= 4 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

// CTAs of a cluster that split K between them.  An SM's time is that of its
// CTAs' chunks and of starting them (some 2.3 chunks); two CTAs on an SM hide
// one another's waits (0.87 of the time).  A cluster lies within a group of 16
// SMs or a few more, so sizes that leave part of 16 x CTAs per SM empty fit
// fewer at a time.  One row, 5120 x 5120, split 1 to 8: 18.6, 11.8, 10.0, 11.2,
// 10.3, 9.9, 14.1, 13.5 us (6 is taken); 17408 x 5120: 20.9, 19.0 (taken), 24.9,
// 24.6, 27.6, 32.2, 33.1, 36.1 us.
static int linear_split(int64_t tiles, int chunks, int per_sm) {
  int best = 1;
  int64_t best_cost = 0;
  for (int s = 1; s <= 8 && (s == 1 || 2 * s <= chunks); ++s) {
    const int64_t group = 16 * per_sm, slots = num_sms() * (group / s * s) / 16;  // per_sm x SMs, less what stays empty
    const int64_t turns = (tiles * s * per_sm + slots - 1) / slots;               // of one CTA per SM
    const int64_t weight = turns > 1 && per_sm > 1 ? 87 * turns : 100 * turns;
    const int64_t cost = weight * (10 * ((chunks + s - 1) / s) + 23);
    if (s == 1 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

// Whether the wide tiles fill most of the SMs; below that the narrow kernel,
// whose clusters split K, ends sooner (wide against narrow, inner 5120: 300 rows
// of 5120 outputs, 60 tiles, 44 and 40 us; 512 rows, 80 tiles, 46 and 78; 200 rows
// of 17408, 136 tiles, 48 and 76; 333 x 1000 x 2080, 12 tiles, 43 and 15).
static bool linear_wide(int64_t rows, int64_t outs) {
  return rows > 128 && (rows + 127) / 128 * ((outs + kWideN - 1) / kWideN) >= num_sms() / 2;
}

template <bool BF16, int NT>
static int launch_terms(const TermsParams& T, cudaStream_t s) {
  const int64_t units = (T.rows + NT - 1) / NT * (NT / terms_rows(NT)) * T.chunks;
  linear_terms_kernel<BF16, NT><<<static_cast<unsigned>((units * 16 + 255) / 256), 256, 0, s>>>(T);
  return check_launch();
}

template <bool BF16>
static int launch_wide(const TermsParams& T, const uint8_t* packed, const LinearParams& P, cudaStream_t s) {
  using Tile = WideTile<BF16 ? 2 : 3>;
  CUtensorMap map;
  int status = make_tensor_map_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, packed, P.inner / 2, P.outs, P.inner / 2, kLinK / 2, kWideN,
                                  CU_TENSOR_MAP_SWIZZLE_NONE);
  if (status != MXW_OK) return status;
  status = launch_terms<BF16, 128>(T, s);
  if (status != MXW_OK) return status;
  auto kernel = linear_wide_kernel<BF16>;
  static std::atomic<uint64_t> done{0};
  status = set_max_smem_once(reinterpret_cast<const void*>(kernel), Tile::kSmem, done);
  if (status != MXW_OK) return status;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((P.outs + kWideN - 1) / kWideN), static_cast<unsigned>((P.rows + 127) / 128));
  cfg.blockDim = dim3(kWideThreads);
  cfg.dynamicSmemBytes = Tile::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, map, P);
  return err == cudaSuccess ? MXW_OK : record_cuda_error(err);
}

template <bool BF16, int NT>
static int launch_linear(const TermsParams& T, const uint8_t* packed, const LinearParams& P, cudaStream_t s) {
  constexpr int TERMS = BF16 ? 2 : 3;
  using Tile = LinearTile<NT, TERMS>;
  const int64_t tiles = (P.rows + NT - 1) / NT;
  CUtensorMap map;
  int status = make_tensor_map_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, packed, P.inner / 2, P.outs, P.inner / 2, kLinK / 2, kLinM,
                                  CU_TENSOR_MAP_SWIZZLE_NONE);
  if (status != MXW_OK) return status;
  if constexpr (!Tile::kFused) {
    status = launch_terms<BF16, NT>(T, s);
    if (status != MXW_OK) return status;
  }

  auto kernel = linear_kernel<BF16, NT>;
  static std::atomic<uint64_t> done{0};
  status = set_max_smem_once(reinterpret_cast<const void*>(kernel), Tile::kSmem, done);
  if (status != MXW_OK) return status;
  const int64_t row_tiles = (P.outs + kLinM - 1) / kLinM;
  const int split = linear_split(row_tiles * tiles, P.chunks, NT <= 32 ? 2 : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(split), static_cast<unsigned>(row_tiles), static_cast<unsigned>(tiles));
  cfg.blockDim = dim3(Tile::kThreads);
  cfg.dynamicSmemBytes = Tile::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(split), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = Tile::kFused ? 1 : 2;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, map, P);
  return err == cudaSuccess ? MXW_OK : record_cuda_error(err);
}

template <bool BF16>
static int launch_linear_rows(const TermsParams& T, const uint8_t* packed, const LinearParams& P, cudaStream_t s) {
  if (linear_wide(P.rows, P.outs)) return launch_wide<BF16>(T, packed, P, s);
  switch (linear_tile(P.rows)) {
    case 16:
      return launch_linear<BF16, 16>(T, packed, P, s);
    case 32:
      return launch_linear<BF16, 32>(T, packed, P, s);
    case 64:
      return launch_linear<BF16, 64>(T, packed, P, s);
    default:
      return launch_linear<BF16, 128>(T, packed, P, s);
  }
}

}  // namespace mxw

using namespace mxw;

extern "C" size_t mxw_linear_workspace_size(int64_t rows, int64_t inner, int dtype) {
  if (rows <= 0 || inner <= 0 || (dtype != MXW_BF16 && dtype != MXW_F16)) return 0;
  const int64_t nt = linear_tile(rows), terms = dtype == MXW_BF16 ? 2 : 3;
  if (nt == 16) return 16;  // the terms stay in shared memory
  const int64_t sf_tiles = nt < 128 ? (terms * nt + 127) / 128 : terms;
  const int64_t per_chunk = terms * nt * kLinK + sf_tiles * kLinSfBytes;
  return static_cast<size_t>((rows + nt - 1) / nt * ((inner + kLinK - 1) / kLinK) * per_chunk);
}

extern "C" int mxw_linear_mxfp4(const void* x, int dtype, int64_t rows, int64_t inner, int64_t ldx,
                                const uint8_t* packed, const uint8_t* scales, int64_t outs, const void* bias, int act,
                                const void* residual, int64_t ldr, void* y, void* workspace, size_t workspace_bytes,
                                uint32_t* flags, void* stream) {
  if (rows < 0 || outs < 0 || inner <= 0 || inner % 32 != 0 || ldx < inner) return MXW_EINVAL;
  if (dtype != MXW_BF16 && dtype != MXW_F16) return MXW_EINVAL;
  if (act < MXW_ACT_NONE || act > MXW_ACT_GELU) return MXW_EINVAL;
  if (residual && ldr < outs) return MXW_EINVAL;
  if (rows == 0 || outs == 0) return MXW_OK;
  if (!x || !packed || !scales || !y || !workspace) return MXW_EINVAL;
  if (reinterpret_cast<uintptr_t>(packed) % 16 != 0 || reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return MXW_EINVAL;
  if (workspace_bytes < mxw_linear_workspace_size(rows, inner, dtype)) return MXW_EINVAL;
  // Grid limits: 65535 tiles of 128 outputs and of 128 rows; 2^32 groups of four rows' 128 inputs.
  if (outs > 65535ll * kLinM || rows > 65535ll * 128 || inner > (1ll << 30)) return MXW_EUNSUPPORTED;
  if ((rows + 256) / 4 * ((inner + kLinK - 1) / kLinK) >= (1ll << 32) - 16) return MXW_EUNSUPPORTED;
  TermsParams T{};
  T.x = x;
  T.ldx = ldx;
  T.rows = rows;
  T.inner = inner;
  T.chunks = static_cast<int>((inner + kLinK - 1) / kLinK);
  T.x_vec = ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  T.terms = static_cast<uint8_t*>(workspace);
  LinearParams P{};
  P.scales = scales;
  P.x = x;
  P.ldx = ldx;
  P.x_vec = T.x_vec;
  P.terms = T.terms;
  P.bias = bias;
  P.residual = residual;
  P.ldr = ldr;
  P.y = y;
  P.rows = rows;
  P.outs = outs;
  P.inner = inner;
  P.chunks = T.chunks;
  P.act = act;
  P.words = inner % 128 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0;
  P.pairs = outs % 2 == 0 && reinterpret_cast<uintptr_t>(y) % 4 == 0 &&
            (!residual || (ldr % 2 == 0 && reinterpret_cast<uintptr_t>(residual) % 4 == 0));
  P.flags = flags;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MXW_BF16 ? launch_linear_rows<true>(T, packed, P, s) : launch_linear_rows<false>(T, packed, P, s);
}
