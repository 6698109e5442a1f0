// K9: a paged key/value cache in MXFP4: writing rows, reading them back, and
// copying pages.
//
// One layer of the cache is
//   codes  [pages][2 (key, value)][kv heads][page tokens][dim / 2]
//   scales [pages][2][kv heads][page tokens][dim / 32]
// with every row encoded as the quantizer encodes a weight row (E2M1, element
// 2j in the low nibble; E8M0 per 32 elements) under its `rtn` rule:
//   e = floor(log2 amax) - 2, plus 1 when amax >= 1.75 2^floor(log2 amax)
// clamped to [-127, 127].  Token `slot` lives in page slot / page_tokens.
//
// All three kernels move bytes once.  Page copies run at HBM's rate (400
// pages of 16 layers, 0.9 GB read and written, in 135 us: 6.6 TB/s); appending and
// reading back are bound by the encoding's instructions in large calls (16,384
// bf16 tokens of 8 heads of 128 written and read back: 44 us where their bytes
// take 26) and by the launches in small ones (4.5 us for both).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdlib.h>

#include "common.cuh"
#include "f16mma.cuh"
#include "runtime.h"

namespace mxw {

constexpr int kKvThreads = 256;

struct KvRows {
  uint8_t* codes;
  uint8_t* scales;
  const int64_t* slots;
  int64_t tokens, n_slots;  // slots of the pool
  int heads, dim, page_shift;
  int units;      // eight-element pieces of a token: 2 heads dim / 8
  int per_block;  // tokens per block
  float zero, negzero;  // 0 and -0 that the compiler does not know (mul2_rounded)
};

// Where piece `r` of a token lies: part (0 key, 1 value), head, first element.
struct KvPiece {
  int part, head, d;
};
__device__ __forceinline__ KvPiece kv_piece(const KvRows& P, int r) {
  const int shift = P.dim == 128 ? 4 : 3;
  const int hh = r >> shift;
  const int part = hh >= P.heads ? 1 : 0;
  return {part, hh - part * P.heads, (r & ((1 << shift) - 1)) * 8};
}

// The row's index among all rows of the pool.
__device__ __forceinline__ int64_t kv_row(const KvRows& P, int64_t slot, const KvPiece& p) {
  const int64_t page = slot >> P.page_shift, offset = slot & ((1 << P.page_shift) - 1);
  return (((page * 2 + p.part) * P.heads + p.head) << P.page_shift) + offset;
}

// Eight elements of one row, as they are; VEC: 16-byte aligned.
template <int DT, bool VEC>
struct KvRaw {
  static constexpr int kWords = DT == MXW_F32 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (VEC) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * (DT == MXW_F32 ? 4 : 2));
#pragma unroll
      for (int k = 0; k < kWords / 4; ++k) reinterpret_cast<uint4*>(w)[k] = src[k];
    } else if constexpr (DT == MXW_F32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = static_cast<const uint32_t*>(p)[i + k];
    } else {
      const uint16_t* src = static_cast<const uint16_t*>(p) + i;
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = src[2 * k] | (static_cast<uint32_t>(src[2 * k + 1]) << 16);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = 0;
  }
  // Elements 2k and 2k + 1.
  __device__ __forceinline__ f2 pair(int k) const {
    if constexpr (DT == MXW_F32) return {bits_f32(w[2 * k]), bits_f32(w[2 * k + 1])};
    if constexpr (DT == MXW_BF16) return {bits_f32(w[k] << 16), bits_f32(w[k] & 0xffff0000u)};
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    return {f.x, f.y};
  }
  // The largest magnitude as bits of the type: ordered, NaN above infinity.
  __device__ __forceinline__ uint32_t largest() const {
    if constexpr (DT == MXW_F32) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, w[k] & 0x7fffffffu);
      return m;
    }
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
  }
  // And those bits as fp32 bits.
  static __device__ __forceinline__ uint32_t to_f32_bits(uint32_t m) {
    if constexpr (DT == MXW_F32) return m;
    if constexpr (DT == MXW_BF16) return m << 16;
    const uint16_t h = static_cast<uint16_t>(m);
    return f32_bits(__half2float(*reinterpret_cast<const __half*>(&h)));
  }
};

struct KvSource {
  const void *key, *value;
  int64_t key_token, key_head, value_token, value_head;  // strides in elements
};

// Eight elements per thread, a block of 32 per four neighbours: the largest
// magnitude over two shuffles, one 4-byte store of codes each, and the first
// of them stores the scale.  TOK tokens per thread, loads first: with one, a
// block's life is one chain of dependent loads and HBM waits (kKvAhead has
// the times).
template <int DT, bool VEC, int TOK>
__global__ void __launch_bounds__(kKvThreads) kv_append_kernel(const KvRows P, const KvSource S) {
  const int sub = P.per_block == 1 ? 0 : static_cast<int>(threadIdx.x) / P.units;
  const int first = static_cast<int>(threadIdx.x) - sub * P.units;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * P.per_block * TOK + sub;
  // The loop count is the block's, so that the shuffles see whole warps.
  for (int r0 = 0; r0 < P.units; r0 += P.per_block == 1 ? kKvThreads : P.units) {
    const int r = first + r0;
    const bool on = sub < P.per_block && r < P.units;
    const KvPiece p = kv_piece(P, on ? r : 0);
    const void* src = p.part ? S.value : S.key;
    const int64_t step = p.part ? S.value_token : S.key_token;
    const int64_t at = p.head * (p.part ? S.value_head : S.key_head) + p.d;
    KvRaw<DT, VEC> raw[TOK];
    int64_t slot[TOK];
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      const int64_t token = token0 + static_cast<int64_t>(k) * P.per_block;
      const bool in = on && token < P.tokens;
      slot[k] = in ? P.slots[token] : -1;
      if (in)
        raw[k].load(src, token * step + at);
      else
        raw[k].clear();
    }
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      uint32_t top = raw[k].largest();
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t amax = KvRaw<DT, VEC>::to_f32_bits(top);
      // Exponent of the block (the quantizer's rtn rule, its non-finite cases
      // included: -127 for a NaN or zero maximum, 127 for an infinite one).
      int e;
      if (amax > 0x7f800000u || amax == 0u) {
        e = -127;
      } else if (amax == 0x7f800000u) {
        e = 127;
      } else {
        const uint32_t safe = max(amax, 0x00800000u);
        e = static_cast<int>(safe >> 23) - 129 + ((safe & 0x7fffffu) >= 0x600000u ? 1 : 0);
        e = max(e, -127);
      }
      if (slot[k] >= 0 && slot[k] < P.n_slots) {
        const float inv = exp2i(-e);
        const unsigned long long inv2 = pack2(inv, inv), nz2 = pack2(P.negzero, P.negzero), z2 = pack2(P.zero, P.zero);
        uint32_t bytes[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f2 v = raw[k].pair(i);
          f2 x = unpack2(add2(mul2_rounded(pack2(v.x, v.y), inv2, nz2), z2));  // -0 + 0 = 0: code 0
          if (amax > 0x7f800000u) {  // a NaN takes the last code, without a sign
            if (x.x != x.x) x.x = 6.0f;
            if (x.y != x.y) x.y = 6.0f;
          }
          bytes[i] = e2m1x2(x.x, x.y);
        }
        const uint32_t word = __byte_perm(__byte_perm(bytes[0], bytes[1], 0x0040), __byte_perm(bytes[2], bytes[3], 0x0040), 0x5410);
        const int64_t row = kv_row(P, slot[k], p);
        *reinterpret_cast<uint32_t*>(P.codes + row * (P.dim / 2) + p.d / 2) = word;
        if ((r & 3) == 0) P.scales[row * (P.dim / 32) + p.d / 32] = static_cast<uint8_t>(e + 127);
      }
    }
  }
}

__device__ __forceinline__ void kv_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void kv_store8(__nv_bfloat16* p, const float (&v)[8]) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ void kv_store8(__half* p, const float (&v)[8]) {
  __half2 h[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) h[k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}

// Rows read back as values, [tokens][heads][dim] each; zeros for a slot that
// lies outside the pool.
template <typename OUT, int TOK>
__global__ void __launch_bounds__(kKvThreads) kv_gather_kernel(const KvRows P, OUT* key, OUT* value) {
  const int sub = P.per_block == 1 ? 0 : static_cast<int>(threadIdx.x) / P.units;
  if (sub >= P.per_block) return;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * P.per_block * TOK + sub;
  int64_t slot[TOK];
#pragma unroll
  for (int k = 0; k < TOK; ++k) {
    const int64_t token = token0 + static_cast<int64_t>(k) * P.per_block;
    slot[k] = token < P.tokens ? P.slots[token] : -1;
    if (slot[k] >= P.n_slots) slot[k] = -1;
  }
  for (int r = static_cast<int>(threadIdx.x) - sub * P.units; r < P.units; r += P.per_block == 1 ? kKvThreads : P.units) {
    const KvPiece p = kv_piece(P, r);
    uint32_t word[TOK], byte[TOK];
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      word[k] = byte[k] = 0;  // reads as zeros
      if (slot[k] >= 0) {
        const int64_t row = kv_row(P, slot[k], p);
        word[k] = *reinterpret_cast<const uint32_t*>(P.codes + row * (P.dim / 2) + p.d / 2);
        byte[k] = P.scales[row * (P.dim / 32) + p.d / 32];
      }
    }
#pragma unroll
    for (int k = 0; k < TOK; ++k) {
      const int64_t token = token0 + static_cast<int64_t>(k) * P.per_block;
      if (token >= P.tokens) break;
      const float sc = exp2i(static_cast<int>(byte[k]) - 127);
      uint32_t h[4];
      e2m1x8_to_f16x2(word[k], h);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = __fmul_rn(q.x, sc);
        v[2 * i + 1] = __fmul_rn(q.y, sc);
      }
      kv_store8((p.part ? value : key) + (token * P.heads + p.head) * P.dim + p.d, v);
    }
  }
}

// --------------------------------------------------------------- page copies
//
// The pairs travel as a kernel argument: no copy to the device, nothing to
// keep alive until the launch runs, and the call can be captured in a graph.
// Two sizes: 16 KB of arguments cost the host 6.8 us a call, 512 bytes 3.8.
template <int N>
struct PagePairs {
  int32_t source[N], target[N];
};

struct PageCopy {
  uint8_t* codes;
  uint8_t* scales;
  int64_t pages, layers;
  int64_t code_vec, scale_vec;  // 16-byte vectors of one page
};

constexpr int kCopyVecs = 4;  // vectors per thread: enough loads in flight to cover HBM's latency

template <int N>
__global__ void __launch_bounds__(kKvThreads) copy_pages_kernel(const PageCopy P, const __grid_constant__ PagePairs<N> pairs) {
  const int64_t layer = blockIdx.z;
  const int i = blockIdx.y;
  const int64_t vecs = P.code_vec + P.scale_vec;
  const int64_t src = layer * P.pages + pairs.source[i], dst = layer * P.pages + pairs.target[i];
  uint4* codes = reinterpret_cast<uint4*>(P.codes);
  uint4* scales = reinterpret_cast<uint4*>(P.scales);
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kKvThreads * kCopyVecs) + threadIdx.x;
  uint4 v[kCopyVecs];
#pragma unroll
  for (int k = 0; k < kCopyVecs; ++k) {
    const int64_t j = base + k * kKvThreads;
    if (j < P.code_vec)
      v[k] = codes[src * P.code_vec + j];
    else if (j < vecs)
      v[k] = scales[src * P.scale_vec + j - P.code_vec];
  }
#pragma unroll
  for (int k = 0; k < kCopyVecs; ++k) {
    const int64_t j = base + k * kKvThreads;
    if (j < P.code_vec)
      codes[dst * P.code_vec + j] = v[k];
    else if (j < vecs)
      scales[dst * P.scale_vec + j - P.code_vec] = v[k];
  }
}

template <int N>
static int launch_copy(const PageCopy& P, const int64_t* source, const int64_t* target, int64_t n, cudaStream_t s) {
  const unsigned blocks =
      static_cast<unsigned>((P.code_vec + P.scale_vec + kKvThreads * kCopyVecs - 1) / (kKvThreads * kCopyVecs));
  PagePairs<N> pairs;
  for (int64_t done = 0; done < n; done += N) {
    const int now = static_cast<int>(std::min<int64_t>(N, n - done));
    for (int i = 0; i < N; ++i) {
      pairs.source[i] = i < now ? static_cast<int32_t>(source[done + i]) : 0;
      pairs.target[i] = i < now ? static_cast<int32_t>(target[done + i]) : 0;
    }
    copy_pages_kernel<N><<<dim3(blocks, static_cast<unsigned>(now), static_cast<unsigned>(P.layers)), kKvThreads, 0, s>>>(
        P, pairs);
    const int status = check_launch();
    if (status != MXW_OK) return status;
  }
  return MXW_OK;
}

static bool kv_shape_ok(int64_t pages, int64_t heads, int64_t page, int64_t dim) {
  if (dim != 64 && dim != 128) return false;
  if (page != 16 && page != 32 && page != 64 && page != 128) return false;
  return pages >= 0 && pages <= 0x7fffffff && heads >= 1 && heads <= 1024;
}

static KvRows kv_rows(uint8_t* codes, uint8_t* scales, const int64_t* slots, int64_t tokens, int64_t pages,
                      int64_t heads, int64_t page, int64_t dim) {
  KvRows P{};
  P.codes = codes;
  P.scales = scales;
  P.slots = slots;
  P.tokens = tokens;
  P.n_slots = pages * page;
  P.heads = static_cast<int>(heads);
  P.dim = static_cast<int>(dim);
  P.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  P.units = static_cast<int>(2 * heads * dim / 8);
  P.per_block = std::max(1, kKvThreads / P.units);
  P.zero = 0.0f;
  P.negzero = -0.0f;
  return P;
}

// Tokens per thread: kKvAhead once every SM has a block of them, one below
// (append of 64, 592, 1184, 2368, 16,384 bf16 tokens of 8 heads of 128: 3.9,
// 5.2, 7.2, 11.3, 60.7 us with one, 5.1, 5.0, 6.2, 8.7, 44 us with four).
constexpr int kKvAhead = 4;
static int kv_tokens_per_thread(const KvRows& P) {
  return P.tokens >= static_cast<int64_t>(P.per_block) * kKvAhead * num_sms() ? kKvAhead : 1;
}
static unsigned kv_grid(const KvRows& P, int tok) {
  const int64_t each = static_cast<int64_t>(P.per_block) * tok;
  return static_cast<unsigned>((P.tokens + each - 1) / each);
}

template <int DT, bool VEC>
static void launch_append(const KvRows& P, const KvSource& S, cudaStream_t s) {
  const int tok = kv_tokens_per_thread(P);
  if (tok == 1)
    kv_append_kernel<DT, VEC, 1><<<kv_grid(P, tok), kKvThreads, 0, s>>>(P, S);
  else
    kv_append_kernel<DT, VEC, kKvAhead><<<kv_grid(P, tok), kKvThreads, 0, s>>>(P, S);
}
template <int DT>
static void launch_append(const KvRows& P, const KvSource& S, bool vec, cudaStream_t s) {
  if (vec)
    launch_append<DT, true>(P, S, s);
  else
    launch_append<DT, false>(P, S, s);
}

template <typename OUT>
static void launch_gather(const KvRows& P, void* key, void* value, cudaStream_t s) {
  const int tok = kv_tokens_per_thread(P);
  if (tok == 1)
    kv_gather_kernel<OUT, 1><<<kv_grid(P, tok), kKvThreads, 0, s>>>(P, static_cast<OUT*>(key), static_cast<OUT*>(value));
  else
    kv_gather_kernel<OUT, kKvAhead><<<kv_grid(P, tok), kKvThreads, 0, s>>>(P, static_cast<OUT*>(key), static_cast<OUT*>(value));
}

}  // namespace mxw

using namespace mxw;

extern "C" int mxw_kv_append(uint8_t* codes, uint8_t* scales, int64_t pages, int64_t heads, int64_t page_tokens,
                             int64_t dim, const void* key, const void* value, int dtype, int64_t key_token,
                             int64_t key_head, int64_t value_token, int64_t value_head, const int64_t* slots,
                             int64_t tokens, void* stream) {
  if (!kv_shape_ok(pages, heads, page_tokens, dim) || tokens < 0) return MXW_EINVAL;
  if (dtype != MXW_BF16 && dtype != MXW_F16 && dtype != MXW_F32) return MXW_EINVAL;
  if (key_token < 0 || key_head < 0 || value_token < 0 || value_head < 0) return MXW_EINVAL;
  if (tokens == 0 || pages == 0) return MXW_OK;
  if (!codes || !scales || !key || !value || !slots) return MXW_EINVAL;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return MXW_EINVAL;
  if (tokens > 0x7fffffff) return MXW_EUNSUPPORTED;
  const KvRows P = kv_rows(codes, scales, slots, tokens, pages, heads, page_tokens, dim);
  const KvSource S{key, value, key_token, key_head, value_token, value_head};
  const int64_t strides = key_token | key_head | value_token | value_head;
  const bool vec = strides % 8 == 0 && reinterpret_cast<uintptr_t>(key) % 16 == 0 && reinterpret_cast<uintptr_t>(value) % 16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MXW_BF16)
    launch_append<MXW_BF16>(P, S, vec, s);
  else if (dtype == MXW_F16)
    launch_append<MXW_F16>(P, S, vec, s);
  else
    launch_append<MXW_F32>(P, S, vec, s);
  return check_launch();
}

extern "C" int mxw_kv_gather(const uint8_t* codes, const uint8_t* scales, int64_t pages, int64_t heads,
                             int64_t page_tokens, int64_t dim, const int64_t* slots, int64_t tokens, int dtype,
                             void* key, void* value, void* stream) {
  if (!kv_shape_ok(pages, heads, page_tokens, dim) || tokens < 0) return MXW_EINVAL;
  if (dtype != MXW_BF16 && dtype != MXW_F16 && dtype != MXW_F32) return MXW_EINVAL;
  if (tokens == 0) return MXW_OK;
  if ((pages > 0 && (!codes || !scales)) || !slots || !key || !value) return MXW_EINVAL;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(key) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(value) % 16 != 0)
    return MXW_EINVAL;
  if (tokens > 0x7fffffff) return MXW_EUNSUPPORTED;
  const KvRows P = kv_rows(const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales), slots, tokens, pages, heads,
                           page_tokens, dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MXW_BF16)
    launch_gather<__nv_bfloat16>(P, key, value, s);
  else if (dtype == MXW_F16)
    launch_gather<__half>(P, key, value, s);
  else
    launch_gather<float>(P, key, value, s);
  return check_launch();
}

extern "C" int mxw_copy_pages(uint8_t* codes, uint8_t* scales, int64_t layers, int64_t pages, int64_t code_bytes,
                              int64_t scale_bytes, const int64_t* source, const int64_t* target, int64_t n,
                              void* stream) {
  if (layers < 0 || pages < 0 || pages > 0x7fffffff || n < 0) return MXW_EINVAL;
  if (code_bytes <= 0 || scale_bytes <= 0 || code_bytes % 16 != 0 || scale_bytes % 16 != 0) return MXW_EINVAL;
  if (layers == 0 || n == 0) return MXW_OK;
  if (!codes || !scales || !source || !target) return MXW_EINVAL;
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || reinterpret_cast<uintptr_t>(scales) % 16 != 0) return MXW_EINVAL;
  if (layers > 65535 || code_bytes + scale_bytes > (1ll << 40)) return MXW_EUNSUPPORTED;
  for (int64_t i = 0; i < n; ++i)
    if (source[i] < 0 || source[i] >= pages || target[i] < 0 || target[i] >= pages) return MXW_EINVAL;
  // Copies of one call run in no order: a target may be neither a source nor another copy's target.
  uint8_t* seen = static_cast<uint8_t*>(calloc(static_cast<size_t>(pages), 1));
  if (!seen) return MXW_EUNSUPPORTED;
  bool clash = false;
  for (int64_t i = 0; i < n; ++i) {
    clash |= seen[target[i]] != 0;
    seen[target[i]] = 1;
  }
  for (int64_t i = 0; i < n; ++i) clash |= seen[source[i]] != 0;
  free(seen);
  if (clash) return MXW_EINVAL;
  PageCopy P{};
  P.codes = codes;
  P.scales = scales;
  P.pages = pages;
  P.layers = layers;
  P.code_vec = code_bytes / 16;
  P.scale_vec = scale_bytes / 16;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return n <= 64 ? launch_copy<64>(P, source, target, n, s) : launch_copy<2000>(P, source, target, n, s);
}
