// K11: attention over the MXFP4 cache for prompts, on the tcgen05 tensor cores.
//
// The same function as K10 where a sequence brings many query rows and the time
// is that of the products.  A block owns 256 rows (two tiles of 128; a row is
// one query of one of the heads that share a key/value head) and walks the keys
// in tiles of 64:
//   S = Q K^T   kind::mxf8f6f4: K's codes and scales go to the tensor cores as
//               they are cached; Q is split into E4M3 terms once (terms.cuh)
//   O += P V    kind::f16: P from TMEM, V decoded to f16 in shared memory.  V's
//               scales run across the contraction, so they are multiplied into
//               the codes relative to the largest so far (times 2^13): exact
//               down to 2^-27 of it, and rows with smaller ones are done again
//               (kAttSpan).
// Warps 0-3 and 4-7 are the softmax of the two row tiles, a thread a row: no
// exchange between threads.  P = 2^(x - m + 7) is rounded to f16 (11 bits; the
// sum is taken in fp32 before); m is raised only when a score passes it by 8, so
// the accumulator, which lives in TMEM, is seldom rescaled.  Warps 8-11 bring
// keys and values (cp.async a row piece at a time: pages may end anywhere in a
// tile), spread K's codes and decode V; warps 12 and 13 issue the products of a
// row tile each, so that one's waits are covered by the other's products.
// What bounds it: the chain of a row tile from scores to probabilities to the
// next scores, some 2700 cycles per 64 keys, in which the products take 1300
// (the scores' narrow ones are held back by their operands' shared-memory reads)
// and the 16,384 exponentials 1024.  Four prompts of up to 3001 new tokens over
// up to 1000 cached ones, 40 heads over 8 of 128, bf16: 590 us, 507 TFLOP/s; f16, with
// three terms, 610 us.
#include "attention.cuh"
#include "blockscale.cuh"
#include "common.cuh"
#include "runtime.h"
#include "terms.cuh"

namespace mxw {

constexpr int kPromptKeys = 64;
constexpr int kPromptRows = 128;  // rows of a tile
constexpr int kPromptThreads = 14 * 32;
constexpr int kPromptRaw = 4;     // stages of copies
constexpr int kPromptKv = 3;      // decoded tiles: one in the scores' product, one in the values', one being made

template <int D, int TERMS>
struct PromptShape {
  static constexpr int kBlocks = D / 32;
  static constexpr int kQTerm = kPromptRows * 128;             // a term of a row tile: rows of 128 bytes
  static constexpr int kQ = TERMS * (kQTerm + kLinSfBytes);    // terms, then their scales
  static constexpr int kK = kPromptKeys * 128 + kLinSfBytes;   // spread codes, then scales
  static constexpr int kV = kPromptKeys * D * 2;
  static constexpr int kKStride = (kK + 1023) / 1024 * 1024;
  static constexpr int kRawCodes = kPromptKeys * D / 2, kRawScales = kPromptKeys * kBlocks;
  static constexpr int kRawStage = 2 * (kRawCodes + kRawScales);  // [K codes][V codes][K scales][V scales]
  static constexpr int kQStride = (kQ + 1023) / 1024 * 1024;
  static constexpr int kSmem = 2 * kQStride + kPromptKv * (kKStride + kV) + kPromptRaw * kRawStage + 1024 + 512;
  // TMEM columns: S and O and P of both row tiles, the scales of Q and of two key tiles.
  static constexpr int kS = 0, kO = 2 * kPromptKeys, kP = kO + 2 * D, kSfQ = kP + kPromptKeys, kSfK = kSfQ + 8 * TERMS;
  static_assert(kSfK + 16 <= 512, "TMEM has 512 columns");
};

// D[128 x N] (+)= A B with A [128 x 16] f16 in TMEM.
__device__ __forceinline__ void mma_f16_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 32 columns of TMEM, without the wait; and the store.
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Barrier 1 over 128 threads; true when all of them bring true.
__device__ __forceinline__ bool named_barrier_and(bool on) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred.aligned q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(on))
      : "memory");
  return all != 0;
}

// The block's rows and keys: the same for every role.
struct PromptUnit {
  int q0, queries, length;
  int rows;    // of this block's 256 (0: none)
  int row0;    // first, among the sequence's queries x group
  int first;   // key that some row sees
  int lo, hi;  // and from it, rounded down to 16, to the last
  int tiles;
};

__device__ __forceinline__ PromptUnit prompt_unit(const AttParams& P, int b, int row0) {
  PromptUnit u;
  const int64_t first = P.start[b], last = P.start[b + 1];
  u.q0 = static_cast<int>(max(static_cast<int64_t>(0), min(first, P.tokens)));
  u.queries = static_cast<int>(max(static_cast<int64_t>(0), min(last, P.tokens) - u.q0));
  const int64_t held = P.table_width << P.page_shift;
  u.length = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(P.lengths[b]), held)));
  u.row0 = row0;
  u.rows = max(0, min(2 * kPromptRows, u.queries * P.group - row0));
  const int pos0 = u.length - u.queries + row0 / P.group;
  const int pos1 = u.length - u.queries + (row0 + max(u.rows, 1) - 1) / P.group;
  u.first = P.window > 0 ? max(0, pos0 - P.window + 1) : 0;
  u.lo = u.first / 16 * 16;
  u.hi = P.causal ? max(0, min(pos1 + 1, u.length)) : u.length;
  u.tiles = max(0, (u.hi - u.lo + kPromptKeys - 1) / kPromptKeys);
  return u;
}

template <bool BF16, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) attention_prompt_kernel(const AttParams P) {
  constexpr int TERMS = BF16 ? 2 : 3;
  using Shape = PromptShape<D, TERMS>;
  constexpr int BLOCKS = Shape::kBlocks;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = align_smem<1024>(smem_raw);
  uint8_t* q_smem = smem;                                  // [2 row tiles]
  uint8_t* k_smem = q_smem + 2 * Shape::kQStride;          // [3]
  uint8_t* v_smem = k_smem + kPromptKv * Shape::kKStride;  // [3]
  uint8_t* raw_smem = v_smem + kPromptKv * Shape::kV;      // [4]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(raw_smem + kPromptRaw * Shape::kRawStage);  // [2]
  uint64_t* kv_full = q_full + 2;             // [3]
  uint64_t* kv_empty = kv_full + kPromptKv;   // [3]
  uint64_t* s_full = kv_empty + kPromptKv;    // [2 row tiles]
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* o_done = p_full + 2;
  int* tile_ref = reinterpret_cast<int*>(o_done + 2);  // [3] largest scale byte of the values up to the tile
  uint32_t* tile_in = reinterpret_cast<uint32_t*>(tile_ref + kPromptKv);  // [3][2] keys whose page is one of the pool's, as bits
  int* warp_ref = reinterpret_cast<int*>(tile_in + 2 * kPromptKv);           // [2][4]
  uint32_t* tile_low = reinterpret_cast<uint32_t*>(warp_ref + 8);  // [3] and the smallest but zero, less one
  uint32_t* warp_low = tile_low + kPromptKv;                       // [2][4]
  uint32_t* tmem_slot = warp_low + 8;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.x, b = blockIdx.y;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPromptKv; ++i) {
      mbar_init(&kv_full[i], 4);
      mbar_init(&kv_empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 12) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  att_clear_rest<BF16>(P, D, (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x,
                       static_cast<int64_t>(gridDim.x) * gridDim.y * gridDim.z);

  // Row tiles from the last on: under a causal mask those see the most keys.
  // (A block takes one when the caller's bound on the queries holds.)
  const int n_units = (prompt_unit(P, b, 0).queries * P.group + 2 * kPromptRows - 1) / (2 * kPromptRows);
  bool ok = true;
  int kv = 0;     // key tiles so far (all roles count alike)
  int count[2] = {0, 0};  // key tiles so far of each row tile
  int made[2] = {0, 0};   // and its sets of queries
  for (int z = n_units - 1 - static_cast<int>(blockIdx.z); z >= 0; z -= static_cast<int>(gridDim.z)) {
    const PromptUnit u = prompt_unit(P, b, z * 2 * kPromptRows);
    if (u.rows == 0) continue;
    if (!ok) {  // a wait gave up: no more waits, and what this warp would have written is NaN
      for (int r = 32 * warp; warp < 8 && r < min(32 * warp + 32, u.rows); ++r) {
        const int at = u.row0 + r, i_q = at / P.group;
        const int64_t row = static_cast<int64_t>(u.q0 + i_q) * P.heads + head * P.group + (at - i_q * P.group);
        for (int c = lane; c < D; c += 32) att_store<BF16>(P.out, row * D + c, NAN);
        if (lane == 0 && P.lse) P.lse[row] = NAN;
      }
      continue;
    }
    const bool second = u.rows > kPromptRows;

    if (warp < 8) {
      // ------------------------------------------------------------ softmax
      const int x = warp >> 2, quarter = warp & 3;
      const int r = 32 * quarter + lane;  // this thread's row of the tile
      const int row = x * kPromptRows + r;
      if (x == 1 && !second) {
        ;
      } else {
        // The tile's queries as terms: 16 (D = 128) or 8 lanes a row, eight elements each.
        if (u.tiles > 0) {
          constexpr int PARTS = D / 8, PER = 32 / PARTS;
          const int part = lane % PARTS;
          uint8_t* qt = q_smem + x * Shape::kQStride;
#pragma unroll 4
          for (int k = 0; k < 32; k += PER) {
            const int rr = 32 * quarter + k + lane / PARTS, at = u.row0 + x * kPromptRows + rr;
            const bool in = x * kPromptRows + rr < u.rows;
            const int i = in ? at / P.group : 0, h = in ? at - i * P.group : 0;
            const uint16_t* src = static_cast<const uint16_t*>(P.query) + static_cast<int64_t>(u.q0 + i) * P.q_token +
                                  static_cast<int64_t>(head * P.group + h) * P.q_head + part * 8;
            const uint4 v = load_x8(src, in, P.q_vec);
            split_x8<BF16, 128, PARTS>(v, rr, part, qt, qt + TERMS * Shape::kQTerm, true);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[x]);
        }
        const bool live = row < u.rows;
        const int at = u.row0 + (live ? row : 0), i_q = at / P.group;
        const int pos = u.length - u.queries + i_q;
        const int key_hi = P.causal ? max(0, pos + 1) : u.length;
        const int key_lo = P.window > 0 ? max(0, pos - P.window + 1) : 0;
        // Key tiles between these bounds need no mask for any row of the warp.
        const int warp_last = min(x * kPromptRows + 32 * quarter + 31, u.rows - 1), warp_first = min(x * kPromptRows + 32 * quarter, u.rows - 1);
        const int pos_first = u.length - u.queries + (u.row0 + warp_first) / P.group;
        const int pos_last = u.length - u.queries + (u.row0 + warp_last) / P.group;
        const int open_hi = P.causal ? max(0, pos_first + 1) : u.length;
        const int open_lo = P.window > 0 ? max(0, pos_last - P.window + 1) : 0;
        const uint32_t lanes = static_cast<uint32_t>(32 * quarter) << 16;
        const uint32_t s_t = tmem + lanes + Shape::kS + x * kPromptKeys, o_t = tmem + lanes + Shape::kO + x * D;
        const uint32_t p_t = tmem + lanes + Shape::kP + x * (kPromptKeys / 2);
        float m = -INFINITY, l = 0.0f;
        int ref = 0;  // scale byte that the accumulator is relative to
        uint32_t low = 0xffffffffu;  // the smallest but zero so far, less one
        for (int t = 0; t < u.tiles; ++t) {
          const int n = count[x] + t;
          if (!__all_sync(0xffffffffu, mbar_wait_cycles(&s_full[x], n & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t s0[32], s1[32];
          tmem_load32(s_t, s0);
          tmem_load32(s_t + 32, s1);
          // (kv_full completed before the products were issued: this wait only orders the two reads.)
          const int buf = (kv + t) % kPromptKv;
          if (!__all_sync(0xffffffffu, mbar_wait_cycles(&kv_full[buf], (kv + t) / kPromptKv & 1))) {
            ok = false;
            break;
          }
          const int ref_t = *reinterpret_cast<volatile int*>(&tile_ref[buf]);
          low = min(low, *reinterpret_cast<volatile uint32_t*>(&tile_low[buf]));
          const uint32_t in0 = *reinterpret_cast<volatile uint32_t*>(&tile_in[2 * buf]);
          const uint32_t in1 = *reinterpret_cast<volatile uint32_t*>(&tile_in[2 * buf + 1]);
          tmem_wait_load();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[x]);
          const int key = u.lo + t * kPromptKeys;
          if (key < open_lo || key + kPromptKeys > open_hi) {
            const int from = key_lo - key, to = key_hi - key;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (j < from || j >= to) s0[j] = 0xff800000u;
              if (j + 32 < from || j + 32 >= to) s1[j] = 0xff800000u;
            }
          }
          if ((in0 & in1) != 0xffffffffu) {
            // Keys whose page is not one of the pool's.
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (!((in0 >> j) & 1u)) s0[j] = 0xff800000u;
              if (!((in1 >> j) & 1u)) s1[j] = 0xff800000u;
            }
          }
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; j += 4)
#pragma unroll
            for (int k = 0; k < 4; ++k) tops[k] = fmaxf(tops[k], fmaxf(bits_f32(s0[j + k]), bits_f32(s1[j + k])));
          float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          top = __fmul_rn(top, P.scale_log2);
          // The accumulator and P belong to the last tile's product until that
          // is done: seldom waited for here, else when the exponentials are.
          const bool raise = top > __fadd_rn(m, kAttSlack);
          const bool rescale = __any_sync(0xffffffffu, raise) || ref_t > ref;
          if (rescale) {
            if (t > 0 && !__all_sync(0xffffffffu, mbar_wait_cycles(&o_done[x], (n - 1) & 1))) {
              ok = false;
              break;
            }
            const float up = raise ? fmaxf(m, top) : m;
            const float fm = m == up ? 1.0f : ex2(__fsub_rn(m, up));
            m = up;
            l = __fmul_rn(l, fm);
            const float f = __fmul_rn(fm, ref_t > ref ? exp2i(max(ref - ref_t, -149)) : 1.0f);
            ref = max(ref, ref_t);
            if (t > 0) {
              tc_fence_after();
#pragma unroll
              for (int c = 0; c < D; c += 16) {
                float o[16];
                uint32_t w[16];
                tmem_ld_32x32b_x16(o_t + c, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] = f32_bits(__fmul_rn(o[j], f));
                tmem_store16(o_t + c, w);
              }
            }
          }
          const float base = __fsub_rn(kAttLift, m == -INFINITY ? 0.0f : m);
          const unsigned long long f2 = pack2(P.scale_log2, P.scale_log2), b2 = pack2(base, base);
          unsigned long long sum2 = 0ull, sum3 = 0ull;
          uint32_t p0[16], p1[16];
          auto probabilities = [&](const uint32_t (&s)[32], uint32_t (&p)[16]) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const struct f2 x2 = unpack2(fma2(pack2(bits_f32(s[2 * j]), bits_f32(s[2 * j + 1])), f2, b2));
              const float a = ex2(x2.x), c = ex2(x2.y);
              if (j & 1)
                sum2 = add2(sum2, pack2(a, c));
              else
                sum3 = add2(sum3, pack2(a, c));
              p[j] = pack_f16x2(a, c);
            }
          };
          probabilities(s0, p0);
          probabilities(s1, p1);
          if (!rescale && t > 0 && !__all_sync(0xffffffffu, mbar_wait_cycles(&o_done[x], (n - 1) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          tmem_store16(p_t, p0);
          tmem_store16(p_t + 16, p1);
          const struct f2 sums = unpack2(add2(sum2, sum3));
          l = __fadd_rn(l, __fadd_rn(sums.x, sums.y));
          tmem_wait_store();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x]);
        }
        if (u.tiles > 0 && ok) {
          if (!__all_sync(0xffffffffu, mbar_wait_cycles(&o_done[x], (count[x] + u.tiles - 1) & 1))) ok = false;
          tc_fence_after();
        }
        bool wide = ok && ref - static_cast<int>(low + 1u) > kAttSpan;  // may be: the same in all warps of the block
        if (wide) {
          AttRange<D> range;
          range.look(P, b, head, u.first, u.hi, 0, 1);
          wide = range.wide();
        }
        if (wide) {
          for (int k = 0; k < 32 && x * kPromptRows + 32 * quarter + k < u.rows; ++k) {
            const int at_k = u.row0 + x * kPromptRows + 32 * quarter + k, i_k = at_k / P.group;
            const int h_k = head * P.group + at_k - i_k * P.group, pos_k = u.length - u.queries + i_k;
            float v[D / 32];
            const float lse2 = att_row_wide<BF16, D>(
                P, b, head, static_cast<const uint16_t*>(P.query) + static_cast<int64_t>(u.q0 + i_k) * P.q_token + static_cast<int64_t>(h_k) * P.q_head,
                P.window > 0 ? max(0, pos_k - P.window + 1) : 0, P.causal ? min(pos_k + 1, u.length) : u.length, v);
            const int64_t row_k = static_cast<int64_t>(u.q0 + i_k) * P.heads + h_k;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) att_store<BF16>(P.out, row_k * D + lane * (D / 32) + c, __fmul_rn(v[c], kAttWideUnit));
            if (lane == 0 && P.lse) P.lse[row_k] = __fmul_rn(lse2, 0.69314718055994531f);
          }
        }
        if (!ok) l = NAN;  // a wait gave up: NaN, whether or not anybody reads the flags
        const bool seen = !(l == 0.0f);  // NaN counts as seen
        const float inv = seen ? __fdiv_rn(1.0f, l) : 0.0f;
        const float back = exp2i(max(ref - 140, -149));
        const int64_t out_row = static_cast<int64_t>(u.q0 + i_q) * P.heads + head * P.group + (at - i_q * P.group);
        uint16_t* out = static_cast<uint16_t*>(P.out) + out_row * D;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (u.tiles > 0) {
            tmem_load32(o_t + c, o);
            tmem_wait_load();
          }
          if (live && !wide) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float a = seen ? __fmul_rn(__fmul_rn(bits_f32(o[j + 2 * k]), inv), back) : 0.0f;
                const float e = seen ? __fmul_rn(__fmul_rn(bits_f32(o[j + 2 * k + 1]), inv), back) : 0.0f;
                if constexpr (BF16) {
                  const __nv_bfloat162 h2 = __floats2bfloat162_rn(a, e);
                  w[k] = *reinterpret_cast<const uint32_t*>(&h2);
                } else {
                  w[k] = pack_f16x2(a, e);
                }
              }
              *reinterpret_cast<uint4*>(out + c + j) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (live && !wide && P.lse) P.lse[out_row] = seen ? __fmul_rn(__fadd_rn(m, __fsub_rn(log2f(l), kAttLift)), 0.69314718055994531f) : -INFINITY;
        tc_fence_before();
      }
    } else if (warp < 12) {
      // -------------------------------------------------- keys and values in
      const int e = threadIdx.x - 256;
      const int32_t* table = P.table + static_cast<int64_t>(b) * P.table_ld;
      const int page_mask = (1 << P.page_shift) - 1;
      // Bytes of a page, from a key to its value, and this thread's places in a page (rows apart).
      const uint32_t page_codes = 2u * P.kv_heads * (D / 2) << P.page_shift, page_scales = 2u * P.kv_heads * BLOCKS << P.page_shift;
      const int64_t to_values = static_cast<int64_t>(P.kv_heads) * (D / 2) << P.page_shift;
      // Pieces of 16 bytes: D / 32 per row.  A thread's pieces lie 128 / BLOCKS rows apart.
      constexpr int PIECES = kPromptKeys * BLOCKS / 128;  // per thread: 2 or 1
      constexpr int SCALES = Shape::kRawScales / 16;      // pieces of a tensor's scales: 16 / BLOCKS keys each, of one
      const int key_e = e / BLOCKS;                       // page, as tiles start at multiples of 16
      const int scale_key = e % SCALES * (16 / BLOCKS);
      const uint8_t* codes = P.codes + (static_cast<int64_t>(head) * (D / 2) << P.page_shift) + e % BLOCKS * 16;
      const uint8_t* scales = P.scales + (static_cast<int64_t>(head) * BLOCKS << P.page_shift) +
                              (e >= SCALES ? static_cast<int64_t>(P.kv_heads) * BLOCKS << P.page_shift : 0);
      // Pages of this thread's next copies, read a tile ahead: -1 past the last key.
      int next[PIECES], next_scale = -1;
      auto look_up = [&](int t) {
        const int key = u.lo + t * kPromptKeys;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int k = key + key_e + 128 / BLOCKS * j;
          next[j] = k < u.hi ? table[k >> P.page_shift] : -1;
          if (k < u.hi && next[j] < 0) next[j] = 0x7fffffff;
        }
        if (e < 2 * SCALES) next_scale = key + scale_key < u.hi ? table[(key + scale_key) >> P.page_shift] : -1;
      };
      uint32_t strays = 0;  // tiles (mod 4) where this thread met a page that is not one of the pool's
      auto issue = [&](int t) {
        if (t < u.tiles) {
          const int n = kv + t;
          const uint32_t st = smem_u32(raw_smem) + (n % kPromptRaw) * Shape::kRawStage;
          const int key = u.lo + t * kPromptKeys;
          uint32_t stray = 0;
#pragma unroll
          for (int j = 0; j < PIECES; ++j) {
            const bool in = static_cast<uint32_t>(next[j]) < static_cast<uint32_t>(P.pages);
            stray |= !in && next[j] >= 0 ? 1u : 0u;
            const int offset = (key + key_e + 128 / BLOCKS * j) & page_mask;
            const uint8_t* kc = codes + static_cast<uint64_t>(in ? static_cast<uint32_t>(next[j]) : 0u) * page_codes + offset * (D / 2);
            const uint32_t bytes = in ? 16u : 0u;
            cp_async16(st + (e + 128 * j) * 16, kc, bytes);
            cp_async16(st + Shape::kRawCodes + (e + 128 * j) * 16, kc + to_values, bytes);
          }
          if (e < 2 * SCALES) {
            const bool in = static_cast<uint32_t>(next_scale) < static_cast<uint32_t>(P.pages);
            const uint8_t* sc = scales + static_cast<uint64_t>(in ? static_cast<uint32_t>(next_scale) : 0u) * page_scales + ((key + scale_key) & page_mask) * BLOCKS;
            cp_async16(st + 2 * Shape::kRawCodes + e * 16, sc, in ? 16u : 0u);
          }
          strays = (strays & ~(1u << (n & 3))) | (stray << (n & 3));
          look_up(t + 1);
        }
        cp_async_commit();
      };
      // The largest scale byte of a tile's values (bit 8: a stray page) and the
      // smallest but zero, by warps, a tile ahead.  Keys that no row sees have no
      // say.  (A zero byte is a block of zeros, or of values under 6 x 2^-127,
      // which count as zeros next to larger ones.)
      int sv[PIECES], sv_next[PIECES], ref = 0;
      auto find_top = [&](int t) {
        if (t >= u.tiles) return;
        const int n = kv + t;
        const uint8_t* vs = raw_smem + (n % kPromptRaw) * Shape::kRawStage + 2 * Shape::kRawCodes + Shape::kRawScales;
        int top = 0;
        uint32_t low = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int key = u.lo + t * kPromptKeys + key_e + 128 / BLOCKS * j;
          sv_next[j] = key >= u.first && key < u.hi ? vs[e + 128 * j] : 0;
          top = max(top, sv_next[j]);
          low = min(low, static_cast<uint32_t>(sv_next[j]) - 1u);
        }
        top = __reduce_max_sync(0xffffffffu, top | static_cast<int>((strays >> (n & 3)) & 1u) << 8);
        low = __reduce_min_sync(0xffffffffu, low);
        if (lane == 0) {
          warp_ref[(n & 1) * 4 + warp - 8] = top;
          warp_low[(n & 1) * 4 + warp - 8] = low;
        }
      };
      look_up(0);
      issue(0);
      issue(1);
      issue(2);
      cp_async_wait<2>();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      find_top(0);
      for (int t = 0; t < u.tiles; ++t) {
        const int n = kv + t, buf = n % kPromptKv;
        cp_async_wait<1>();  // the next tile is here
        // All warps' copies and findings, and all are done with the stage
        // refilled below.  All four warps go on, or none.
        ok = named_barrier_and(ok);
        if (!ok) break;
        issue(t + 3);
        const int* found = warp_ref + (n & 1) * 4;
        int top = max(max(found[0], found[1]), max(found[2], found[3]));
        const uint32_t* lows = warp_low + (n & 1) * 4;
        const uint32_t low = min(min(lows[0], lows[1]), min(lows[2], lows[3]));
        const bool stray = top >= 256;
        if (stray) top = max(max(found[0] & 255, found[1] & 255), max(found[2] & 255, found[3] & 255));
        ref = max(ref, top);
#pragma unroll
        for (int j = 0; j < PIECES; ++j) sv[j] = sv_next[j];
        find_top(t + 1);
        const uint8_t* raw = raw_smem + (n % kPromptRaw) * Shape::kRawStage;
        const uint8_t* ks = raw + 2 * Shape::kRawCodes;
        if (n >= kPromptKv) ok = __all_sync(0xffffffffu, mbar_wait_cycles(&kv_empty[buf], (n / kPromptKv - 1) & 1));
        if (!ok) continue;  // to the barrier, where the other warps learn of it
        if (e == 0) {
          tile_ref[buf] = ref;
          tile_low[buf] = low;
        }
        if (e < kPromptKeys) {
          uint32_t bits = 0xffffffffu;
          if (stray) {
            const int k = u.lo + t * kPromptKeys + e;
            bits = __ballot_sync(0xffffffffu, k >= u.hi || static_cast<uint32_t>(table[k >> P.page_shift]) < static_cast<uint32_t>(P.pages));
          }
          if (lane == 0) tile_in[2 * buf + (e >> 5)] = bits;
        }
        uint8_t* kd = k_smem + buf * Shape::kKStride;
        uint8_t* vd = v_smem + buf * Shape::kV;
        if (e < kPromptKeys) {
          const uint32_t word = D == 128 ? reinterpret_cast<const uint32_t*>(ks)[e] : reinterpret_cast<const uint16_t*>(ks)[e];
          *reinterpret_cast<uint32_t*>(kd + kPromptKeys * 128 + (e & 31) * 16 + (e >> 5) * 4) = word;
        }
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int unit = e + 128 * j, key = unit / BLOCKS, p = unit % BLOCKS;
          // Keys: 32 codes to slots 2p and 2p + 1 of the row's 128 bytes, swizzled over eight rows.
          const uint4 kw = reinterpret_cast<const uint4*>(raw)[unit];
          uint8_t* row = kd + key * 128;
          *reinterpret_cast<uint2*>(row + (((2 * p) ^ (key & 7)) << 4)) = make_uint2(kw.x, kw.y);
          *reinterpret_cast<uint2*>(row + (((2 * p + 1) ^ (key & 7)) << 4)) = make_uint2(kw.z, kw.w);
          // Values: 32 channels to four 16-byte slots of the key's row in a box of 64 channels.
          const uint4 vw = reinterpret_cast<const uint4*>(raw + Shape::kRawCodes)[unit];
          const int drop = ref - sv[j];
          const uint32_t factor = drop < 28 ? static_cast<uint32_t>(28 - drop) << 10 : 0u;  // f16 2^(13 - drop)
          const uint32_t f2 = factor * 0x10001u;
          uint8_t* box = vd + (p >> 1) * (kPromptKeys * 128) + key * 128;
          const uint32_t words[4] = {vw.x, vw.y, vw.z, vw.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t h[4];
            e2m1x8_to_f16x2(words[w], h);
            *reinterpret_cast<uint4*>(box + ((((p & 1) * 4 + w) ^ (key & 7)) << 4)) =
                make_uint4(hmul2(h[0], f2), hmul2(h[1], f2), hmul2(h[2], f2), hmul2(h[3], f2));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[buf]);
      }
      cp_async_wait<0>();
      ok = named_barrier_and(ok);  // before the next rows' copies, or the end of all four
    } else {
      // ------------------------------------- products of row tile warp - 12
      constexpr uint32_t idesc_s = make_idesc_e4m3_e2m1(128, kPromptKeys);
      constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (8u << 24);  // f16, B MN-major
      const int x = warp - 12;
      const bool leader = elect_one();
      const uint32_t qb = smem_u32(q_smem) + x * Shape::kQStride, ksm = smem_u32(k_smem), vsm = smem_u32(v_smem);
      const uint32_t sfq = tmem + Shape::kSfQ + x * 4 * TERMS;
      auto reached = [&](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, mbar_wait_cycles(bar, phase & 1)) != 0; };
      if (x == 1 && !second) {
        // No rows: the tiles' buffers still count this warp's word.
        for (int t = 0; t < u.tiles && ok; ++t) {
          const int n = kv + t, buf = n % kPromptKv;
          ok = reached(&kv_full[buf], n / kPromptKv);
          if (ok && leader) mbar_arrive(&kv_empty[buf]);
          __syncwarp();
        }
      } else if (u.tiles > 0) {
        ok = reached(&q_full[x], made[x]);
        for (int t = 0; t <= u.tiles && ok; ++t) {
          if (t < u.tiles) {
            // S = Q K^T, once the softmax has read the last tile's.
            const int n = kv + t, buf = n % kPromptKv;
            ok = reached(&kv_full[buf], n / kPromptKv) && (count[x] + t == 0 || reached(&s_free[x], count[x] + t - 1));
            if (!ok) break;
            tc_fence_after();
            const uint32_t kb = ksm + buf * Shape::kKStride;
            const uint32_t sfk = tmem + Shape::kSfK + 8 * x + 4 * (n & 1);
            const uint32_t a_lo = desc_k_sw128_lo(qb), b_lo = desc_k_sw128_lo(kb);
            if (leader) {
              if (t == 0) {
#pragma unroll
                for (int k = 0; k < TERMS; ++k) tmem_cp_scales(sfq + 4 * k, qb + TERMS * Shape::kQTerm + k * kLinSfBytes);
              }
              tmem_cp_scales(sfk, kb + kPromptKeys * 128);
#pragma unroll
              for (int k = 0; k < TERMS; ++k)
#pragma unroll
                for (int kk = 0; kk < BLOCKS; ++kk)
                  mma_mxf8f6f4(tmem + Shape::kS + x * kPromptKeys, desc_of(kDescKSw128Hi, a_lo + k * (Shape::kQTerm >> 4) + 2 * kk),
                               desc_of(kDescKSw128Hi, b_lo + 2 * kk), mx_idesc_scale_byte(idesc_s, kk), sfq + 4 * k, sfk,
                               (k > 0 || kk > 0) ? 1u : 0u);
              mma_commit(&s_full[x]);
            }
            __syncwarp();
          }
          if (t > 0) {
            // O += P V of the tile before.
            const int n = kv + t - 1, buf = n % kPromptKv;
            ok = reached(&p_full[x], count[x] + t - 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t vb = vsm + buf * Shape::kV;
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < kPromptKeys / 16; ++kk)
                mma_f16_tmem(tmem + Shape::kO + x * D, tmem + Shape::kP + x * (kPromptKeys / 2) + 8 * kk,
                             make_smem_desc_mn_sw128(vb + kk * 2048, kPromptKeys * 128, 1024), idesc_o, (t > 1 || kk > 0) ? 1u : 0u);
              mma_commit(&o_done[x]);
              mma_commit(&kv_empty[buf]);
            }
            __syncwarp();
          }
        }
      }
    }
    if (u.tiles > 0) {
      kv += u.tiles;
      count[0] += u.tiles;
      ++made[0];
      if (second) {
        count[1] += u.tiles;
        ++made[1];
      }
    }
  }
  if (!ok && P.flags) atomicOr(P.flags, MXW_FLAG_TIMEOUT);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool BF16, int D>
static int launch_prompt(const AttParams& P, int64_t row_tiles, cudaStream_t s) {
  using Shape = PromptShape<D, BF16 ? 2 : 3>;
  auto kernel = attention_prompt_kernel<BF16, D>;
  static std::atomic<uint64_t> done{0};
  const int status = set_max_smem_once(reinterpret_cast<const void*>(kernel), Shape::kSmem, done);
  if (status != MXW_OK) return status;
  const dim3 grid(static_cast<unsigned>(P.kv_heads), static_cast<unsigned>(P.seqs), static_cast<unsigned>(row_tiles));
  kernel<<<grid, kPromptThreads, Shape::kSmem, s>>>(P);
  return check_launch();
}

static int64_t prompt_tiles(int64_t group, int64_t max_queries) {
  return std::max<int64_t>(1, std::min<int64_t>((max_queries * group + 2 * kPromptRows - 1) / (2 * kPromptRows), 65535));
}

// One block holds an SM and takes a sequence's keys whole, where the decoding
// kernel spreads them over the GPU: it needs enough blocks, and rows to fill
// its tiles.  Here against there, 40 heads over 8: one sequence of 16 queries
// and 4000 keys (8 blocks) 85 and 31 us; eight of them (64 blocks) 86 and 90; one
// of 256 queries and 2256 keys (40 blocks) 70 and 104; 32 of 16 queries and 2000
// keys 108 and 178.
bool attention_prompt_fits(int64_t seqs, int64_t heads, int64_t kv_heads, int64_t max_queries) {
  const int64_t group = heads / kv_heads;
  return max_queries * group > kPromptRows / 2 && seqs * kv_heads * prompt_tiles(group, max_queries) >= num_sms() / 5;
}

int launch_attention_prompt(const AttParams& P, int bf16, int dim, int64_t max_queries, cudaStream_t s) {
  const int64_t tiles = prompt_tiles(P.group, max_queries);
  if (bf16) return dim == 128 ? launch_prompt<true, 128>(P, tiles, s) : launch_prompt<true, 64>(P, tiles, s);
  return dim == 128 ? launch_prompt<false, 128>(P, tiles, s) : launch_prompt<false, 64>(P, tiles, s);
}

}  // namespace mxw
