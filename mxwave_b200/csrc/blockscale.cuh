// Block-scaled tcgen05 products (kind::mxf8f6f4) in inline PTX, sm_100a: the
// tensor cores read E2M1 and E4M3 operands with one E8M0 scale per 32 elements
// of the contraction, which is MXFP4 as the quantizer stores it.
#pragma once

#include <stdint.h>

#include "tcgen05.cuh"
#include "tma.cuh"

namespace mxw {

// Instruction descriptor, kind::mxf8f6f4: A = E2M1, B = E4M3, E8M0 scales,
// fp32 D, both operands K-major.  The two scale ids (which byte of a TMEM
// scale word the instruction takes) are OR-ed in by mx_idesc_scale_byte.
__host__ __device__ constexpr uint32_t make_idesc_e2m1_e4m3(int m, int n) {
  return (5u << 7)                                   // A format: E2M1
         | (0u << 10)                                // B format: E4M3
         | (static_cast<uint32_t>(n >> 3) << 17)     // N / 8
         | (1u << 23)                                // scale format: E8M0
         | (static_cast<uint32_t>(m >> 4) << 24);    // M / 16
}

// The same with A = E4M3 and B = E2M1.
__host__ __device__ constexpr uint32_t make_idesc_e4m3_e2m1(int m, int n) {
  return (0u << 7) | (5u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 4) << 24);
}

// A K-major 128-byte-swizzled operand: the descriptor's upper half, and the
// lower for a 1024-byte aligned address (advance by 2 per 32 bytes of K).
constexpr uint32_t kDescKSw128Hi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_sw128_lo(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint64_t desc_of(uint32_t hi, uint32_t lo) {
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ uint32_t mx_idesc_scale_byte(uint32_t idesc, uint32_t byte) {
  return idesc | (byte << 4) | (byte << 29);
}

// D[128 x N] (+)= (A 2^sa) (B 2^sb)^T over 32 elements of K.
__device__ __forceinline__ void mma_mxf8f6f4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t sfa_tmem, uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
      : "memory");
}

// Copies the scales of 128 operand rows x 4 blocks (512 bytes of shared memory,
// [row % 32][row / 32][block]) to four TMEM columns of all four lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t saddr) {
  const uint64_t desc = make_smem_desc_k_noswz(saddr, 0, 128);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// One lane of a converged warp.  The issuing warp runs its loop whole and lets
// this lane issue: its addresses and descriptors then stay in uniform
// registers, where a single-lane branch moves each operand there anew (some 65
// cycles per instruction).
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on != 0;
}

// mbar_wait with its limit counted in SM cycles (2 s at 2 GHz), and no timer
// read by a wait that is over at once.
__device__ __forceinline__ bool mbar_wait_cycles(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long start = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() - start > 4000000000ll) return false;
  }
  return true;
}

// Untiled asynchronous copies into shared memory.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(smem_dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t saddr, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Programmatic dependent launch: wait for the kernel before this one in the
// stream; let the next one be scheduled.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace mxw
