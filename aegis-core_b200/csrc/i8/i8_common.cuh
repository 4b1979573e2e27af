#pragma once
// Device pieces shared by the 8-bit product's kernels: the kind::i8 forms of
// tcgen05.mma, and the scaled store of an accumulator.
#include "../common.cuh"
#include "../ptx.cuh"
#include "i8.h"

namespace aegis::i8 {

inline constexpr int BK = 128;  // int8 codes of a k-block: one 128-byte swizzle row

// Instruction descriptor, kind::i8: D = S32 (bits 4-5 = 2), A and B signed
// 8-bit (bits 7-9 and 10-12 = 1), both K-major, N >> 3 (bits 17-22), M >> 4
// (bits 24-28), no saturation.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t(N) >> 3) << 17) | ((uint32_t(M) >> 4) << 24);
}

// D[tmem] (+)= A[smem desc] * B[smem desc] over 32 codes of K, int32 accumulators.
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Barrier of the cluster's threads that orders no memory operation: a thread that has
// passed it knows only that every other one has come to it. Loads whose values have been
// used before, and remote arrivals that were waited for where they go, are over then;
// a remote store or arrival that nobody has waited for is not. cluster_sync's release
// covers those, and waits for this thread's stores to C to be visible too (0.7 us).
__device__ __forceinline__ void cluster_step() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// 16 bytes of another CTA's shared memory (a shared::cluster address).
__device__ __forceinline__ int4 ld_cluster_v4(uint32_t cluster_addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// One value of a vector of the output type (the bias), as float.
__device__ __forceinline__ float load_as_f32(const void* p, long long i, Out t) {
  if (t == Out::F32) return static_cast<const float*>(p)[i];
  if (t == Out::BF16) return Elem<__nv_bfloat16>::to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return Elem<__half>::to_f32(static_cast<const __half*>(p)[i]);
}

// A token's scale, s * f: f is 1, but for scales from 2^97 on, with which a sum of up
// to 2^31 would leave float's range before the channel's scale brings it back. Those are
// taken 2^64 smaller (the product with any channel's scale is then below the range only
// where it is 0) and the result 2^64 larger, both exact. Small scales need nothing: a
// whole number times one of float's smallest is not rounded.
struct TokenScale {
  float s, f;
};
__device__ __forceinline__ TokenScale token_scale(float sa) {
  const bool large = fabsf(sa) >= 0x1p97f;
  return {large ? sa * 0x1p-64f : sa, large ? 0x1p64f : 1.f};
}

// acc * a_scale * w_scale (+ bias). The conversion of acc to float rounds sums
// above 2^24 (relative 2^-24); each step is one float rounding, written as
// separate intrinsics so every kernel gives the same bits.
__device__ __forceinline__ float scaled(int acc, float s, float sw) { return __fmul_rn(__fmul_rn(float(acc), s), sw); }
__device__ __forceinline__ float scaled(int acc, const TokenScale& sa, float sw) {
  const float v = scaled(acc, sa.s, sw);
  return sa.f == 1.f ? v : __fmul_rn(v, sa.f);
}
__device__ __forceinline__ float scaled(int acc, const TokenScale& sa, float sw, float bias) {
  return __fadd_rn(scaled(acc, sa, sw), bias);
}

__device__ __forceinline__ void store_one(void* c, long long i, float v, Out t) {
  if (t == Out::F32) static_cast<float*>(c)[i] = v;
  else if (t == Out::BF16) static_cast<__nv_bfloat16*>(c)[i] = Elem<__nv_bfloat16>::from_f32(v);
  else static_cast<__half*>(c)[i] = Elem<__half>::from_f32(v);
}

}  // namespace aegis::i8
