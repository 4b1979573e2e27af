#pragma once
// Rows of 8-bit codes from any byte address into rows that TMA can read: starting
// on 128-byte boundaries and filled up with zeros to whole 128-code blocks.
//
// Bound: memory, one read and one write of the rows; the copy of a layer's weights
// mostly stays in L2 for the product that follows. A lane puts 4 codes together
// from the two aligned words that hold them, a warp writes 128 bytes at a time; 8
// such pieces of a row are on their way at once. The product's own loads from
// unaligned rows, shifted on their way into the shared-memory ring, reached 1.4 TB/s
// for few tokens and a tenth of the tensor rate for many. B200, us, that and this
// copy with the product: 1 x 14336 x 4095 43, 32; 256 x 14336 x 4095 120, 37;
// 2048 x 4096 x 4095 220, 37.
#include "i8_common.cuh"

namespace aegis::i8 {

struct AlignJob {
  const int8_t* src;
  long long ld;
  int8_t* dst;
  long long tasks;  // rows x segments
};
struct AlignArgs {
  AlignJob job[2];  // matrices of the same K, one launch
  int K;
  int padded;    // columns of a row of dst: K up to whole blocks of 128
  int segments;  // pieces of 1024 columns of such a row
};

inline constexpr int kAlignThreads = 256, kAlignWords = 8;

__global__ void __launch_bounds__(kAlignThreads) i8_align_kernel(const __grid_constant__ AlignArgs a) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = int(threadIdx.x & 31);
  long long task = (long long)blockIdx.x * (kAlignThreads / 32) + (threadIdx.x >> 5);
  const bool second = task >= a.job[0].tasks;
  if (second) task -= a.job[0].tasks;
  const AlignJob job = second ? a.job[1] : a.job[0];
  if (task >= job.tasks) return;
  const long long row = task / a.segments;
  const int k0 = int(task - row * a.segments) * (128 * kAlignWords) + lane * 4;
  const int8_t* src = job.src + row * job.ld;
  int8_t* dst = job.dst + row * a.padded;
  const int mis = int(reinterpret_cast<uintptr_t>(src) & 3u);  // that of src + k too: k is a multiple of 4
  uint32_t lo[kAlignWords], hi[kAlignWords];
#pragma unroll
  for (int u = 0; u < kAlignWords; ++u) {
    const int k = k0 + 128 * u;
    lo[u] = hi[u] = 0;
    // Words that lie inside the row; those across its ends are put together below.
    const uint32_t* q = reinterpret_cast<const uint32_t*>(src + k - mis);
    if (k >= mis && k - mis + 4 <= a.K) lo[u] = *q;
    if (mis != 0 && k - mis + 8 <= a.K) hi[u] = q[1];
  }
#pragma unroll
  for (int u = 0; u < kAlignWords; ++u) {
    const int k = k0 + 128 * u;
    if (k >= a.padded) break;
    uint32_t v = __funnelshift_r(lo[u], hi[u], uint32_t(mis) * 8u);
    if (k < mis || k - mis + (mis != 0 ? 8 : 4) > a.K) {
      v = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k + i < a.K) v |= uint32_t(uint8_t(src[k + i])) << (8 * i);
    }
    *reinterpret_cast<uint32_t*>(dst + k) = v;
  }
}

}  // namespace aegis::i8
