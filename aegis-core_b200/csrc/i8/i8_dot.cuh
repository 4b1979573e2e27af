#pragma once
// The 8-bit product for up to 8 tokens, on CUDA cores: each warp takes 4
// channels, its lanes read the channels' codes side by side and multiply them
// with the tokens' (dp4a: 4 products a lane and instruction), and the lanes'
// int32 sums are added with one warp reduction each. No shared-memory ring, TMEM
// or cluster, whose set-up and hand-overs take the tensor-core kernel (i8_stream.cuh)
// as long as a small layer's weights take to arrive.
//
// Bound: the weight stream. A token's codes come out of L1 after the first
// warp's read; 4 channels share each read. dp4a runs at 64 lanes a clock and
// SM; 8 tokens at the weights' rate from DRAM (23 B a clock and SM) would keep it three
// quarters busy: more tokens belong on the tensor cores. B200, cold L2: 1 x 4096 x 4096
// 6.0 us (2.8 TB/s; launch to launch 1.4 and the first loads' 1.2 are half of it).
//
// `parts` warps share 4 channels, every parts-th piece of K each, when the
// channels alone do not fill the GPU; their sums meet in shared memory. Whole
// numbers: the result does not depend on it.
#include "i8_common.cuh"

namespace aegis::i8 {

struct DotArgs {
  int M, N, K;
  int parts;          // warps of a block that share channels: 1, 2, 4 or 8
  int weights_early;  // as StreamArgs
  const int8_t* A;
  const int8_t* W;
  long long lda, ldw, ldc;
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  void* C;
  Out out;
};

inline constexpr int kDotThreads = 256, kDotWarps = kDotThreads / 32, kDotChannels = 4;

// 16 codes at column k of a row whose pieces are 16-byte aligned; codes from column K on
// are zero. Plain loads: the grid before this one may have written the codes while this
// one was starting, and the read-only path could miss that.
__device__ __forceinline__ uint4 piece16(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t v[4] = {0, 0, 0, 0};
  for (int i = 0; k + i < K; ++i) {
    const uint32_t b = uint8_t(row[k + i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] |= (i >> 2) == j ? b << (8 * (i & 3)) : 0u;
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// MT tokens (M of them real). Every row of A and W starts on a 16-byte boundary; K > 0.
template <int MT>
__global__ void __launch_bounds__(kDotThreads, 2) i8_dot_kernel(const __grid_constant__ DotArgs a) {
  constexpr int C = kDotChannels;
  __shared__ int sums[kDotWarps][C * MT];
  const int warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31);
  const int part = warp & (a.parts - 1);
  const int group = int(blockIdx.x) * (kDotWarps / a.parts) + warp / a.parts;
  const int n0 = group * C;
  // Channels beyond the last one repeat it: their sums are not stored.
  const int8_t* w[C];
#pragma unroll
  for (int c = 0; c < C; ++c) w[c] = a.W + (long long)min(n0 + c, a.N - 1) * a.ldw;
  int acc[C][MT];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[c][m] = 0;

  constexpr int U = MT <= 2 ? 4 : 2;  // pieces of each channel on their way: 128 or 64 bytes a lane and channel
  constexpr int kPiece = 512;         // codes of a row that a warp reads at once
  const int stride = a.parts * kPiece;
  int k = part * kPiece + lane * 16;
  uint4 ww[U][C];
  auto load_weights = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c)
        ww[u][c] = k0 + u * stride < a.K ? piece16(w[c], k0 + u * stride, a.K) : make_uint4(0, 0, 0, 0);
  };
  if (a.weights_early) {
    load_weights(k);
  } else if (lane % 8 == 0) {
    // A hint: lines of the first pieces into L2 while the previous grid ends.
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (k + u * stride < a.K) ptx::prefetch_l2(w[c] + k + u * stride);
  }
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  if (!a.weights_early) load_weights(k);
  while (true) {
    // Registers of a step that is done are filled with the next one's codes at once.
    const int next = k + U * stride;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int ku = k + u * stride;
      uint4 x[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m)
        x[m] = ku < a.K && m < a.M ? piece16(a.A + (long long)m * a.lda, ku, a.K) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint4 v = ww[u][c];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          int s = acc[c][m];
          s = __dp4a(int(v.x), int(x[m].x), s);
          s = __dp4a(int(v.y), int(x[m].y), s);
          s = __dp4a(int(v.z), int(x[m].z), s);
          acc[c][m] = __dp4a(int(v.w), int(x[m].w), s);
        }
        ww[u][c] = next + u * stride < a.K ? piece16(w[c], next + u * stride, a.K) : make_uint4(0, 0, 0, 0);
      }
    }
    if (__all_sync(0xffffffffu, next >= a.K)) break;
    k = next;
  }

#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int s = __reduce_add_sync(0xffffffffu, acc[c][m]);
      if (lane == 0) sums[warp][c * MT + m] = s;
    }
  __syncthreads();
  // One output a thread: the block's groups x C channels x M tokens, channels side by side.
  const int groups = kDotWarps / a.parts;
  for (int i = int(threadIdx.x); i < groups * C * a.M; i += kDotThreads) {
    const int m = i / (groups * C), j = i - m * groups * C;
    const int g = j / C, c = j % C;
    const int n = (int(blockIdx.x) * groups + g) * C + c;
    if (n >= a.N) continue;
    int s = 0;
    for (int p = 0; p < a.parts; ++p) s += sums[g * a.parts + p][c * MT + m];
    const TokenScale sa = token_scale(a.a_scale[m]);
    const float sw = a.w_scale[n];
    const float v = a.bias ? scaled(s, sa, sw, load_as_f32(a.bias, n, a.out)) : scaled(s, sa, sw);
    store_one(a.C, (long long)m * a.ldc + n, v, a.out);
  }
}

}  // namespace aegis::i8
