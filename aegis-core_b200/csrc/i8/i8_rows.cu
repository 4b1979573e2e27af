// The row operations that make 8-bit operands: root-mean-square norm (with the
// residual's addition) and silu(gate) * up, each row quantised with one scale.
//
// Mathematics. With t the row's values before scaling and m = max |t|, the
// code is q = round(127 t / m): the norm's factor 1 / rms is the same for the
// whole row and drops out of q; it enters the scale alone, m / rms / 127. For the
// norm t = h * weight is a product of two 16-bit numbers, exact in float; so q
// is a definite whole number, and both operations give exactly the nearest one
// (of t in 64 bits): the quotient is taken in float, whose error is below
// kBand, and the few elements that come nearer than that to the border between
// two codes are computed again in double. Codes therefore do not depend on a
// row's layout, its neighbours or the number of threads.
//
// Bound: memory. One block holds one row in registers (up to 32 elements a
// thread), reads it once and writes it once; rows beyond 32768 elements take
// two passes, the second one out of L2.
#include <algorithm>

#include "../common.cuh"
#include "../ptx.cuh"
#include "i8.h"

namespace aegis::i8 {
namespace {

enum Mode : int { kNorm = 0, kAddNorm = 1, kSilu = 2 };

struct RowArgs {
  int cols;
  const void* x;  // or gate
  long long ldx;
  const void* r;  // residual, or up
  long long ldr;
  const void* w;
  float eps;
  void* h;
  long long ldh;
  int8_t* q;
  long long ldq;
  float* scale;
  int vec;    // every 16-bit row and the weight start on 16-byte boundaries
  int vec_q;  // every row of q starts on an 8-byte boundary
};

// |127 t / m| in float is off by less than this. Norm: t and m are exact, the
// factor 127 / m and the product round once each: 127 * 2 * 2^-24 = 1.5e-5.
// Silu: t and m carry the errors of expf (2 ulp), the sum, the quotient and
// the product, below 5 * 2^-24 * 1.5 each: 127 * 17 * 2^-24 = 1.3e-4.
template <int MODE>
constexpr float kBand = MODE == kSilu ? 2.5e-4f : 3e-5f;
// How far below the float maximum the true one can lie, relative: both carry the error above.
constexpr float kNearMax = 1.f - 4e-6f;
// Row maxima below this leave float's range of full precision: the row is done in double.
constexpr float kTiny = 1e-30f;

// 8 elements from column c on (those beyond cols: 0).
template <class T>
__device__ __forceinline__ uint4 load8(const T* row, int c, int cols, bool vec) {
  if (vec && c + 8 <= cols) return *reinterpret_cast<const uint4*>(row + c);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < cols) v[i >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(row)[c + i]) << (16 * (i & 1));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
template <class T>
__device__ __forceinline__ void store8(T* row, int c, int cols, bool vec, uint4 v) {
  if (vec && c + 8 <= cols) {
    *reinterpret_cast<uint4*>(row + c) = v;
    return;
  }
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < cols) reinterpret_cast<uint16_t*>(row)[c + i] = uint16_t(u[i >> 1] >> (16 * (i & 1)));
}
template <class T>
__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Elem<T>::pair_to_f32(u[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void store_codes(int8_t* row, int c, int cols, bool vec, const int (&q)[8]) {
  const uint32_t lo = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | uint32_t(q[3] & 255) << 24;
  const uint32_t hi = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | uint32_t(q[7] & 255) << 24;
  if (vec && c + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = int8_t(q[i]);
  }
}

// The rows a block works on, and the row's t in 64 bits from what is in memory.
template <class T, int MODE>
struct Row {
  const T* x;
  const T* r;
  const T* w;
  T* h;
  __device__ Row(const RowArgs& a, long long i)
      : x(static_cast<const T*>(a.x) + i * a.ldx),
        r(MODE == kNorm ? nullptr : static_cast<const T*>(a.r) + i * a.ldr),
        w(static_cast<const T*>(a.w)),
        h(MODE == kAddNorm ? static_cast<T*>(a.h) + i * a.ldh : nullptr) {}
  // h may be x or residual itself: after this thread has stored its h, only h is read.
  __device__ double norm_input(int c) const { return double(Elem<T>::to_f32(MODE == kAddNorm ? h[c] : x[c])); }
  __device__ double t64(int c) const {
    if constexpr (MODE == kSilu) {
      const double g = double(Elem<T>::to_f32(x[c])), u = double(Elem<T>::to_f32(r[c]));
      if (g == 0.0 || u == 0.0) return 0.0;
      return g / (1.0 + exp(-g)) * u;
    } else {
      return norm_input(c) * double(Elem<T>::to_f32(w[c]));
    }
  }
};

template <class T, int MODE>
__device__ __forceinline__ void eval8(const RowArgs& a, const Row<T, MODE>& row, int c, float (&t)[8], float& ss) {
  float x[8], y[8];
  unpack8<T>(load8(row.x, c, a.cols, a.vec), x);
  if constexpr (MODE == kSilu) {
    unpack8<T>(load8(row.r, c, a.cols, a.vec), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = x[i] / (1.f + expf(-x[i])) * y[i];
    // expf(-x) overflows below -88: the quotient is then -0, as it should be
    // in float (kTiny covers rows where that is all there is).
  } else {
    if constexpr (MODE == kAddNorm) {
      unpack8<T>(load8(row.r, c, a.cols, a.vec), y);
      uint4 hv;
      hv.x = Elem<T>::pack(x[0] + y[0], x[1] + y[1]);
      hv.y = Elem<T>::pack(x[2] + y[2], x[3] + y[3]);
      hv.z = Elem<T>::pack(x[4] + y[4], x[5] + y[5]);
      hv.w = Elem<T>::pack(x[6] + y[6], x[7] + y[7]);
      store8(row.h, c, a.cols, a.vec, hv);
      unpack8<T>(hv, x);
    }
    unpack8<T>(load8(row.w, c, a.cols, a.vec), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = x[i] * y[i];
      ss = fmaf(x[i], x[i], ss);
    }
  }
}

// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }

// Every thread of the block gets the block's results; `buf` may be used again after the next barrier.
template <int THREADS>
__device__ __forceinline__ float2 block_max_sum(float m, float s, float2* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  constexpr int W = THREADS / 32;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  float2 v = buf[0];
#pragma unroll
  for (int i = 1; i < W; ++i) {
    v.x = max_nan(v.x, buf[i].x);
    v.y += buf[i].y;
  }
  return v;
}
template <int THREADS>
__device__ __forceinline__ double block_reduce64(double v, bool sum, double* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double u = __shfl_xor_sync(0xffffffffu, v, o);
    v = sum ? v + u : fmax(v, u);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < THREADS / 32; ++i) v = sum ? v + buf[i] : fmax(v, buf[i]);
  return v;
}

// VPT pieces of 8 elements a thread in registers; VPT = 0: rows of any length, two passes.
template <class T, int MODE, int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS) i8_row_kernel(const __grid_constant__ RowArgs a) {
  __shared__ float2 buf[THREADS / 32];
  __shared__ double buf64[THREADS / 32];
  // Programmatic dependent launch: nothing is read before the grids this one
  // depends on have completed. The kernels after this one may start once every
  // block has come this far, so what came before it has completed for them too.
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const Row<T, MODE> row(a, blockIdx.x);
  int8_t* q = a.q + (long long)blockIdx.x * a.ldq;
  float t[VPT ? VPT : 1][8];
  float m = 0.f, ss = 0.f;
  if constexpr (VPT > 0) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * THREADS + int(threadIdx.x)) * 8;
      if (c < a.cols) {
        eval8<T, MODE>(a, row, c, t[v], ss);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max_nan(fabsf(t[v][i]), m);
      }
    }
  } else {
    for (int c = int(threadIdx.x) * 8; c < a.cols; c += THREADS * 8) {
      eval8<T, MODE>(a, row, c, t[0], ss);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(fabsf(t[0][i]), m);
    }
  }
  const float2 red = block_max_sum<THREADS>(m, ss, buf);
  m = red.x;
  ss = red.y;

  // Not finite: codes 0, scale NaN. (A finite t from an h that is not: inf * 0 is NaN, so t shows it.)
  if (!(m <= 3.4028235e38f)) {
    const int zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int c = int(threadIdx.x) * 8; c < a.cols; c += THREADS * 8) store_codes(q, c, a.cols, a.vec_q, zero);
    if (threadIdx.x == 0) a.scale[blockIdx.x] = __int_as_float(0x7fc00000);
    return;
  }
  // The row's maximum in 64 bits: that of the elements which can be it.
  const bool slow = m < kTiny;  // every element in double
  double m64 = double(m);
  if (MODE == kSilu || slow) {
    double mine = 0.0;
    if (slow) {
      for (int c = int(threadIdx.x) * 8; c < a.cols; c += THREADS * 8)
        for (int i = 0; i < 8 && c + i < a.cols; ++i) mine = fmax(mine, fabs(row.t64(c + i)));
    } else {
      const float near = m * kNearMax;
#pragma unroll(VPT ? VPT : 1)
      for (int v = 0; v < (VPT ? VPT : 1 << 30); ++v) {
        const int c = (v * THREADS + int(threadIdx.x)) * 8;
        if (c >= a.cols) break;
        float tt[8], unused = 0.f;
        if constexpr (VPT == 0) eval8<T, MODE>(a, row, c, tt, unused);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (fabsf(VPT ? t[VPT ? v : 0][i] : tt[i]) >= near && c + i < a.cols) mine = fmax(mine, fabs(row.t64(c + i)));
      }
    }
    m64 = block_reduce64<THREADS>(mine, false, buf64);
  }
  if constexpr (MODE == kSilu) {
    if (threadIdx.x == 0) a.scale[blockIdx.x] = float(m64 / 127.0);
  } else {
    // Squares that left float's range are summed again in double.
    double sum = double(ss);
    if (!(ss < 1e37f) || ss < 1e-25f) {
      double s64 = 0.0;
      for (int c = int(threadIdx.x) * 8; c < a.cols; c += THREADS * 8)
        for (int i = 0; i < 8 && c + i < a.cols; ++i) s64 += row.norm_input(c + i) * row.norm_input(c + i);
      sum = block_reduce64<THREADS>(s64, true, buf64);
    }
    if (threadIdx.x == 0)
      a.scale[blockIdx.x] = m64 > 0.0 ? float(m64 / (127.0 * sqrt(sum / a.cols + double(a.eps)))) : 0.f;
  }

  const float inv = slow ? 0.f : 127.f / float(m64);
#pragma unroll(VPT ? VPT : 1)
  for (int v = 0; v < (VPT ? VPT : 1 << 30); ++v) {
    const int c = (v * THREADS + int(threadIdx.x)) * 8;
    if (c >= a.cols) break;
    float tt[8], unused = 0.f;
    if constexpr (VPT == 0) {
      if constexpr (MODE == kAddNorm) {  // h is stored: the sum must not be taken again
#pragma unroll
        for (int i = 0; i < 8; ++i) tt[i] = c + i < a.cols ? float(row.t64(c + i)) : 0.f;
      } else {
        eval8<T, MODE>(a, row, c, tt, unused);
      }
    }
    int code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float z = (VPT ? t[VPT ? v : 0][i] : tt[i]) * inv;
      const float n = rintf(z);
      code[i] = int(n);
      if (slow || fabsf(fabsf(z - n) - 0.5f) < kBand<MODE>)
        code[i] = c + i < a.cols && m64 > 0.0 ? int(rint(127.0 * row.t64(c + i) / m64)) : 0;
    }
    store_codes(q, c, a.cols, a.vec_q, code);
  }
}

template <class T, int MODE, int THREADS, int VPT>
cudaError_t launch(const RowArgs& a, int rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, &i8_row_kernel<T, MODE, THREADS, VPT>, a);
}

template <class T, int MODE>
cudaError_t run(const RowArgs& a, int rows, cudaStream_t s) {
  const int c = a.cols;
  if (c <= 1024) return launch<T, MODE, 128, 1>(a, rows, s);
  if (c <= 2048) return launch<T, MODE, 256, 1>(a, rows, s);
  if (c <= 4096) return launch<T, MODE, 256, 2>(a, rows, s);
  if (c <= 8192) return launch<T, MODE, 512, 2>(a, rows, s);
  if (c <= 16384) return launch<T, MODE, 512, 4>(a, rows, s);
  if (c <= 32768) return launch<T, MODE, 1024, 4>(a, rows, s);
  return launch<T, MODE, 1024, 0>(a, rows, s);
}

bool aligned16(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

RowArgs make_args(const RowOp& o) {
  RowArgs a{};
  a.cols = o.cols;
  a.x = o.x;
  a.ldx = o.ldx;
  a.r = o.residual;
  a.ldr = o.ldr;
  a.w = o.weight;
  a.eps = o.eps;
  a.h = o.h;
  a.ldh = o.ldh;
  a.q = static_cast<int8_t*>(o.q);
  a.ldq = o.ldq;
  a.scale = o.scale;
  a.vec = aligned16(o.x, o.ldx) && (!o.residual || aligned16(o.residual, o.ldr)) &&
          (!o.weight || aligned16(o.weight, 8)) && (!o.h || aligned16(o.h, o.ldh));
  a.vec_q = (reinterpret_cast<uintptr_t>(o.q) & 7u) == 0 && o.ldq % 8 == 0;
  return a;
}

}  // namespace

cudaError_t rmsnorm(const RowOp& o, cudaStream_t s) {
  if (o.rows == 0) return cudaSuccess;
  const RowArgs a = make_args(o);
  if (o.residual)
    return o.bf16 ? run<__nv_bfloat16, kAddNorm>(a, o.rows, s) : run<__half, kAddNorm>(a, o.rows, s);
  return o.bf16 ? run<__nv_bfloat16, kNorm>(a, o.rows, s) : run<__half, kNorm>(a, o.rows, s);
}

cudaError_t silu_mul(const RowOp& o, cudaStream_t s) {
  if (o.rows == 0) return cudaSuccess;
  const RowArgs a = make_args(o);
  return o.bf16 ? run<__nv_bfloat16, kSilu>(a, o.rows, s) : run<__half, kSilu>(a, o.rows, s);
}

}  // namespace aegis::i8
