// The row operations that make 8-bit operands: root-mean-square norm (with the
// residual's addition) and silu(gate) * up, each row quantised with one scale.
//
// Mathematics. With t the row's values before scaling and m = max |t|, the
// code is q = round(127 t / m): the norm's factor 1 / rms is the same for the
// whole row and drops out of q; it enters the scale alone, m / rms / 127. For the
// norm t = h * weight is a product of two 16-bit numbers, exact in float; so q
// is a definite whole number, and both operations give exactly the nearest one
// (of t in 64 bits): z = 127 t / m is taken in float, with a bound on its error,
// and the few elements that come nearer than that to the border between two
// codes are computed again in double. Codes therefore do not depend on a row's
// layout, its neighbours or the number of threads.
//
// Bound: memory, and instruction issue not far behind: 24 instructions an element and
// 64% of the issue slots for the norm with its residual, 19 and 62% without, 20 and 60%
// for silu, whose exponential and reciprocal take half of their unit's time too. The blocks that fit the GPU walk the rows, a thread
// with up to 32 elements, so what a row costs besides its elements (reduction,
// barrier) is spread over many. A thread copies its elements of the next row to
// shared memory while it works on this one, and reads them itself, so the copies
// need no barrier and no row's loads wait for the reduction of the one before. t
// stays in registers between the maximum and the codes. One barrier a row: silu's
// elements at a border need the maximum in 64 bits, which its holder works out
// meanwhile; they are set right after the next row's barrier. Few rows take more threads
// with fewer elements each, for latency. Rows beyond 32768 elements, and rows
// that do not start on 16-byte boundaries, are read directly.
//
// The norm's squares are summed in 64 bits and its scale is rounded once, as silu's is:
// a scale off by its last bit moves results of the product that takes it. Against
// sums in float, the plain norm of 8192 x 4096 takes 24.4 us instead of 22.1 (a
// conversion and a 64-bit operation an element), everything else within 4%.
//
// B200, cold L2: norm with the residual 8192 x 4096 42.7 us (5.5 TB/s of the bytes it
// must move), without 24.4 (4.1); silu 4096 x 14336 55.7 (5.3), 8192 x 4864 42.5
// (4.7), 16384 x 1024 20.8 (4.0: a row's fixed costs); a row of 4096 2.1.
#include <algorithm>

#include "../common.cuh"
#include "../gpu_target.h"
#include "../ptx.cuh"
#include "i8.h"

namespace aegis::i8 {
namespace {

enum Mode : int { kNorm = 0, kAddNorm = 1, kSilu = 2 };

struct RowArgs {
  int rows, cols;
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
  double per_col;  // 1 / cols
  int vec;    // every 16-bit row and the weight start on 16-byte boundaries
  int vec_q;  // every row of q starts on an 8-byte boundary
};

// The error of z = t * (127 / m) in float, relative, with u = 2^-24.
// Norm: t and m are exact; the factor and the product round once each: 2 u.
// Silu, t = (x y) / (1 + e) with e = 2^(-x log2 e): x y is exact (two 16-bit factors);
// the power's argument is off by 1.25 u |x| log2 e, the power by that and by 4 u; the
// sum u, the reciprocal 2 u, the product u; then the factor (m and the quotient
// rounded) 2 u and the last product u: (1.25 |x| + 11) u, the first part for negative
// x alone. An x y above float's range makes the maximum infinite, one below it is off
// by less than 2^-149, both fine (kTiny).
// The factor may come from the float maximum, off by (1.25 |x| + 8) u itself.
constexpr float kBorderNorm = 1.5e-7f;
__device__ __forceinline__ float border_silu(float gate) { return fmaf(gate, 1.6e-7f, 1.4e-6f); }
// How far below the float maximum the true one can lie, relative.
__device__ __forceinline__ float near_max(float gate) { return 1.f - fmaf(gate, 1.5e-7f, 1.25e-6f); }
// What that error bound needs: e far from overflow. Rows with gates below -kMostGate are done in double.
constexpr float kMostGate = 80.f;
// Rows whose largest magnitude is below this are done in double: float's range ends near.
constexpr float kTiny = 1e-20f;
constexpr double kMost = 3.4028234663852886e38;  // the largest float
// Adding it takes a float below 2^22 to the nearest whole number (ties to
// even) and leaves that number's two's complement in the low bits, without
// the conversion unit, which the exponential and the reciprocal need.
constexpr float kRound = 12582912.f;  // 1.5 * 2^23
constexpr float kNearBorder = 0.4999999f;

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
// Two floats in a register pair: sm_100 adds, multiplies and fuses both at once.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 both(f32x2 v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// The largest magnitude of three, a NaN if one is.
__device__ __forceinline__ float max_abs_nan(float a, float2 b) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b.x), "f"(b.y));
  return d;
}
template <class T>
__device__ __forceinline__ f32x2 widen(uint32_t v) {
  const float2 f = Elem<T>::pair_to_f32(v);
  return pair(f.x, f.y);
}
template <class T>
__device__ __forceinline__ uint32_t narrow(f32x2 v) {
  const float2 f = both(v);
  return Elem<T>::pack(f.x, f.y);
}
// 8 codes to columns c.. of a row.
__device__ __forceinline__ void store_codes(int8_t* row, int c, int cols, bool vec, uint2 q) {
  if (vec && c + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = int8_t((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
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
      if ((g == 0.0 && fabs(u) <= kMost) || (u == 0.0 && fabs(g) <= kMost)) return 0.0;  // 0 times infinity is NaN
      return g / (1.0 + exp(-g)) * u;
    } else {
      return norm_input(c) * double(Elem<T>::to_f32(w[c]));
    }
  }
};

// 2^x, off by at most 2^-22, relative.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / x, off by at most 2^-23, for x from 1 to 2^126.
__device__ __forceinline__ float fast_reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x * sigmoid(x) * y.
__device__ __forceinline__ f32x2 silu_mul(f32x2 x, f32x2 y) {
  const float2 p = both(mul2(x, pair(-1.44269504f, -1.44269504f)));
  const float2 d = both(add2(pair(fast_exp2(p.x), fast_exp2(p.y)), pair(1.f, 1.f)));
  return mul2(mul2(x, y), pair(fast_reciprocal(d.x), fast_reciprocal(d.y)));
}

template <class T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };

// What a thread gathers of its elements in a row.
template <class T>
struct Stats {
  using P = typename Pair<T>::type;
  float m = 0.f;   // max |t|
  double ss = 0.0; // squares (norm): exact products, summed in 64 bits so that the scale rounds once
  uint32_t low = 0;  // least gate, two at a time (silu)
  __device__ void least_gate(uint32_t g) {
    const P l = __hmin2(reinterpret_cast<const P&>(low), reinterpret_cast<const P&>(g));
    low = reinterpret_cast<const uint32_t&>(l);
  }
  __device__ float gate() const {  // magnitude of the least gate below 0
    const float2 f = Elem<T>::pair_to_f32(low);
    return -fminf(f.x, f.y);
  }
};

// t of 8 elements, given the packed inputs; returns what is normalised (h, or x).
template <class T, int MODE>
__device__ __forceinline__ uint4 eval8(uint4 xv, uint4 yv, uint4 wv, f32x2 (&t)[4], Stats<T>& st) {
  uint32_t x[4] = {xv.x, xv.y, xv.z, xv.w};
  const uint32_t y[4] = {yv.x, yv.y, yv.z, yv.w}, w[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (MODE == kAddNorm) x[i] = narrow<T>(add2(widen<T>(x[i]), widen<T>(y[i])));
    const f32x2 f = widen<T>(x[i]);
    if constexpr (MODE == kSilu) {
      t[i] = silu_mul(f, widen<T>(y[i]));
      st.least_gate(x[i]);
    } else {
      t[i] = mul2(f, widen<T>(w[i]));
      const float2 v = both(f);
      st.ss = fma(double(v.x), double(v.x), st.ss);
      st.ss = fma(double(v.y), double(v.y), st.ss);
    }
    st.m = max_abs_nan(st.m, both(t[i]));
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}
// The same from memory, columns c.. of a row; stores h.
template <class T, int MODE>
__device__ __forceinline__ void load_eval8(const RowArgs& a, const Row<T, MODE>& row, int c, f32x2 (&t)[4],
                                           Stats<T>& st) {
  const uint4 none = make_uint4(0, 0, 0, 0);
  const uint4 h = eval8<T, MODE>(load8(row.x, c, a.cols, a.vec),
                                 MODE == kNorm ? none : load8(row.r, c, a.cols, a.vec),
                                 MODE == kSilu ? none : load8(row.w, c, a.cols, a.vec), t, st);
  if constexpr (MODE == kAddNorm) store8(row.h, c, a.cols, a.vec, h);
}

// A block's results: max |t|, the magnitude of the least gate. Magnitudes are
// compared as the bits of floats without a sign, where a NaN is above infinity.
// The squares' sum is kept by warp: only the scale needs it (norm_scale).
struct Found {
  float m, gate;
  double ss;
};
__device__ __forceinline__ float max_bits(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int MODE>
__device__ __forceinline__ Found block_find(float m, double ss, float gate, int* any, Found* buf) {
  const int W = int(blockDim.x) / 32;
  const int lane = int(threadIdx.x & 31);
  Found f;
  f.m = max_bits(fabsf(m));
  f.gate = MODE == kSilu ? max_bits(fabsf(gate)) : 0.f;
  f.ss = MODE != kSilu ? warp_sum(ss) : 0.0;
  if (lane == 0) buf[threadIdx.x >> 5] = f;
  if (MODE == kSilu) *any = __syncthreads_or(*any);
  else __syncthreads();
  if (W > 1) {
    f.m = max_bits(lane < W ? buf[lane].m : 0.f);
    if (MODE == kSilu) f.gate = max_bits(lane < W ? buf[lane].gate : 0.f);
  }
  return f;
}
// max that keeps a NaN.
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }

// The block's sum or maximum in double. Out of line: rare rows only.
__device__ __noinline__ double block_reduce64(double v, bool sum, double* buf) {
  for (int o = 16; o > 0; o >>= 1) {
    const double u = __shfl_xor_sync(0xffffffffu, v, o);
    v = sum ? v + u : max_nan(v, u);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int i = 1; i < int(blockDim.x) / 32; ++i) v = sum ? v + buf[i] : max_nan(v, buf[i]);
  return v;
}

// The code of column c in 64 bits.
template <class T, int MODE>
__device__ __forceinline__ int code64(const Row<T, MODE>& row, int c, double m64) {
  return int(rint(127.0 * row.t64(c) / m64));
}
template <class T, int MODE>
__device__ __forceinline__ double abs_t64(const Row<T, MODE>& row, int c) {
  return fabs(row.t64(c));
}

// A whole row in double: rows of zeros, rows that are not finite, and those for
// which float's range or precision does not do. Each thread reads the columns whose h
// it stored itself. Out of line, and called where nothing else is alive.
template <class T, int MODE>
__device__ __noinline__ void row_in_double(const RowArgs& a, int ri, double* buf) {
  const Row<T, MODE> row(a, ri);
  int8_t* q = a.q + (long long)ri * a.ldq;
  const int cols = a.cols, step = int(blockDim.x) * 8;
  double m = 0.0, s = 0.0;
  for (int c0 = int(threadIdx.x) * 8; c0 < cols; c0 += step)
    for (int c = c0; c < min(c0 + 8, cols); ++c) {
      m = max_nan(fabs(row.t64(c)), m);
      if (MODE != kSilu) s += row.norm_input(c) * row.norm_input(c);
    }
  m = block_reduce64(m, false, buf);
  if (MODE != kSilu) s = block_reduce64(s, true, buf);
  // t is finite in 32 bits, and so is h (an infinite h gives an infinite t, or NaN where the weight is 0).
  const bool fine = m <= kMost;
  for (int c0 = int(threadIdx.x) * 8; c0 < cols; c0 += step)
    for (int c = c0; c < min(c0 + 8, cols); ++c)
      q[c] = fine && m > 0.0 ? int8_t(code64<T, MODE>(row, c, m)) : int8_t(0);
  if (threadIdx.x == 0) {
    float scale = float(m / 127.0);
    if (MODE != kSilu) scale = m > 0.0 ? float(m / (127.0 * sqrt(s / cols + double(a.eps)))) : 0.f;
    a.scale[ri] = fine ? scale : __int_as_float(0x7fc00000);
  }
}

__device__ __forceinline__ float at(const f32x2 (&t)[4], int i) {
  const float2 f = both(t[i >> 1]);
  return i & 1 ? f.y : f.x;
}

// 8 codes n from t. An element nearer to a border than z's error, border |z|, has
// to be taken again: with d the distance from z to n, d > 1/2 - border (|n| + 1/2).
// `most`, the largest d, is a first test: above first_test(border), where |n| is taken
// as 127, there may be one among the 8. A test with n^2 in it (three more paired
// products an element pair) passed fewer pieces and cost more.
__device__ __forceinline__ uint2 quantise8(const f32x2 (&t)[4], float inv, float& most) {
  uint32_t code[8];
  most = 0.f;
  const f32x2 inv2 = pair(inv, inv), up = pair(kRound, kRound);
  const f32x2 minus = pair(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 r = fma2(t[i], inv2, up), n = fma2(r, minus, up);  // -n
    most = max_abs_nan(most, both(fma2(t[i], inv2, n)));
    const float2 f = both(r);
    code[2 * i] = __float_as_uint(f.x);
    code[2 * i + 1] = __float_as_uint(f.y);
  }
  const uint32_t a = __byte_perm(code[0], code[1], 0x0040), b = __byte_perm(code[2], code[3], 0x0040);
  const uint32_t d = __byte_perm(code[4], code[5], 0x0040), e = __byte_perm(code[6], code[7], 0x0040);
  return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(d, e, 0x5410));
}
__device__ __forceinline__ float first_test(float border) { return kNearBorder - 127.5f * border; }
// A bit for each of the 8 elements that is nearer to a border than that.
__device__ __forceinline__ uint32_t near_border(const f32x2 (&t)[4], float inv, float border) {
  uint32_t near = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = __fsub_rn(fmaf(at(t, i), inv, kRound), kRound);
    near |= fmaf(fabsf(n) + 0.5f, border, fabsf(fmaf(at(t, i), inv, -n))) > kNearBorder ? 1u << i : 0u;
  }
  return near;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Whether a row has to be taken in double: `gates` (silu, any thread's), a largest
// magnitude that is tiny or not finite.
template <int MODE>
__device__ __forceinline__ bool needs_double(const Found& f, int gates) {
  return !(f.m >= kTiny && f.m <= 3.4028235e38f) || (MODE == kSilu && gates);
}

// The norm's scale, m / sqrt(mean h^2 + eps) / 127, in 64 bits and rounded once: the
// first warp joins the warps' sums that block_find left in buf and stores it. After
// the codes, since nothing else of the row waits for it.
__device__ __forceinline__ void norm_scale(const RowArgs& a, int ri, float m, const Found* buf) {
  if (threadIdx.x >= 32) return;
  const int W = int(blockDim.x) / 32, lane = int(threadIdx.x);
  const double ss = warp_sum(lane < W ? buf[lane].ss : 0.0);
  if (lane == 0) a.scale[ri] = float(double(m) * (1.0 / 127.0) * rsqrt(fma(ss, a.per_col, double(a.eps))));
}

// What a silu row leaves to do until the next row's barrier.
template <class T>
struct Behind {
  const RowArgs& a;
  unsigned long long* top64;  // row maxima in 64 bits, of three rows in turn: the bits
                              // of a double that is not negative order as it does
  uint32_t border_bits = 0;   // elements of row `row` at a border
  int row = -1;
  unsigned slot = 0;          // its place in top64
  unsigned turn = 0;          // the present row's: 0, 1, 2, 0, ...

  __device__ int column(int i) const {  // of the thread's i-th element
    return ((i >> 3) * int(blockDim.x) + int(threadIdx.x)) * 8 + (i & 7);
  }
  // After the present row's barrier: the next row's slot (its last readers are past the barrier).
  __device__ void begin() {
    if (threadIdx.x == 0) top64[turn == 2 ? 0 : turn + 1] = 0;
  }
  // Element i of this thread can be row ri's maximum.
  __device__ void candidate(int ri, int i) const {
    const double d = abs_t64<T, kSilu>(Row<T, kSilu>(a, ri), column(i));
    atomicMax(&top64[turn], (unsigned long long)__double_as_longlong(d));
  }
  // Between the barriers of the next row and the one after it (or behind a barrier
  // of its own). Where this is called, t is no longer needed: kept over what is in
  // here it cost a third of the registers.
  __device__ void settle() {
    if (row < 0) return;
    const double top = __longlong_as_double((long long)top64[slot]);
    if (threadIdx.x == 0) a.scale[row] = float(top / 127.0);
    if (border_bits) {
      const Row<T, kSilu> r(a, row);
      for (; border_bits; border_bits &= border_bits - 1) {
        const int c = column(__ffs(int(border_bits)) - 1);
        if (c < a.cols) a.q[(long long)row * a.ldq + c] = int8_t(code64<T, kSilu>(r, c, top));
      }
    }
    row = -1;
  }
  // The end of row ri: settles the row before, and leaves `bits` of this one for later (done: nothing).
  __device__ void end(int ri, uint32_t bits, bool done) {
    settle();
    if (!done) {
      border_bits = bits;
      row = ri;
      slot = turn;
    }
    turn = turn == 2 ? 0 : turn + 1;
  }
};

// Elements of a norm row at a border, a bit each of this thread's.
template <class T, int MODE>
__device__ __forceinline__ void set_codes(const RowArgs& a, int ri, uint32_t bits, float m) {
  const Row<T, MODE> row(a, ri);
  for (; bits; bits &= bits - 1) {
    const int i = __ffs(int(bits)) - 1;
    const int c = ((i >> 3) * int(blockDim.x) + int(threadIdx.x)) * 8 + (i & 7);
    if (c < a.cols) a.q[(long long)ri * a.ldq + c] = int8_t(code64<T, MODE>(row, c, double(m)));
  }
}

constexpr unsigned kLater = 0x7fc00001;  // a NaN no kernel gives: marks the scale of a row that is still to be done

// Many rows. Blocks of as many threads as a row of 32 elements a thread takes;
// every row starts on a 16-byte boundary (q's on 8) and has whole pieces.
constexpr int kPieces = 4;
template <class T, int MODE, int MOST, int BLOCKS>
__global__ void __launch_bounds__(MOST, BLOCKS) i8_rows_kernel(const __grid_constant__ RowArgs a) {
  extern __shared__ uint4 ahead[];  // the next row: [piece][source][thread]
  __shared__ Found buf[2][32];
  __shared__ double buf64[32];
  __shared__ unsigned long long top64[3];
  constexpr int kSources = MODE == kNorm ? 1 : 2;
  const int tid = int(threadIdx.x), step = int(blockDim.x) * 8, c0 = tid * 8;
  if (tid < 3) top64[tid] = 0;
  // Programmatic dependent launch: nothing is read before the grids this one
  // depends on have completed. The kernels after this one may start once every
  // block has come this far, so what came before it has completed for them too.
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();

  const int pieces = c0 < a.cols ? min(kPieces, (a.cols - 1 - c0) / step + 1) : 0;
  const int rows_ahead = int(gridDim.x);
  const T* x = static_cast<const T*>(a.x) + (long long)blockIdx.x * a.ldx + c0;
  const T* r = MODE == kNorm ? nullptr : static_cast<const T*>(a.r) + (long long)blockIdx.x * a.ldr + c0;
  const T* w = MODE == kSilu ? nullptr : static_cast<const T*>(a.w) + (pieces ? c0 : 0);
  T* h = MODE == kAddNorm ? static_cast<T*>(a.h) + (long long)blockIdx.x * a.ldh + c0 : nullptr;
  int8_t* q = a.q + (long long)blockIdx.x * a.ldq + c0;
  const uint32_t mine = ptx::smem_addr(ahead) + uint32_t(tid) * 16u, source = blockDim.x * 16u;
  auto copy_piece = [&](int v) {
    copy16(mine + uint32_t(v * kSources) * source, x + v * step);
    if (MODE != kNorm) copy16(mine + uint32_t(v * kSources + 1) * source, r + v * step);
  };
  // Pieces beyond the row's end are zeros throughout: they change no maximum or sum,
  // so only copies and stores ask for them (branches around the rest cost a tenth).
#pragma unroll
  for (int v = 0; v < kPieces; ++v) {
    if (v < pieces) {
      copy_piece(v);
    } else {
      for (int i = 0; i < kSources; ++i) ahead[(v * kSources + i) * int(blockDim.x) + tid] = make_uint4(0, 0, 0, 0);
    }
  }
  copy_commit();

  Behind<T> behind{a, top64};
  bool later = false;
  unsigned par = 0;
  for (int ri = int(blockIdx.x);; par ^= 1u) {
    const bool more = a.rows - ri > rows_ahead;
    x += (long long)rows_ahead * a.ldx;
    if (MODE != kNorm) r += (long long)rows_ahead * a.ldr;
    f32x2 t[kPieces][4];
    Stats<T> st;
    copy_wait<0>();
#pragma unroll
    for (int v = 0; v < kPieces; ++v) {
      const uint4 xv = ptx::ld_shared_v4(mine + uint32_t(v * kSources) * source);
      const uint4 yv = MODE == kNorm ? xv : ptx::ld_shared_v4(mine + uint32_t(v * kSources + 1) * source);
      const uint4 hv = eval8<T, MODE>(
          xv, yv, MODE == kSilu ? xv : *reinterpret_cast<const uint4*>(v < pieces ? w + v * step : w), t[v], st);
      if (MODE == kAddNorm && v < pieces) *reinterpret_cast<uint4*>(h + v * step) = hv;
      if (more && v < pieces) copy_piece(v);
    }
    copy_commit();
    const int in_double = MODE == kSilu && st.gate() > kMostGate;
    int any = in_double;
    const Found f = block_find<MODE>(st.m, st.ss, st.gate(), &any, buf[par]);
    if (MODE == kSilu) behind.begin();
    const bool done = needs_double<MODE>(f, any);
    uint32_t near = 0, can = 0;
    if (done) {
      later = true;
      if (tid == 0) a.scale[ri] = __uint_as_float(kLater);
    } else {
      const float inv = 127.f / f.m;
      const float border = MODE == kSilu ? border_silu(f.gate) : kBorderNorm;
      float most[kPieces];
#pragma unroll
      for (int v = 0; v < kPieces; ++v) {
        const uint2 codes = quantise8(t[v], inv, most[v]);
        if (v < pieces) *reinterpret_cast<uint2*>(q + v * step) = codes;
      }
#pragma unroll
      for (int v = 0; v < kPieces; ++v)
        if (most[v] > first_test(border)) near |= near_border(t[v], inv, border) << (8 * v);
      // The maximum in 64 bits is that of the elements which can be it.
      const float least = f.m * near_max(f.gate);
      if (MODE == kSilu && st.m >= least) {
#pragma unroll
        for (int v = 0; v < kPieces; ++v)
#pragma unroll
          for (int i = 0; i < 8; ++i) can |= fabsf(at(t[v], i)) >= least ? 1u << (8 * v + i) : 0u;
      }
      if (MODE != kSilu) norm_scale(a, ri, f.m, buf[par]);
    }
    if constexpr (MODE == kSilu) {
      for (; can; can &= can - 1) behind.candidate(ri, __ffs(int(can)) - 1);
      behind.end(ri, near, done);
    } else if (near) {
      set_codes<T, MODE>(a, ri, near, f.m);
    }
    if (!more) break;
    ri += rows_ahead;
    q += (long long)rows_ahead * a.ldq;
    if (MODE == kAddNorm) h += (long long)rows_ahead * a.ldh;
  }
  if constexpr (MODE == kSilu) {
    __syncthreads();
    behind.settle();
  }
  if (later) {  // the same for all threads
    __syncthreads();
    for (int ri = int(blockIdx.x);; ri += rows_ahead) {
      if (__float_as_uint(*const_cast<volatile float*>(a.scale + ri)) == kLater) row_in_double<T, MODE>(a, ri, buf64);
      if (a.rows - ri <= rows_ahead) break;
    }
  }
}

// Any rows, one a block: few rows, rows of any alignment, and with VPT = 0 of any
// length (VPT pieces of 8 elements a thread; 0: as many as it takes, read twice).
template <class T, int MODE, int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) i8_row_kernel(const __grid_constant__ RowArgs a) {
  __shared__ Found buf[32];
  __shared__ double buf64[32];
  __shared__ unsigned long long top64[3];
  constexpr int kKept = VPT ? VPT : 1;
  const int tid = int(threadIdx.x), ri = int(blockIdx.x);
  auto piece = [&](int v) { return (v * THREADS + tid) * 8; };
  if (tid < 3) top64[tid] = 0;
  ptx::griddep_wait();  // as above
  ptx::griddep_launch_dependents();
  const Row<T, MODE> row(a, ri);
  int8_t* q = a.q + (long long)ri * a.ldq;
  f32x2 t[kKept][4];
  Stats<T> st;
  if constexpr (VPT > 0) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      if (piece(v) < a.cols) load_eval8<T, MODE>(a, row, piece(v), t[v], st);
  } else {
    for (int v = 0; piece(v) < a.cols; ++v) load_eval8<T, MODE>(a, row, piece(v), t[0], st);
  }
  int any = MODE == kSilu && st.gate() > kMostGate;
  const Found f = block_find<MODE>(st.m, st.ss, st.gate(), &any, buf);
  if (needs_double<MODE>(f, any)) {
    row_in_double<T, MODE>(a, ri, buf64);
    return;
  }
  Behind<T> behind{a, top64};
  const float inv = 127.f / f.m;
  const float border = MODE == kSilu ? border_silu(f.gate) : kBorderNorm;
  const float least = f.m * near_max(f.gate);
  if constexpr (VPT > 0) {
    uint32_t near = 0, can = 0;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
      if (piece(v) < a.cols) {
        float most;
        store_codes(q, piece(v), a.cols, a.vec_q, quantise8(t[v], inv, most));
        if (most > first_test(border)) near |= near_border(t[v], inv, border) << (8 * v);
      }
    if constexpr (MODE == kSilu) {
      if (st.m >= least) {
#pragma unroll
        for (int v = 0; v < VPT; ++v)
          if (piece(v) < a.cols)
#pragma unroll
            for (int i = 0; i < 8; ++i) can |= fabsf(at(t[v], i)) >= least ? 1u << (8 * v + i) : 0u;
        for (; can; can &= can - 1) behind.candidate(ri, __ffs(int(can)) - 1);
      }
      behind.end(ri, near, false);
      __syncthreads();
      behind.settle();
    } else if (near) {
      set_codes<T, MODE>(a, ri, near, f.m);
    }
    if (MODE != kSilu) norm_scale(a, ri, f.m, buf);
  } else {
    double m64 = double(f.m);
    if constexpr (MODE == kSilu) {
      for (int v = 0; piece(v) < a.cols; ++v) {
        Stats<T> unused;
        load_eval8<T, MODE>(a, row, piece(v), t[0], unused);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (fabsf(at(t[0], i)) >= least) behind.candidate(ri, 8 * v + i);
      }
      behind.end(ri, 0, false);
      __syncthreads();
      behind.settle();
      m64 = __longlong_as_double((long long)top64[0]);  // the first row's slot
    }
    for (int v = 0; piece(v) < a.cols; ++v) {
      const int c = piece(v);
      if constexpr (MODE == kAddNorm) {  // h is stored: the sum must not be taken again
#pragma unroll
        for (int i = 0; i < 4; ++i)
          t[0][i] = pair(c + 2 * i < a.cols ? float(row.t64(c + 2 * i)) : 0.f,
                         c + 2 * i + 1 < a.cols ? float(row.t64(c + 2 * i + 1)) : 0.f);
      } else {
        Stats<T> unused;
        load_eval8<T, MODE>(a, row, c, t[0], unused);
      }
      float most;
      store_codes(q, c, a.cols, a.vec_q, quantise8(t[0], inv, most));
      if (most > first_test(border))
        for (uint32_t b = near_border(t[0], inv, border); b; b &= b - 1) {
          const int k = c + __ffs(int(b)) - 1;
          if (k < a.cols) q[k] = int8_t(code64<T, MODE>(row, k, m64));
        }
    }
    if (MODE != kSilu) norm_scale(a, ri, f.m, buf);
  }
}

cudaLaunchConfig_t launch_config(unsigned grid, unsigned block, size_t smem, cudaStream_t s, cudaLaunchAttribute* pdl) {
  pdl->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl->val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  return cfg;
}

template <class T, int MODE, int THREADS, int VPT>
cudaError_t launch_row(const RowArgs& a, cudaStream_t s) {
  cudaLaunchAttribute pdl;
  const cudaLaunchConfig_t cfg = launch_config(unsigned(a.rows), THREADS, 0, s, &pdl);
  return cudaLaunchKernelEx(&cfg, &i8_row_kernel<T, MODE, THREADS, VPT>, a);
}

template <class T, int MODE, int MOST, int BLOCKS>
cudaError_t launch_rows(const RowArgs& a, int threads, int sms, cudaStream_t s) {
  auto* kern = &i8_rows_kernel<T, MODE, MOST, BLOCKS>;
  constexpr int kBytes = kPieces * 16 * (MODE == kNorm ? 1 : 2);  // a thread's share
  static gpu::SmemOptIn optin;
  if (const cudaError_t e = optin.ensure(reinterpret_cast<const void*>(kern), size_t(kBytes) * MOST); e != cudaSuccess)
    return e;
  const int fit = std::min(MOST * BLOCKS / threads, 32);
  cudaLaunchAttribute pdl;
  const cudaLaunchConfig_t cfg = launch_config(unsigned(std::min(a.rows, sms * fit)), unsigned(threads),
                                               size_t(kBytes) * threads, s, &pdl);
  return cudaLaunchKernelEx(&cfg, kern, a);
}
template <class T, int MODE>
cudaError_t launch_rows(const RowArgs& a, int sms, cudaStream_t s) {
  const int threads = ceil_div(a.cols, 32 * 8 * kPieces) * 32;
  // About 900 threads an SM at 72 registers, in blocks that fit the row (silu 16384 x
  // 1024: 31 us with 16 blocks an SM at most, 24 with 28); the plain norm is level to 3%
  // faster with fewer and 80 registers.
  if (threads <= 128) return launch_rows<T, MODE, 128, MODE == kNorm ? 6 : 7>(a, threads, sms, s);
  if (threads <= 224) return launch_rows<T, MODE, 224, 4>(a, threads, sms, s);
  if (threads <= 288) return launch_rows<T, MODE, 288, 3>(a, threads, sms, s);
  if (threads <= 448) return launch_rows<T, MODE, 448, 2>(a, threads, sms, s);
  return launch_rows<T, MODE, 1024, 1>(a, threads, sms, s);
}

template <class T, int MODE>
cudaError_t run(const RowArgs& a, cudaStream_t s) {
  const gpu::Target* d = gpu::this_device();
  if (!d) return cudaErrorInvalidDevice;
  const int c = a.cols;
  if (c > 32768) return launch_row<T, MODE, 1024, 0>(a, s);
  if (a.vec && a.vec_q && c % 8 == 0 && a.rows > 2 * d->sms) return launch_rows<T, MODE>(a, d->sms, s);
  if (c <= 1024) return launch_row<T, MODE, 128, 1>(a, s);
  // Many rows: as many elements a thread as registers hold, for what a row costs besides.
  // B200, us, one piece a thread and this: norm 8192 x 4095 121, 91; silu 2000 x 1501
  // 20.1, 10.4. At 300 rows of 3001, 5.3 and 6.1.
  const bool many = a.rows > 4 * d->sms;
  if (many && c <= 2048) return launch_row<T, MODE, 128, 2>(a, s);
  if (many && c <= 4096) return launch_row<T, MODE, 128, 4>(a, s);
  if (many && c <= 8192) return launch_row<T, MODE, 256, 4>(a, s);
  if (c <= 4096) return launch_row<T, MODE, 512, 1>(a, s);
  // Blocks of 1024 threads take an SM's registers: the fastest for a row or two, but
  // behind a product they wait for SMs to empty, blocks of 512 find room beside its
  // last CTAs. Feed-forward block of 1 and 16 tokens (4096, 14336), us: 37.5, 45.6
  // with 1024 threads, 38.0, 42.5 with 512.
  const bool few = a.rows <= 8;
  if (c <= 8192) return few ? launch_row<T, MODE, 1024, 1>(a, s) : launch_row<T, MODE, 512, 2>(a, s);
  if (c <= 16384) return few ? launch_row<T, MODE, 1024, 2>(a, s) : launch_row<T, MODE, 512, 4>(a, s);
  return launch_row<T, MODE, 1024, 4>(a, s);
}

bool aligned16(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

RowArgs make_args(const RowOp& o) {
  RowArgs a{};
  a.rows = o.rows;
  a.cols = o.cols;
  a.x = o.x;
  a.ldx = o.ldx;
  a.r = o.residual;
  a.ldr = o.ldr;
  a.w = o.weight;
  a.eps = o.eps;
  a.per_col = 1.0 / double(o.cols);
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
    return o.bf16 ? run<__nv_bfloat16, kAddNorm>(a, s) : run<__half, kAddNorm>(a, s);
  return o.bf16 ? run<__nv_bfloat16, kNorm>(a, s) : run<__half, kNorm>(a, s);
}

cudaError_t silu_mul(const RowOp& o, cudaStream_t s) {
  if (o.rows == 0) return cudaSuccess;
  const RowArgs a = make_args(o);
  return o.bf16 ? run<__nv_bfloat16, kSilu>(a, s) : run<__half, kSilu>(a, s);
}

}  // namespace aegis::i8
