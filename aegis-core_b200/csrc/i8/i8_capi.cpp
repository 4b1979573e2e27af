// C ABI of the 8-bit operators (include/aegis_i8.h). Arguments are checked
// before any CUDA call; CUDA and launch errors become status codes, and the
// calling thread's device is put back.
#include "aegis_i8.h"

#include <cuda_runtime.h>

#include <cstdio>
#include <cstring>
#include <string>

#include "../common.cuh"
#include "../status.h"
#include "aegis/gemm.h"
#include "i8.h"

namespace {

using aegis::i8::Gemm;
using aegis::i8::Out;
using aegis::i8::RowOp;

thread_local std::string t_error;

// The text is kept if memory allows; the status is returned either way.
int fail(int status, const char* fn, const char* what) noexcept {
  try {
    t_error = fn;
    t_error += ": ";
    t_error += what;
  } catch (...) {
  }
  return status;
}
int bad(const char* fn, const char* what) noexcept { return fail(AEGIS_ERR_INVALID_ARGUMENT, fn, what); }
int fail_cuda(const char* fn, cudaError_t e, bool launch) noexcept {
  cudaGetLastError();  // clear a non-sticky error so it does not leak into the next call
  return fail(e == cudaErrorMemoryAllocation ? AEGIS_ERR_OUT_OF_MEMORY
              : e == cudaErrorStreamCaptureUnsupported || !launch ? AEGIS_ERR_CUDA
                                                                 : AEGIS_ERR_LAUNCH_FAILED,
              fn, e == cudaErrorNotSupported ? "needs an sm_100 device" : cudaGetErrorString(e));
}

// The calling thread's device for the duration of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    error_ = cudaGetDevice(&was_);
    if (error_ == cudaSuccess && was_ != device) {
      error_ = cudaSetDevice(device);
      moved_ = error_ == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(was_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  cudaError_t error() const { return error_; }

 private:
  int was_ = 0;
  bool moved_ = false;
  cudaError_t error_;
};

template <class F>
int on_device(int device, const char* fn, F&& body, bool launch = true) {
  if (device < 0) return fail(AEGIS_ERR_NO_DEVICE, fn, "no such CUDA device");
  OnDevice scope(device);
  if (scope.error() != cudaSuccess) {
    cudaGetLastError();
    return fail(AEGIS_ERR_NO_DEVICE, fn, "no such CUDA device");
  }
  // The device's status word is made by its first launch, whichever operator's: the next one may be captured.
  unsigned* status = nullptr;
  cudaError_t e = launch ? aegis::status::word(&status) : cudaSuccess;
  if (e == cudaSuccess) e = body();
  return e == cudaSuccess ? AEGIS_OK : fail_cuda(fn, e, launch);
}

bool size_ok(long long n) { return n >= 0 && n <= aegis::gemm::kMaxDim; }
bool dtype16(int t) { return t == AEGIS_DTYPE_F16 || t == AEGIS_DTYPE_BF16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// nullptr, or what is wrong.
const char* check(const Gemm& g, int out_dtype) {
  if (!dtype16(out_dtype) && out_dtype != AEGIS_DTYPE_F32)
    return "out_dtype must be AEGIS_DTYPE_F16, AEGIS_DTYPE_BF16 or AEGIS_DTYPE_F32";
  if (!size_ok(g.M) || !size_ok(g.N) || g.K < 0) return "negative size or a size above 2^31 - 2^20";
  if (g.K > AEGIS_I8_MAX_K) return "K above AEGIS_I8_MAX_K: the int32 sum could overflow";
  if (g.M == 0 || g.N == 0) return nullptr;
  if (g.K > 0 && (!g.A || !g.W)) return "A or W is NULL";
  if (!g.C || !g.a_scale || !g.w_scale) return "C, a_scale or w_scale is NULL";
  if (g.lda < g.K || g.ldw < g.K || g.ldc < g.N) return "a row stride is smaller than the row";
  const size_t es = out_dtype == AEGIS_DTYPE_F32 ? 4 : 2;
  if (!aligned(g.a_scale, 4) || !aligned(g.w_scale, 4) || !aligned(g.C, es) || !aligned(g.bias, es))
    return "a scale, the bias or C is not aligned to its elements";
  return nullptr;
}

const char* check_rows(const RowOp& o, int dtype) {
  if (!dtype16(dtype)) return "dtype must be AEGIS_DTYPE_F16 or AEGIS_DTYPE_BF16";
  if (!size_ok(o.rows) || !size_ok(o.cols)) return "negative size or a size above 2^31 - 2^20";
  if (o.rows == 0) return nullptr;
  if (o.cols == 0) return "rows of no elements have no scale (cols is 0)";
  if (!o.x || !o.q || !o.scale) return "an operand is NULL";
  if (o.ldx < o.cols || o.ldq < o.cols) return "a row stride is smaller than the row";
  if (!aligned(o.x, 2) || !aligned(o.residual, 2) || !aligned(o.weight, 2) || !aligned(o.h, 2) ||
      !aligned(o.scale, 4))
    return "an operand is not aligned to its elements";
  return nullptr;
}

const char* check_norm(const RowOp& o, int dtype) {
  if (const char* w = check_rows(o, dtype)) return w;
  if (!(o.eps >= 0.f) || o.eps > 3.4e38f) return "eps must be a finite number, 0 or more";
  if (o.rows == 0) return nullptr;
  if (!o.weight) return "weight is NULL";
  if (o.residual && (!o.h || o.ldr < o.cols || o.ldh < o.cols))
    return "with a residual, h must be given, and the strides of both be at least cols";
  if (!o.residual && o.h) return "h without a residual (h would be x)";
  if (o.h && ((o.h == o.x && o.ldh != o.ldx) || (o.h == o.residual && o.ldh != o.ldr)))
    return "h in the place of x or residual needs the same row stride";
  return nullptr;
}

size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// The workspace of a feed-forward block.
struct MlpSpace {
  size_t q1, s1, gu, q2, s2, w1, w2, bytes;
  long long ld1, ldgu, ld2;
  bool copy1, copy2;  // the weights' rows need a copy that TMA can address
  MlpSpace(int M, int K, int F, const void* w_gate_up, int64_t ld_gate_up, const void* w_down, int64_t ld_down) {
    ld1 = (long long)up(size_t(K), 16);
    ldgu = (long long)up(2 * size_t(F), 8);
    ld2 = (long long)up(size_t(F), 16);
    if (M == 0) {
      bytes = 0;
      return;
    }
    size_t at = 0;
    auto take = [&](size_t n) {
      const size_t was = at;
      at = up(at + n, 256);
      return was;
    };
    q1 = take(size_t(M) * size_t(ld1));
    s1 = take(size_t(M) * 4);
    gu = take(size_t(M) * size_t(ldgu) * 2);
    q2 = take(size_t(M) * size_t(ld2));
    s2 = take(size_t(M) * 4);
    copy1 = !aegis::i8::tma_rows(w_gate_up, ld_gate_up, 2 * F);
    copy2 = !aegis::i8::tma_rows(w_down, ld_down, K);
    w1 = take(copy1 ? 2 * size_t(F) * aegis::i8::aligned_cols(K) : 0);
    w2 = take(copy2 ? size_t(K) * aegis::i8::aligned_cols(F) : 0);
    bytes = at;
  }
};

const char* check_mlp_sizes(int M, int K, int F) {
  if (!size_ok(M)) return "negative size or a size above 2^31 - 2^20";
  if (K < 1 || K > AEGIS_I8_MAX_K || F < 1 || F > AEGIS_I8_MAX_K) return "K and F must be from 1 to AEGIS_I8_MAX_K";
  return nullptr;
}

}  // namespace

extern "C" {

const char* aegis_i8_last_error_string(void) { return t_error.c_str(); }

int aegis_i8_synchronize(int device, void* stream) {
  const char* fn = "aegis_i8_synchronize";
  unsigned bits = 0, block = 0;
  const int s = on_device(device, fn, [&] {
    if (const cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream)); e != cudaSuccess) return e;
    return aegis::status::take(&bits, &block);
  }, false);
  if (s != AEGIS_OK) return s;
  if (bits == 0) return AEGIS_OK;
  char b[160];
  std::snprintf(b, sizeof b,
                "kernel watchdog fired (status bits 0x%x, first block %u): a bounded wait ran out; that launch's "
                "output is not valid",
                bits, block ? block - 1 : 0);
  return fail(AEGIS_ERR_CUDA, fn, b);
}

int aegis_i8_gemm_workspace(int M, int N, int K, const void* A, int64_t lda, const void* W, int64_t ldw,
                            size_t* bytes) {
  const char* fn = "aegis_i8_gemm_workspace";
  if (!bytes) return bad(fn, "bytes is NULL");
  if (!size_ok(M) || !size_ok(N) || K < 0) return bad(fn, "negative size or a size above 2^31 - 2^20");
  if (K > AEGIS_I8_MAX_K) return bad(fn, "K above AEGIS_I8_MAX_K: the int32 sum could overflow");
  const aegis::i8::GemmSpace need = aegis::i8::gemm_space(A, lda, W, ldw, M, N, K);
  *bytes = M == 0 || N == 0 ? 0 : need.w + need.a;
  return AEGIS_OK;
}

int aegis_i8_gemm(int device, void* stream, int out_dtype, int M, int N, int K, const void* A, int64_t lda,
                  const void* W, int64_t ldw, const float* a_scale, const float* w_scale, const void* bias, void* C,
                  int64_t ldc, void* workspace, size_t workspace_bytes) {
  const char* fn = "aegis_i8_gemm";
  Gemm g;
  g.A = A;
  g.W = W;
  g.a_scale = a_scale;
  g.w_scale = w_scale;
  g.bias = bias;
  g.C = C;
  g.M = M;
  g.N = N;
  g.K = K;
  g.lda = lda;
  g.ldw = ldw;
  g.ldc = ldc;
  if (const char* w = check(g, out_dtype)) return bad(fn, w);
  g.out = static_cast<Out>(out_dtype);
  if (M == 0 || N == 0) return AEGIS_OK;
  const aegis::i8::GemmSpace need = aegis::i8::gemm_space(A, lda, W, ldw, M, N, K);
  if (need.w + need.a > 0) {
    if (!workspace || workspace_bytes < need.w + need.a)
      return fail(AEGIS_ERR_BUFFER_TOO_SMALL, fn, "the workspace is smaller than aegis_i8_gemm_workspace asks for");
    if (!aligned(workspace, 256)) return bad(fn, "the workspace is not 256-byte aligned");
  }
  g.workspace = workspace;
  return on_device(device, fn, [&] { return aegis::i8::gemm(g, static_cast<cudaStream_t>(stream)); });
}

int aegis_i8_rmsnorm(int device, void* stream, int dtype, int rows, int cols, const void* x, int64_t ldx,
                     const void* residual, int64_t ldr, const void* weight, float eps, void* h, int64_t ldh, void* q,
                     int64_t ldq, float* scale) {
  const char* fn = "aegis_i8_rmsnorm";
  RowOp o;
  o.bf16 = dtype == AEGIS_DTYPE_BF16;
  o.rows = rows;
  o.cols = cols;
  o.x = x;
  o.ldx = ldx;
  o.residual = residual;
  o.ldr = ldr;
  o.weight = weight;
  o.eps = eps;
  o.h = h;
  o.ldh = ldh;
  o.q = q;
  o.ldq = ldq;
  o.scale = scale;
  if (const char* w = check_norm(o, dtype)) return bad(fn, w);
  if (rows == 0) return AEGIS_OK;
  return on_device(device, fn, [&] { return aegis::i8::rmsnorm(o, static_cast<cudaStream_t>(stream)); });
}

int aegis_i8_silu_mul(int device, void* stream, int dtype, int rows, int cols, const void* gate, int64_t ldg,
                      const void* up, int64_t ldu, void* q, int64_t ldq, float* scale) {
  const char* fn = "aegis_i8_silu_mul";
  RowOp o;
  o.bf16 = dtype == AEGIS_DTYPE_BF16;
  o.rows = rows;
  o.cols = cols;
  o.x = gate;
  o.ldx = ldg;
  o.residual = up;
  o.ldr = ldu;
  o.q = q;
  o.ldq = ldq;
  o.scale = scale;
  if (const char* w = check_rows(o, dtype)) return bad(fn, w);
  if (rows == 0) return AEGIS_OK;
  if (!up) return bad(fn, "an operand is NULL");
  if (ldu < cols) return bad(fn, "a row stride is smaller than the row");
  return on_device(device, fn, [&] { return aegis::i8::silu_mul(o, static_cast<cudaStream_t>(stream)); });
}

int aegis_i8_mlp_workspace(int M, int K, int F, const void* w_gate_up, int64_t ld_gate_up, const void* w_down,
                           int64_t ld_down, size_t* bytes) {
  const char* fn = "aegis_i8_mlp_workspace";
  if (!bytes) return bad(fn, "bytes is NULL");
  if (const char* w = check_mlp_sizes(M, K, F)) return bad(fn, w);
  *bytes = MlpSpace(M, K, F, w_gate_up, ld_gate_up, w_down, ld_down).bytes;
  return AEGIS_OK;
}

int aegis_i8_mlp(int device, void* stream, int dtype, int M, int K, int F, const void* x, int64_t ldx,
                 const void* residual, int64_t ldr, const void* norm_weight, float eps, const void* w_gate_up,
                 int64_t ld_gate_up, const float* s_gate_up, const void* w_down, int64_t ld_down, const float* s_down,
                 void* h, int64_t ldh, void* y, int64_t ldy, void* workspace, size_t workspace_bytes) {
  const char* fn = "aegis_i8_mlp";
  if (const char* w = check_mlp_sizes(M, K, F)) return bad(fn, w);
  if (!dtype16(dtype)) return bad(fn, "dtype must be AEGIS_DTYPE_F16 or AEGIS_DTYPE_BF16");
  if (M == 0) return AEGIS_OK;
  const MlpSpace at(M, K, F, w_gate_up, ld_gate_up, w_down, ld_down);
  if (!workspace || workspace_bytes < at.bytes)
    return fail(AEGIS_ERR_BUFFER_TOO_SMALL, fn, "the workspace is smaller than aegis_i8_mlp_workspace asks for");
  if (!aligned(workspace, 256)) return bad(fn, "the workspace is not 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  const Out out = static_cast<Out>(dtype);

  RowOp norm;
  norm.bf16 = dtype == AEGIS_DTYPE_BF16;
  norm.rows = M;
  norm.cols = K;
  norm.x = x;
  norm.ldx = ldx;
  norm.residual = residual;
  norm.ldr = ldr;
  norm.weight = norm_weight;
  norm.eps = eps;
  norm.h = h;
  norm.ldh = ldh;
  norm.q = ws + at.q1;
  norm.ldq = at.ld1;
  norm.scale = reinterpret_cast<float*>(ws + at.s1);
  if (const char* w = check_norm(norm, dtype)) return bad(fn, w);

  Gemm g1;
  g1.A = norm.q;
  g1.lda = at.ld1;
  g1.a_scale = norm.scale;
  g1.W = w_gate_up;
  g1.ldw = ld_gate_up;
  g1.w_scale = s_gate_up;
  g1.C = ws + at.gu;
  g1.ldc = at.ldgu;
  g1.M = M;
  g1.N = 2 * F;
  g1.K = K;
  g1.out = out;
  g1.weights_settled = true;
  if (const char* w = check(g1, dtype)) return bad(fn, w);

  RowOp act;
  act.bf16 = norm.bf16;
  act.rows = M;
  act.cols = F;
  act.x = ws + at.gu;
  act.ldx = at.ldgu;
  act.residual = ws + at.gu + size_t(F) * 2;
  act.ldr = at.ldgu;
  act.q = ws + at.q2;
  act.ldq = at.ld2;
  act.scale = reinterpret_cast<float*>(ws + at.s2);

  Gemm g2;
  g2.A = act.q;
  g2.lda = at.ld2;
  g2.a_scale = act.scale;
  g2.W = w_down;
  g2.ldw = ld_down;
  g2.w_scale = s_down;
  g2.C = y;
  g2.ldc = ldy;
  g2.M = M;
  g2.N = K;
  g2.K = F;
  g2.out = out;
  g2.weights_settled = true;
  if (const char* w = check(g2, dtype)) return bad(fn, w);

  // Copies first: the products may then read them before the row operations end.
  return on_device(device, fn, [&] {
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (at.copy1) {
      e = aegis::i8::align(w_gate_up, ld_gate_up, 2 * F, K, ws + at.w1, s);
      g1.W = ws + at.w1;
      g1.ldw = (long long)aegis::i8::aligned_cols(K);
    }
    if (at.copy2 && e == cudaSuccess) {
      e = aegis::i8::align(w_down, ld_down, K, F, ws + at.w2, s);
      g2.W = ws + at.w2;
      g2.ldw = (long long)aegis::i8::aligned_cols(F);
    }
    if (e == cudaSuccess) e = aegis::i8::rmsnorm(norm, s);
    if (e == cudaSuccess) e = aegis::i8::gemm(g1, s);
    if (e == cudaSuccess) e = aegis::i8::silu_mul(act, s);
    if (e == cudaSuccess) e = aegis::i8::gemm(g2, s);
    return e;
  });
}

int aegis_i8_gemm_plan_json(int sm_count, int M, int N, int K, char* buf, size_t buf_len, size_t* needed) {
  const char* fn = "aegis_i8_gemm_plan_json";
  if (M < 1 || N < 1 || K < 0 || !size_ok(M) || !size_ok(N) || K > AEGIS_I8_MAX_K)
    return bad(fn, "M and N must be from 1 to 2^31 - 2^20, K from 0 to AEGIS_I8_MAX_K");
  if (sm_count < 1 || sm_count > 4096) return bad(fn, "sm_count must be from 1 to 4096");
  const aegis::i8::GemmPlan p = aegis::i8::plan_gemm(M, N, K, sm_count);
  const char* kernel = p.kernel == aegis::i8::GemmKernel::Pair  ? "pair"
                       : p.kernel == aegis::i8::GemmKernel::Dot ? "dot"
                                                                 : "stream";
  char b[256];
  const int n = std::snprintf(b, sizeof b,
                              "{\"kernel\":\"%s\",\"tile_m\":%d,\"tile_n\":%d,\"splits\":%d,\"tiles\":%lld,\"grid\":%lld}",
                              kernel, p.tile_m, p.tile_n, p.splits, p.tiles, p.grid);
  if (needed) *needed = size_t(n) + 1;
  if (!buf && buf_len == 0) return AEGIS_OK;
  if (!buf) return bad(fn, "buf is NULL but buf_len is not 0");
  if (buf_len < size_t(n) + 1) return fail(AEGIS_ERR_BUFFER_TOO_SMALL, fn, "buffer too small (see needed)");
  std::memcpy(buf, b, size_t(n) + 1);
  return AEGIS_OK;
}

}  // extern "C"
