#pragma once
// Internal host interface of the 8-bit operators (include/aegis_i8.h has the
// definitions). Every function launches on the current device.
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace aegis::i8 {

enum class Out : int { F16 = 0, BF16 = 1, F32 = 2 };

struct Gemm {
  const void* A = nullptr;  // M x K int8
  const void* W = nullptr;  // N x K int8
  const float* a_scale = nullptr;
  const float* w_scale = nullptr;
  const void* bias = nullptr;
  void* C = nullptr;
  int M = 0, N = 0, K = 0;
  long long lda = 0, ldw = 0, ldc = 0;
  Out out = Out::BF16;
  void* workspace = nullptr;  // of gemm_space's bytes, 256-byte aligned
  // The kernel launched just before on this stream is one of this file's row
  // operations, which let their dependents start only after everything before
  // them has completed: the weights may then be read before that kernel ends.
  bool weights_settled = false;
};

// Which kernel runs, and how the work is cut.
enum class GemmKernel { Dot, Stream, Pair };  // i8_dot.cuh, i8_stream.cuh, i8_pair.cuh
inline constexpr int kDotTokens = 8;          // the most tokens Dot takes
struct GemmPlan {
  GemmKernel kernel = GemmKernel::Stream;
  int tile_m = 0;  // tokens a tile
  int tile_n = 0;  // channels a tile (Dot: a warp's)
  int splits = 1;  // slices of K: CTAs of a cluster (Stream), warps (Dot)
  long long tiles = 0, grid = 0;
};
GemmPlan plan_gemm(int M, int N, int K, int sms);

// Whether TMA can address the rows: 16-byte aligned base, and a stride that is a
// multiple of 16 where there is more than one.
bool tma_rows(const void* p, long long ld, int rows);

// Columns of a copy whose rows TMA can address: whole blocks of 128.
constexpr size_t aligned_cols(int K) { return (size_t(K) + 127) / 128 * 128; }
// Makes such a copy (rows x aligned_cols(K) bytes, 128-byte aligned; zeros from column K on).
cudaError_t align(const void* src, long long ld, int rows, int K, void* dst, cudaStream_t s);

// Bytes of the copies a product needs: the weights', then the tokens' (0: its rows do as they are).
struct GemmSpace {
  size_t w = 0, a = 0;
};
GemmSpace gemm_space(const void* A, long long lda, const void* W, long long ldw, int M, int N, int K);

cudaError_t gemm(const Gemm& g, cudaStream_t s);

struct RowOp {
  bool bf16 = false;
  int rows = 0, cols = 0;
  const void* x = nullptr;         // or gate
  long long ldx = 0;
  const void* residual = nullptr;  // or up
  long long ldr = 0;
  const void* weight = nullptr;
  float eps = 0.f;
  void* h = nullptr;
  long long ldh = 0;
  void* q = nullptr;
  long long ldq = 0;
  float* scale = nullptr;
};
cudaError_t rmsnorm(const RowOp& r, cudaStream_t s);
cudaError_t silu_mul(const RowOp& r, cudaStream_t s);

}  // namespace aegis::i8
