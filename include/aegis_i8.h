/*
 * aegis-b200: C ABI of the 8-bit operators (libaegis_i8.so, sm_100a).
 *
 * The 8-bit companion of include/aegis.h: matrix products of int8 codes with
 * one scale a token and one a channel, the two row operations that make such
 * codes from 16-bit activations, and the feed-forward block that runs them in
 * a row. No counterpart in the reference (its GEMM is 16-bit only).
 *
 * Conventions:
 *   - Status codes are those of aegis.h. Nothing exits or aborts the process.
 *     aegis_i8_last_error_string() has the detail of the last failure on the
 *     calling thread.
 *   - Every call names its device and its stream (a cudaStream_t as void*;
 *     NULL is the legacy default stream), is asynchronous on that stream, and
 *     leaves the calling thread's current device as it was. There is no
 *     context: two threads may call at once.
 *   - Nothing is allocated or kept from one call for the next, except, on the
 *     first call of a device, 16 bytes for the watchdog's status and the
 *     kernels' shared-memory limits: make that call, of any operator, before a
 *     stream capture (a no-op does not count). All calls may be captured into
 *     CUDA graphs after that.
 *   - Operands are device pointers of that device. Leading dimensions count
 *     elements, and every alignment is accepted. Rows of codes whose addresses
 *     are multiples of 16 bytes are read as they are, others from an aligned
 *     copy that the call makes in its workspace.
 *   - A workspace is device memory, 256-byte aligned, of the bytes that its
 *     query gives (0: none, NULL will do). It belongs to the call until it has
 *     run: calls that may overlap need one each.
 *   - Outputs may not overlap inputs, unless said otherwise. Elements between
 *     the rows of an output (ld > columns) are left as they are.
 */
#ifndef AEGIS_B200_AEGIS_I8_H
#define AEGIS_B200_AEGIS_I8_H

#include "aegis.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Output type beside AEGIS_DTYPE_F16 and AEGIS_DTYPE_BF16: float. */
#define AEGIS_DTYPE_F32 2

/* Longest sum whose int32 accumulator cannot overflow: 131071 * 128 * 128 < 2^31. */
#define AEGIS_I8_MAX_K 131071

/* Detail of the last failed call on this thread ("" if none). */
AEGIS_API const char* aegis_i8_last_error_string(void);

/* Waits for `stream` and reports a kernel watchdog that fired on `device`
 * since the last check (see aegis_synchronize) as AEGIS_ERR_CUDA. */
AEGIS_API int aegis_i8_synchronize(int device, void* stream);

/* C[m, n] = a_scale[m] * w_scale[n] * sum_k A[m, k] * W[n, k] + bias[n].
 * A: M x K int8 (tokens), row stride lda >= K. W: N x K int8 (channels, the
 * layout of torch.nn.Linear.weight), row stride ldw >= K. a_scale: M floats,
 * w_scale: N floats. bias: N values of out_dtype, or NULL. C: M x N of
 * out_dtype (AEGIS_DTYPE_F16, _BF16 or _F32), row stride ldc >= N.
 * The sum is exact (int32); it is converted to float, scaled (scales may come
 * near the ends of float's range: no step between leaves it), the bias added
 * in float, and rounded once. K = 0: the sum is 0. M or N = 0: no-op.
 * K > AEGIS_I8_MAX_K, negative sizes, too-small strides, null operands:
 * AEGIS_ERR_INVALID_ARGUMENT. Results do not depend on the alignment of the
 * operands or on how the work is split. */
AEGIS_API int aegis_i8_gemm(int device, void* stream, int out_dtype, int M, int N, int K, const void* A, int64_t lda,
                            const void* W, int64_t ldw, const float* a_scale, const float* w_scale,
                            const void* bias, void* C, int64_t ldc, void* workspace, size_t workspace_bytes);
/* Bytes of workspace that call needs: 0 where the addresses of all rows of A and
 * W are multiples of 16 bytes (of a single row: its address alone). Makes no
 * CUDA call. */
AEGIS_API int aegis_i8_gemm_workspace(int M, int N, int K, const void* A, int64_t lda, const void* W, int64_t ldw,
                                      size_t* bytes);

/* For each of `rows` rows of `cols` elements (dtype f16 or bf16):
 *   h = round(x + residual)   (residual NULL: h = x)
 *   t = h * weight,  m = max |t|
 *   scale = m / sqrt(mean(h^2) + eps) / 127
 *   q = 127 * t / m to the nearest whole number, ties to even
 * so q * scale is the row's root-mean-square norm times weight. q is exactly
 * that number, whatever the row's length or layout. m = 0: q = 0, scale = 0. A
 * row with an h or a t that is not finite (t in 32 bits): q = 0, scale = NaN.
 * With a residual, h is stored (row stride ldh); h may be x or residual itself
 * (same pointer and stride). Without one, h must be NULL. weight: cols values
 * of dtype. q: int8, row stride ldq. scale: `rows` floats. eps >= 0.
 * rows = 0: no-op; cols = 0: AEGIS_ERR_INVALID_ARGUMENT. */
AEGIS_API int aegis_i8_rmsnorm(int device, void* stream, int dtype, int rows, int cols, const void* x, int64_t ldx,
                               const void* residual, int64_t ldr, const void* weight, float eps, void* h,
                               int64_t ldh, void* q, int64_t ldq, float* scale);

/* For each row: t = gate / (1 + exp(-gate)) * up, m = max |t|, scale = m / 127,
 * q = 127 * t / m to the nearest whole number, ties to even (of t in 64 bits).
 * gate, up: dtype f16 or bf16, row strides ldg and ldu (halves of one product's
 * rows, say). m = 0 and rows that are not finite: as aegis_i8_rmsnorm. */
AEGIS_API int aegis_i8_silu_mul(int device, void* stream, int dtype, int rows, int cols, const void* gate,
                                int64_t ldg, const void* up, int64_t ldu, void* q, int64_t ldq, float* scale);

/* The gated feed-forward block of M tokens, K wide, F hidden, in one call:
 *   q, s, h = aegis_i8_rmsnorm(x, residual, norm_weight, eps)
 *   gate_up = aegis_i8_gemm(q, w_gate_up)      [M, 2F] of dtype; gate is the first half
 *   q2, s2  = aegis_i8_silu_mul(gate, up)
 *   y       = aegis_i8_gemm(q2, w_down)        [M, K] of dtype
 * with the same results as those four calls. w_gate_up: 2F x K int8, s_gate_up
 * 2F floats; w_down: K x F int8, s_down K floats. Each product starts to read
 * its weights while the row operation before it runs. M = 0: no-op. K and F
 * from 1 to AEGIS_I8_MAX_K. aegis_i8_mlp_workspace makes no CUDA call. */
AEGIS_API int aegis_i8_mlp_workspace(int M, int K, int F, const void* w_gate_up, int64_t ld_gate_up,
                                     const void* w_down, int64_t ld_down, size_t* bytes);
AEGIS_API int aegis_i8_mlp(int device, void* stream, int dtype, int M, int K, int F, const void* x, int64_t ldx,
                           const void* residual, int64_t ldr, const void* norm_weight, float eps,
                           const void* w_gate_up, int64_t ld_gate_up, const float* s_gate_up, const void* w_down,
                           int64_t ld_down, const float* s_down, void* h, int64_t ldh, void* y, int64_t ldy,
                           void* workspace, size_t workspace_bytes);

/* The launch aegis_i8_gemm makes on a device with `sm_count` SMs, as JSON
 * {"kernel":..,"tile_m":..,"tile_n":..,"splits":..,"tiles":..,"grid":..}.
 * Needs no GPU. */
AEGIS_API int aegis_i8_gemm_plan_json(int sm_count, int M, int N, int K, char* buf, size_t buf_len, size_t* needed);

#ifdef __cplusplus
}
#endif

#endif /* AEGIS_B200_AEGIS_I8_H */
