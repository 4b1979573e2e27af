// torch.ops.aegis.*_i8 on CUDA tensors: the C ABI of the 8-bit operators
// (include/aegis_i8.h) as dispatcher kernels. They are C++ because a decode
// step's calls take a few microseconds on the GPU each; the same plumbing in
// Python took 15. Schemas and fake implementations are in aegis_torch.py, which
// loads this library. Arguments are checked here as there.
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/core/stack.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "aegis_i8.h"

namespace {

using at::Tensor;
using std::optional;

void done(int status, const char* name) {
  TORCH_CHECK(status == AEGIS_OK, "aegis::", name, ": status ", status, ": ", aegis_i8_last_error_string());
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return AEGIS_DTYPE_F16;
    case at::kBFloat16: return AEGIS_DTYPE_BF16;
    case at::kFloat: return AEGIS_DTYPE_F32;
    default: return -1;
  }
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// The Autograd kernel of every operator here: there are no derivatives, and an input
// that asks for one must not pass as a constant. It stands at this key, and not in the
// kernels below it, because torch.func's transforms show their gradients and tangents
// only here.
void refuse_derivatives(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const bool reverse = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  if (reverse || forward)
    for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size())) {
      if (!v.isTensor() || !v.toTensor().defined()) continue;
      const Tensor& t = v.toTensor();
      TORCH_CHECK(!reverse || !t.requires_grad(), op.schema().name(),
                  " has no backward pass: call it under torch.no_grad() or detach its inputs");
      TORCH_CHECK(!forward || !t._fw_grad(0).defined(), op.schema().name(),
                  " has no forward derivative: an input has a tangent");
    }
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

void same_device(const char* name, const Tensor& first, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == first.device(), "aegis::", name,
                      ": operands on different devices (", first.device(), " and ", t->device(), ")");
}

void f32_vector(const char* name, const char* what, const Tensor& t, int64_t n) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, "aegis::", name, ": ", what, " must be float32, not ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n, "aegis::", name, ": ", what, " must have shape (", n, ",), not ",
                    t.sizes());
}

void size_fits(const char* name, const Tensor& t) {
  for (const int64_t n : t.sizes())
    TORCH_CHECK_VALUE(n <= (int64_t(1) << 31) - (1 << 20), "aegis::", name, ": a size above 2^31 - 2^20");
}

// The tensor (or a contiguous copy) and its row stride, for rows that are
// contiguous and do not overlap. A single row has no stride of its own: one
// of whole 16-byte pieces then, which every kernel can take.
struct Rows {
  Tensor t;
  int64_t ld;
  explicit Rows(const Tensor& x) {
    const int64_t rows = x.size(0), cols = x.size(1);
    if ((x.stride(1) == 1 || cols <= 1) && (x.stride(0) >= cols || rows <= 1)) {
      t = x;
      ld = rows > 1 ? x.stride(0) : (cols + 15) / 16 * 16;
    } else {
      t = x.contiguous();
      ld = std::max<int64_t>(cols, 1);
    }
  }
  const void* data() const { return t.const_data_ptr(); }
};

// Torch's allocator keeps the block for later work of this stream (512-byte aligned).
Tensor workspace(const Tensor& like, size_t bytes) {
  return bytes ? at::empty({int64_t(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

const float* floats(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }

Tensor matmul_i8(const Tensor& a, const Tensor& w, const Tensor& a_scale, const Tensor& w_scale,
                 const optional<Tensor>& bias_, optional<at::ScalarType> out_dtype) {
  const char* name = "matmul_i8";
  const Tensor bias = bias_ ? *bias_ : Tensor();
  TORCH_CHECK_VALUE(a.dim() == 2 && w.dim() == 2, "aegis::matmul_i8 takes 2-D operands");
  TORCH_CHECK_TYPE(a.scalar_type() == at::kChar && w.scalar_type() == at::kChar,
                   "aegis::matmul_i8: a and w must be int8, not ", a.scalar_type(), " and ", w.scalar_type());
  TORCH_CHECK_VALUE(a.size(1) == w.size(1), "aegis::matmul_i8: a [M, K] and w [N, K] have different K (", a.sizes(), ", ",
                    w.sizes(), ")");
  TORCH_CHECK_VALUE(a.size(1) <= AEGIS_I8_MAX_K, "aegis::matmul_i8: K above ", AEGIS_I8_MAX_K,
                    ": the int32 sum could overflow");
  size_fits(name, a);
  size_fits(name, w);
  const int64_t M = a.size(0), K = a.size(1), N = w.size(0);
  f32_vector(name, "a_scale", a_scale, M);
  f32_vector(name, "w_scale", w_scale, N);
  const at::ScalarType dt = out_dtype ? *out_dtype : bias.defined() ? bias.scalar_type() : at::kBFloat16;
  const int code = code_of(dt);
  TORCH_CHECK_TYPE(code >= 0, "aegis::matmul_i8: out_dtype must be float16, bfloat16 or float32, not ", dt);
  if (bias.defined()) {
    TORCH_CHECK_TYPE(bias.scalar_type() == dt, "aegis::matmul_i8: bias must have the output's type, ", dt);
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == N, "aegis::matmul_i8: bias must have shape (", N, ",), not ",
                      bias.sizes());
  }
  same_device(name, a, {&w, &a_scale, &w_scale, &bias});
  Tensor out = at::empty({M, N}, a.options().dtype(dt));
  if (M == 0 || N == 0) return out;
  const Rows ra(a), rw(w);
  const Tensor sa = a_scale.contiguous(), sw = w_scale.contiguous();
  const Tensor b = bias.defined() ? bias.contiguous() : bias;
  size_t bytes = 0;
  done(aegis_i8_gemm_workspace(int(M), int(N), int(K), ra.data(), ra.ld, rw.data(), rw.ld, &bytes), name);
  const Tensor ws = workspace(a, bytes);
  done(aegis_i8_gemm(a.get_device(), stream_of(a), code, int(M), int(N), int(K), ra.data(), ra.ld, rw.data(), rw.ld,
                     floats(sa), floats(sw), b.defined() ? b.const_data_ptr() : nullptr, out.mutable_data_ptr(), N,
                     ws.defined() ? ws.mutable_data_ptr() : nullptr, bytes),
       name);
  return out;
}

void check_rows(const char* name, const Tensor& x, const Tensor& y, const char* what) {
  TORCH_CHECK_VALUE(x.dim() == 2, "aegis::", name, " takes 2-D operands");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, "aegis::", name,
                   ": operands must be float16 or bfloat16, not ", x.scalar_type());
  TORCH_CHECK_VALUE(x.size(1) > 0, "aegis::", name, ": rows of no elements have no scale");
  size_fits(name, x);
  if (y.defined()) {
    TORCH_CHECK_TYPE(y.scalar_type() == x.scalar_type(), "aegis::", name, ": ", what, " must have x's type, ",
                     x.scalar_type(), ", not ", y.scalar_type());
    TORCH_CHECK_VALUE(y.sizes() == x.sizes(), "aegis::", name, ": ", what, " must have shape ", x.sizes(), ", not ",
                      y.sizes());
  }
}

void check_norm(const char* name, const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  check_rows(name, x, residual, "residual");
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "aegis::", name, ": weight must have x's type, ",
                   x.scalar_type(), ", not ", weight.scalar_type());
  TORCH_CHECK_VALUE(weight.dim() == 1 && weight.size(0) == x.size(1), "aegis::", name, ": weight must have shape (",
                    x.size(1), ",), not ", weight.sizes());
  TORCH_CHECK_VALUE(eps >= 0.0 && eps <= 3.4e38, "aegis::", name, ": eps must be a finite number, 0 or more");
  same_device(name, x, {&residual, &weight});
}

// (q, scale) for the rows of x: int8 rows 16 bytes aligned, one float a row.
std::tuple<Tensor, Tensor> empty_codes(const Tensor& x) {
  const int64_t rows = x.size(0), cols = x.size(1);
  return {at::empty_strided({rows, cols}, {(cols + 15) / 16 * 16, 1}, x.options().dtype(at::kChar)),
          at::empty({rows}, x.options().dtype(at::kFloat))};
}

std::tuple<Tensor, Tensor, Tensor> norm(const char* name, const Tensor& x, const Tensor& residual, const Tensor& weight,
                                        double eps) {
  check_norm(name, x, residual, weight, eps);
  auto [q, scale] = empty_codes(x);
  const int64_t rows = x.size(0), cols = x.size(1);
  Tensor h = residual.defined() ? at::empty({rows, cols}, x.options()) : Tensor();
  if (rows) {
    const Rows rx(x);
    const optional<Rows> rr = residual.defined() ? optional<Rows>(Rows(residual)) : std::nullopt;
    const Tensor w = weight.contiguous();
    done(aegis_i8_rmsnorm(x.get_device(), stream_of(x), code_of(x.scalar_type()), int(rows), int(cols), rx.data(), rx.ld,
                          rr ? rr->data() : nullptr, rr ? rr->ld : 0, w.const_data_ptr(), float(eps),
                          h.defined() ? h.mutable_data_ptr() : nullptr, cols, q.mutable_data_ptr(), q.stride(0),
                          static_cast<float*>(scale.mutable_data_ptr())),
         name);
  }
  return {std::move(q), std::move(scale), std::move(h)};
}

std::tuple<Tensor, Tensor> rmsnorm_i8(const Tensor& x, const Tensor& weight, double eps) {
  auto [q, scale, h] = norm("rmsnorm_i8", x, Tensor(), weight, eps);
  return {std::move(q), std::move(scale)};
}

std::tuple<Tensor, Tensor, Tensor> add_rmsnorm_i8(const Tensor& x, const Tensor& residual, const Tensor& weight,
                                                  double eps) {
  return norm("add_rmsnorm_i8", x, residual, weight, eps);
}

std::tuple<Tensor, Tensor> silu_mul_i8(const Tensor& gate, const Tensor& up) {
  const char* name = "silu_mul_i8";
  check_rows(name, gate, up, "up");
  same_device(name, gate, {&up});
  auto [q, scale] = empty_codes(gate);
  if (gate.size(0)) {
    const Rows g(gate), u(up);
    done(aegis_i8_silu_mul(gate.get_device(), stream_of(gate), code_of(gate.scalar_type()), int(gate.size(0)),
                           int(gate.size(1)), g.data(), g.ld, u.data(), u.ld, q.mutable_data_ptr(), q.stride(0),
                           static_cast<float*>(scale.mutable_data_ptr())),
         name);
  }
  return {std::move(q), std::move(scale)};
}

std::tuple<Tensor, Tensor> mlp_i8(const Tensor& x, const Tensor& residual, const Tensor& norm_weight, double eps,
                                  const Tensor& w_gate_up, const Tensor& s_gate_up, const Tensor& w_down,
                                  const Tensor& s_down) {
  const char* name = "mlp_i8";
  check_norm(name, x, residual, norm_weight, eps);
  TORCH_CHECK_TYPE(w_gate_up.scalar_type() == at::kChar && w_down.scalar_type() == at::kChar,
                   "aegis::mlp_i8: w_gate_up and w_down must be int8, not ", w_gate_up.scalar_type(), " and ",
                   w_down.scalar_type());
  TORCH_CHECK_VALUE(w_gate_up.dim() == 2 && w_down.dim() == 2, "aegis::mlp_i8: w_gate_up and w_down must have two dimensions");
  const int64_t M = x.size(0), K = x.size(1), F = w_down.size(1);
  TORCH_CHECK_VALUE(w_gate_up.size(0) == 2 * F && w_gate_up.size(1) == K && w_down.size(0) == K,
                    "aegis::mlp_i8: x [M, K], w_gate_up [2F, K] and w_down [K, F] do not fit (", x.sizes(), ", ",
                    w_gate_up.sizes(), ", ", w_down.sizes(), ")");
  TORCH_CHECK_VALUE(F > 0 && F <= AEGIS_I8_MAX_K && K <= AEGIS_I8_MAX_K, "aegis::mlp_i8: K and F must be from 1 to ",
                    AEGIS_I8_MAX_K);
  f32_vector(name, "s_gate_up", s_gate_up, 2 * F);
  f32_vector(name, "s_down", s_down, K);
  same_device(name, x, {&w_gate_up, &s_gate_up, &w_down, &s_down});
  Tensor y = at::empty({M, K}, x.options()), h = at::empty({M, K}, x.options());
  if (M) {
    const Rows rx(x), rr(residual), w1(w_gate_up), w2(w_down);
    const Tensor g = norm_weight.contiguous(), s1 = s_gate_up.contiguous(), s2 = s_down.contiguous();
    size_t bytes = 0;
    done(aegis_i8_mlp_workspace(int(M), int(K), int(F), w1.data(), w1.ld, w2.data(), w2.ld, &bytes), name);
    const Tensor ws = workspace(x, bytes);
    done(aegis_i8_mlp(x.get_device(), stream_of(x), code_of(x.scalar_type()), int(M), int(K), int(F), rx.data(), rx.ld,
                      rr.data(), rr.ld, g.const_data_ptr(), float(eps), w1.data(), w1.ld, floats(s1), w2.data(), w2.ld,
                      floats(s2), h.mutable_data_ptr(), K, y.mutable_data_ptr(), K, ws.mutable_data_ptr(), bytes),
         name);
  }
  return {std::move(y), std::move(h)};
}

}  // namespace

TORCH_LIBRARY_IMPL(aegis, CUDA, m) {
  m.impl("matmul_i8", &matmul_i8);
  m.impl("rmsnorm_i8", &rmsnorm_i8);
  m.impl("add_rmsnorm_i8", &add_rmsnorm_i8);
  m.impl("silu_mul_i8", &silu_mul_i8);
  m.impl("mlp_i8", &mlp_i8);
}

TORCH_LIBRARY_IMPL(aegis, Autograd, m) {
  for (const char* name : {"matmul_i8", "rmsnorm_i8", "add_rmsnorm_i8", "silu_mul_i8", "mlp_i8"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_derivatives>());
}
