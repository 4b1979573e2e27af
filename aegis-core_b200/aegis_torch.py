"""torch.ops.aegis: the library's operators as PyTorch operators.

matmul: the 16-bit GEMM.

    import aegis_torch  # registers the op
    C = torch.ops.aegis.matmul(A, B)      # A [M, K], B [K, N], both f16 or both bf16, on one CUDA device

The op calls the C ABI (aegis_gemm_f16_ex / aegis_gemm_bf16_ex through
aegis_capi) on torch's current stream, so it orders with the surrounding torch
work. The dispatcher picks the kernel: the tuned winner for the shape, else
the built-in rule. Operands may be row-major (contiguous) or column-major
(transposed views). Any other stride pattern is copied to a contiguous tensor
first. C is a new row-major tensor of the inputs' dtype (FP32 accumulation).
A fake implementation gives shapes under meta and fake tensors.

It is the Python-side counterpart of the reference's C++ aegis::matmul and
only plumbing: the GEMM is the same C-ABI call every other caller makes.

The 8-bit operators (include/aegis_i8.h has their definitions; sm_100 only):

    q, s    = torch.ops.aegis.rmsnorm_i8(x, weight, eps)                # x [M, K] f16 or bf16
    q, s, h = torch.ops.aegis.add_rmsnorm_i8(x, residual, weight, eps)  # h = x + residual
    y       = torch.ops.aegis.matmul_i8(q, w, s, w_scale, bias=None, out_dtype=torch.bfloat16)  # w [N, K] int8
    q, s    = torch.ops.aegis.silu_mul_i8(gate, up)
    y, h    = torch.ops.aegis.mlp_i8(x, residual, norm_weight, eps, w_gate_up, s_gate_up, w_down, s_down)

They run on torch's current stream of their operands' device, may be captured
into CUDA graphs after one call on the device, and have fake implementations.
Rows may be strided (stride(-1) == 1, rows that do not overlap); other stride
patterns are copied first. The int8 results have rows padded to 16 bytes
(stride(0) is a multiple of 16), which is what the product reads fastest. eps
is taken in 32 bits.
They have no derivatives: an input that requires a gradient while gradients
are recorded, or that carries a forward tangent, is refused, under torch.func's
transforms too.
"""
from __future__ import annotations

import os
import threading

import torch
from torch.library import custom_op

import aegis_capi as ac
import aegis_i8 as i8

_lock = threading.Lock()
_contexts: dict[int, ac.Context] = {}


def _context(device: int) -> ac.Context:
    with _lock:
        ctx = _contexts.get(device)
        if ctx is None:
            ctx = ac.Context(device)
            _contexts[device] = ctx
        return ctx


def _operand(t: torch.Tensor):
    """(tensor, layout, ld) for a 2-D operand: row-major if rows are
    contiguous, column-major if columns are, else a contiguous copy."""
    r, c = t.shape
    if t.stride(1) == 1 and (r <= 1 or t.stride(0) >= c):
        return t, ac.ROW_MAJOR, max(t.stride(0), c, 1)
    if t.stride(0) == 1 and (c <= 1 or t.stride(1) >= r):
        return t, ac.COL_MAJOR, max(t.stride(1), r, 1)
    t = t.contiguous()
    return t, ac.ROW_MAJOR, max(c, 1)


@custom_op("aegis::matmul", mutates_args=())
def matmul(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("aegis::matmul takes 2-D operands")
    if a.shape[1] != b.shape[0]:
        raise ValueError(f"aegis::matmul: inner sizes differ ({tuple(a.shape)} x {tuple(b.shape)})")
    if a.dtype != b.dtype or a.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("aegis::matmul: both operands float16 or both bfloat16")
    if not (a.is_cuda and b.is_cuda) or a.device != b.device:
        raise ValueError("aegis::matmul: both operands on one CUDA device")
    M, K = a.shape
    N = b.shape[1]
    out = torch.empty((M, N), dtype=a.dtype, device=a.device)
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out.zero_()
    a_, la, lda = _operand(a)
    b_, lb, ldb = _operand(b)
    dtype = ac.DTYPE_BF16 if a.dtype == torch.bfloat16 else ac.DTYPE_F16
    ctx = _context(a.device.index if a.device.index is not None else torch.cuda.current_device())
    with torch.cuda.device(a.device):
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        ctx.gemm_ex(la, lb, M, N, K, 1.0, a_.data_ptr(), lda, b_.data_ptr(), ldb, 0.0, out.data_ptr(), N, dtype)
    return out


@matmul.register_fake
def _(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    torch._check(a.dim() == 2 and b.dim() == 2, lambda: "aegis::matmul takes 2-D operands")
    torch._check(a.shape[1] == b.shape[0], lambda: "aegis::matmul: inner sizes differ")
    return a.new_empty((a.shape[0], b.shape[1]))


# ---------------------------------------------------------------- 8-bit operators
_OUT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)

_defs = torch.library.Library("aegis", "FRAGMENT")
_defs.define("matmul_i8(Tensor a, Tensor w, Tensor a_scale, Tensor w_scale, Tensor? bias=None, *, "
             "ScalarType? out_dtype=None) -> Tensor")
_defs.define("rmsnorm_i8(Tensor x, Tensor weight, float eps) -> (Tensor, Tensor)")
_defs.define("add_rmsnorm_i8(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)")
_defs.define("silu_mul_i8(Tensor gate, Tensor up) -> (Tensor, Tensor)")
_defs.define("mlp_i8(Tensor x, Tensor residual, Tensor norm_weight, float eps, Tensor w_gate_up, Tensor s_gate_up, "
             "Tensor w_down, Tensor s_down) -> (Tensor, Tensor)")


def _same_device(name: str, first: torch.Tensor, *others) -> None:
    d = first.device
    for t in others:
        if t is not None and t.device != d:
            raise ValueError(f"aegis::{name}: operands on different devices ({d} and {t.device})")


_MAX_SIZE = 2 ** 31 - 2 ** 20  # the C calls' limit


def _sizes_fit(name: str, *tensors) -> None:
    for t in tensors:
        for n in t.shape:
            if n > _MAX_SIZE:
                raise ValueError(f"aegis::{name}: a size above 2^31 - 2^20")


def _f32_vector(name: str, what: str, t: torch.Tensor, n) -> None:
    if t.dtype != torch.float32:
        raise TypeError(f"aegis::{name}: {what} must be float32, not {t.dtype}")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"aegis::{name}: {what} must have shape ({n},), not {tuple(t.shape)}")


def _check_matmul_i8(a, w, a_scale, w_scale, bias, out_dtype):
    name = "matmul_i8"
    if a.dim() != 2 or w.dim() != 2:
        raise ValueError("aegis::matmul_i8 takes 2-D operands")
    if a.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"aegis::matmul_i8: a and w must be int8, not {a.dtype} and {w.dtype}")
    if a.shape[1] != w.shape[1]:
        raise ValueError(f"aegis::matmul_i8: a [M, K] and w [N, K] have different K ({tuple(a.shape)}, {tuple(w.shape)})")
    if a.shape[1] > i8.MAX_K:
        raise ValueError(f"aegis::matmul_i8: K above {i8.MAX_K}: the int32 sum could overflow")
    _sizes_fit(name, a, w)
    _f32_vector(name, "a_scale", a_scale, a.shape[0])
    _f32_vector(name, "w_scale", w_scale, w.shape[0])
    if out_dtype is None:
        out_dtype = bias.dtype if bias is not None else torch.bfloat16
    if out_dtype not in _OUT_DTYPES:
        raise TypeError(f"aegis::matmul_i8: out_dtype must be float16, bfloat16 or float32, not {out_dtype}")
    if bias is not None:
        if bias.dtype != out_dtype:
            raise TypeError(f"aegis::matmul_i8: bias must have the output's type, {out_dtype}")
        if bias.dim() != 1 or bias.shape[0] != w.shape[0]:
            raise ValueError(f"aegis::matmul_i8: bias must have shape ({w.shape[0]},), not {tuple(bias.shape)}")
    _same_device(name, a, w, a_scale, w_scale, bias)
    return out_dtype


def _matmul_i8_meta(a, w, a_scale, w_scale, bias=None, *, out_dtype=None):
    out_dtype = _check_matmul_i8(a, w, a_scale, w_scale, bias, out_dtype)
    return a.new_empty((a.shape[0], w.shape[0]), dtype=out_dtype)


def _empty_codes(x: torch.Tensor):
    """(q, scale) for the rows of x: int8 rows 16 bytes aligned, one float a row."""
    rows, cols = x.shape
    return (torch.empty_strided((rows, cols), ((cols + 15) // 16 * 16, 1), dtype=torch.int8, device=x.device),
            torch.empty((rows,), dtype=torch.float32, device=x.device))


def _check_rows(name, x, y, what):
    if x.dim() != 2:
        raise ValueError(f"aegis::{name} takes 2-D operands")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"aegis::{name}: operands must be float16 or bfloat16, not {x.dtype}")
    if x.shape[1] == 0:
        raise ValueError(f"aegis::{name}: rows of no elements have no scale")
    _sizes_fit(name, x)
    if y is not None:
        if y.dtype != x.dtype:
            raise TypeError(f"aegis::{name}: {what} must have x's type, {x.dtype}, not {y.dtype}")
        if y.shape != x.shape:
            raise ValueError(f"aegis::{name}: {what} must have shape {tuple(x.shape)}, not {tuple(y.shape)}")


def _check_norm(name, x, residual, weight, eps):
    _check_rows(name, x, residual, "residual")
    if weight.dtype != x.dtype:
        raise TypeError(f"aegis::{name}: weight must have x's type, {x.dtype}, not {weight.dtype}")
    if weight.dim() != 1 or weight.shape[0] != x.shape[1]:
        raise ValueError(f"aegis::{name}: weight must have shape ({x.shape[1]},), not {tuple(weight.shape)}")
    if not 0.0 <= eps <= 3.4e38:
        raise ValueError(f"aegis::{name}: eps must be a finite number, 0 or more")
    _same_device(name, x, residual, weight)


def _rmsnorm_i8_meta(x, weight, eps):
    _check_norm("rmsnorm_i8", x, None, weight, eps)
    return _empty_codes(x)


def _add_rmsnorm_i8_meta(x, residual, weight, eps):
    _check_norm("add_rmsnorm_i8", x, residual, weight, eps)
    return (*_empty_codes(x), x.new_empty(x.shape))


def _check_silu_mul(gate, up):
    _check_rows("silu_mul_i8", gate, up, "up")
    _same_device("silu_mul_i8", gate, up)


def _silu_mul_i8_meta(gate, up):
    _check_silu_mul(gate, up)
    return _empty_codes(gate)


def _check_mlp(x, residual, norm_weight, eps, w_gate_up, s_gate_up, w_down, s_down):
    name = "mlp_i8"
    _check_norm(name, x, residual, norm_weight, eps)
    for what, w in (("w_gate_up", w_gate_up), ("w_down", w_down)):
        if w.dtype != torch.int8:
            raise TypeError(f"aegis::mlp_i8: {what} must be int8, not {w.dtype}")
        if w.dim() != 2:
            raise ValueError(f"aegis::mlp_i8: {what} must have two dimensions")
    K, F = x.shape[1], w_down.shape[1]
    if w_gate_up.shape != (2 * F, K) or w_down.shape[0] != K:
        raise ValueError(f"aegis::mlp_i8: x [M, K], w_gate_up [2F, K] and w_down [K, F] do not fit "
                         f"({tuple(x.shape)}, {tuple(w_gate_up.shape)}, {tuple(w_down.shape)})")
    if F == 0 or F > i8.MAX_K or K > i8.MAX_K:
        raise ValueError(f"aegis::mlp_i8: K and F must be from 1 to {i8.MAX_K}")
    _f32_vector(name, "s_gate_up", s_gate_up, 2 * F)
    _f32_vector(name, "s_down", s_down, K)
    _same_device(name, x, w_gate_up, s_gate_up, w_down, s_down)


def _mlp_i8_meta(x, residual, norm_weight, eps, w_gate_up, s_gate_up, w_down, s_down):
    _check_mlp(x, residual, norm_weight, eps, w_gate_up, s_gate_up, w_down, s_down)
    return x.new_empty(x.shape), x.new_empty(x.shape)


for _name, _meta in (("matmul_i8", _matmul_i8_meta), ("rmsnorm_i8", _rmsnorm_i8_meta),
                     ("add_rmsnorm_i8", _add_rmsnorm_i8_meta), ("silu_mul_i8", _silu_mul_i8_meta),
                     ("mlp_i8", _mlp_i8_meta)):
    _defs.impl(_name, _meta, "Meta")

# The CUDA implementations (csrc/i8/torch_ops.cpp) call libaegis_i8.so. Without these
# libraries matmul is there all the same, and calls of the 8-bit operators raise.
_TORCH_LIB = os.path.join(ac.HERE, "build", "libaegis_torch_i8.so")


def _unavailable(name: str, why: str):
    def call(*args, **kwargs):
        raise RuntimeError(f"aegis::{name}: {why}")
    return call


def _load_i8() -> bool:
    why = f"{_TORCH_LIB} is not built: run `make -C aegis-core_b200 all torch` (or __graft_entry__.build())"
    if os.path.exists(_TORCH_LIB):
        try:
            torch.ops.load_library(_TORCH_LIB)
            return True
        except OSError as e:  # libaegis_i8.so is missing, or another torch's library
            why = f"{_TORCH_LIB} cannot be loaded: {e}"
    for name in ("matmul_i8", "rmsnorm_i8", "add_rmsnorm_i8", "silu_mul_i8", "mlp_i8"):
        _defs.impl(name, _unavailable(name, why), "CUDA")
    return False


I8_LOADED = _load_i8()
