"""The 8-bit operators without a GPU: the library exports exactly the declared
functions, arguments are refused before any CUDA call (C ABI) and under meta
tensors (torch.ops.aegis.*_i8), fake implementations give the shapes and
strides of the results, and the planner's cuts hold over a range of sizes."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import aegis_capi as ac
import aegis_i8 as i8
import aegis_torch  # noqa: F401  (registers the operators)
from conftest import ROOT

HEADER = os.path.join(ROOT, "include", "aegis_i8.h")
ops = torch.ops.aegis
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def test_exports_exactly_the_declared_functions():
    decl = sorted(set(re.findall(r"^AEGIS_API [^(]*?\b(aegis_i8_[a-z0-9_]+)\s*\(", open(HEADER).read(), re.M)))
    out = subprocess.run(["nm", "-D", "--defined-only", i8.LIB_PATH], check=True, capture_output=True, text=True)
    assert sorted({line.split()[-1] for line in out.stdout.splitlines() if line.strip()}) == decl
    assert set(decl) == set(i8._SIGNATURES)


def test_header_is_strict_c11(tmp_path):
    c = tmp_path / "t.c"
    c.write_text('#include "aegis_i8.h"\nint main(void){return AEGIS_I8_MAX_K == 131071 ? 0 : 1;}\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-pedantic",
                    "-I" + os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "t")], check=True)


# ---------------------------------------------------------------- C ABI refusals
P = 4096  # an address that is never used: the checks come first


def gemm(**kw):
    a = dict(device=0, stream=None, out_dtype=1, M=4, N=8, K=32, A=P, lda=32, W=P, ldw=32, sa=P, sw=P, bias=None,
             C=P, ldc=8, ws=None, wsb=0)
    a.update(kw)
    return i8.load().aegis_i8_gemm(*a.values())


def norm(**kw):
    a = dict(device=0, stream=None, dtype=1, rows=4, cols=32, x=P, ldx=32, residual=P, ldr=32, weight=P, eps=1e-5,
             h=2 * P, ldh=32, q=P, ldq=32, scale=P)
    a.update(kw)
    return i8.load().aegis_i8_rmsnorm(*a.values())


def silu(**kw):
    a = dict(device=0, stream=None, dtype=0, rows=4, cols=32, gate=P, ldg=64, up=P + 64, ldu=64, q=P, ldq=32, scale=P)
    a.update(kw)
    return i8.load().aegis_i8_silu_mul(*a.values())


def mlp(**kw):
    a = dict(device=0, stream=None, dtype=1, M=2, K=32, F=64, x=P, ldx=32, residual=P, ldr=32, nw=P, eps=1e-5, wgu=P,
             ldgu=32, sgu=P, wd=P, ldd=64, sd=P, h=2 * P, ldh=32, y=P, ldy=32, ws=P, wsb=1 << 20)
    a.update(kw)
    return i8.load().aegis_i8_mlp(*a.values())


@pytest.mark.parametrize("call,kw,text", [
    (gemm, dict(out_dtype=3), "out_dtype"), (gemm, dict(out_dtype=-1), "out_dtype"),
    (gemm, dict(M=-1), "size"), (gemm, dict(N=-1), "size"), (gemm, dict(K=-1), "size"),
    (gemm, dict(K=131072, lda=131072, ldw=131072), "overflow"),
    (gemm, dict(A=None), "NULL"), (gemm, dict(W=None), "NULL"), (gemm, dict(C=None), "NULL"),
    (gemm, dict(sa=None), "NULL"), (gemm, dict(sw=None), "NULL"),
    (gemm, dict(lda=31), "stride"), (gemm, dict(ldw=31), "stride"), (gemm, dict(ldc=7), "stride"),
    (gemm, dict(C=P + 1), "aligned"), (gemm, dict(sa=P + 2), "aligned"), (gemm, dict(bias=P + 1), "aligned"),
    (gemm, dict(out_dtype=2, C=P + 2), "aligned"),
    (norm, dict(dtype=2), "dtype"), (norm, dict(rows=-1), "size"), (norm, dict(cols=-1), "size"),
    (norm, dict(cols=0), "no elements"), (norm, dict(x=None), "NULL"), (norm, dict(q=None), "NULL"),
    (norm, dict(scale=None), "NULL"), (norm, dict(weight=None), "NULL"), (norm, dict(ldx=31), "stride"),
    (norm, dict(ldq=31), "stride"), (norm, dict(ldr=31), "strides"), (norm, dict(h=None), "h must be given"),
    (norm, dict(residual=None), "without a residual"), (norm, dict(eps=-1.0), "eps"),
    (norm, dict(eps=float("nan")), "eps"), (norm, dict(eps=float("inf")), "eps"),
    (norm, dict(h=P, ldh=40), "same row stride"), (norm, dict(x=P + 1), "aligned"),
    (silu, dict(up=None), "NULL"), (silu, dict(ldu=31), "stride"), (silu, dict(ldg=31), "stride"),
    (silu, dict(cols=0), "no elements"), (silu, dict(dtype=5), "dtype"),
    (mlp, dict(K=0), "from 1"), (mlp, dict(F=0), "from 1"), (mlp, dict(F=131072), "from 1"), (mlp, dict(M=-1), "size"),
    (mlp, dict(dtype=2), "dtype"), (mlp, dict(ws=P + 128), "256"), (mlp, dict(wgu=None), "NULL"),
    (mlp, dict(ldgu=31), "stride"), (mlp, dict(ldd=63), "stride"), (mlp, dict(y=None), "NULL"),
    (mlp, dict(sd=None), "NULL"), (mlp, dict(nw=None), "NULL"),
])
def test_c_abi_refusals(call, kw, text):
    assert call(**kw) == ac.AEGIS_ERR_INVALID_ARGUMENT
    assert text in i8.last_error_string()


def test_c_abi_no_ops_workspace_and_devices():
    assert gemm(M=0) == ac.AEGIS_OK and gemm(N=0, A=None, C=None) == ac.AEGIS_OK
    assert norm(rows=0, x=None) == ac.AEGIS_OK and silu(rows=0) == ac.AEGIS_OK and mlp(M=0, ws=None) == ac.AEGIS_OK
    assert mlp(ws=None) == ac.AEGIS_ERR_BUFFER_TOO_SMALL
    assert mlp(wsb=i8.mlp_workspace(2, 32, 64, P, 32, P, 64) - 1) == ac.AEGIS_ERR_BUFFER_TOO_SMALL
    assert "workspace" in i8.last_error_string()
    assert gemm(device=-1) == ac.AEGIS_ERR_NO_DEVICE and norm(device=1 << 20) == ac.AEGIS_ERR_NO_DEVICE
    # gate_up alone takes M * 2F 16-bit values; rows of codes are padded to 16 bytes.
    least = 3 * (48 + 4 + 2 * 136 + 80 + 4)
    assert least <= i8.mlp_workspace(3, 33, 65, P, 48, P, 80) <= least + 5 * 256
    # weights whose rows are not 16 bytes aligned are copied to rows of whole 128-code blocks
    assert i8.mlp_workspace(3, 33, 65, P, 33, P, 80) >= least + 130 * 128
    assert i8.mlp_workspace(3, 33, 65, P, 48, P + 1, 80) >= least + 33 * 128
    assert i8.mlp_workspace(0, 33, 65, P, 33, P, 65) == 0
    assert i8.load().aegis_i8_mlp_workspace(1, 1, 1, P, 1, P, 1, None) == ac.AEGIS_ERR_INVALID_ARGUMENT
    with pytest.raises(i8.AegisError):
        i8.mlp_workspace(1, 0, 1, P, 16, P, 16)


def test_product_workspace():
    assert i8.gemm_workspace(4, 8, 32, P, 32, P, 48) == 0
    assert i8.gemm_workspace(4, 8, 33, P, 33, P, 48) == 4 * 128
    assert i8.gemm_workspace(4, 8, 129, P, 144, P + 8, 144) == 8 * 256
    assert i8.gemm_workspace(4, 8, 129, P + 1, 144, P, 129) == 12 * 256
    assert i8.gemm_workspace(4, 8, 0, P, 1, P, 1) == 0 and i8.gemm_workspace(0, 8, 33, P, 33, P, 33) == 0
    assert i8.load().aegis_i8_gemm_workspace(-1, 8, 32, P, 32, P, 32, ctypes.byref(ctypes.c_size_t())) != ac.AEGIS_OK
    assert i8.load().aegis_i8_gemm_workspace(4, 8, 32, P, 32, P, 32, None) == ac.AEGIS_ERR_INVALID_ARGUMENT
    assert gemm(K=33, lda=33, ldw=48) == ac.AEGIS_ERR_BUFFER_TOO_SMALL
    assert gemm(K=33, lda=33, ldw=48, ws=P, wsb=4 * 128 - 1) == ac.AEGIS_ERR_BUFFER_TOO_SMALL
    assert gemm(K=33, lda=33, ldw=48, ws=P + 128, wsb=1 << 20) == ac.AEGIS_ERR_INVALID_ARGUMENT


def test_plan_json_protocol():
    f = i8.load().aegis_i8_gemm_plan_json
    need = ctypes.c_size_t(0)
    assert f(148, 4, 4, 4, None, 0, ctypes.byref(need)) == ac.AEGIS_OK and need.value > 20
    buf = ctypes.create_string_buffer(4)
    assert f(148, 4, 4, 4, buf, 4, None) == ac.AEGIS_ERR_BUFFER_TOO_SMALL
    assert f(0, 4, 4, 4, None, 0, None) == ac.AEGIS_ERR_INVALID_ARGUMENT
    assert f(148, 0, 4, 4, None, 0, None) == ac.AEGIS_ERR_INVALID_ARGUMENT
    assert f(148, 4, 4, 131072, None, 0, None) == ac.AEGIS_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("sms", [1, 20, 132, 148])
def test_plans_cover_the_problem(sms):
    for M in (1, 2, 15, 16, 17, 33, 64, 100, 129, 256, 257, 1000, 8192, 100000):
        for N in (1, 64, 127, 128, 129, 4096, 14336, 151936):
            for K in (0, 1, 127, 128, 777, 4096, 131071):
                p = i8.gemm_plan(M, N, K, sms)
                tiles = -(-M // p["tile_m"]) * -(-N // p["tile_n"])
                assert p["tiles"] == tiles
                if p["kernel"] == "pair":
                    assert K > 0 and p["grid"] == 2 * tiles and p["splits"] == 1
                elif p["kernel"] == "dot":
                    # 8 warps a block, `splits` of them on the same channels, each with some of K
                    assert K > 0 and M <= 8 and p["tile_m"] == M and p["splits"] in (1, 2, 4, 8)
                    assert p["grid"] * 8 // p["splits"] >= tiles > (p["grid"] - 1) * 8 // p["splits"]
                    assert p["splits"] == 1 or K >= 512 * p["splits"]
                else:
                    # one CTA of a cluster a slice; at most 8 CTAs a cluster everywhere; no slice without k-blocks
                    assert p["grid"] == tiles * p["splits"] and p["splits"] in (1, 2, 4, 8)
                    assert p["splits"] <= max(1, -(-K // 128))
                    assert p["tile_m"] in (16, 32, 64, 128, 256)
                    # whole rows of the swizzle; a cluster's slices are at most the SMs' slots
                    assert p["tile_n"] % 8 == 0 and 8 <= p["tile_n"] <= 128
                    assert p["splits"] == 1 or p["grid"] <= 2 * sms


# ---------------------------------------------------------------- torch operators
def meta(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_fake_shapes_and_strides():
    a, w = meta(5, 777, dtype=torch.int8), meta(33, 777, dtype=torch.int8)
    sa, sw = meta(5, dtype=F32), meta(33, dtype=F32)
    c = ops.matmul_i8(a, w, sa, sw)
    assert c.shape == (5, 33) and c.dtype == BF16
    assert ops.matmul_i8(a, w, sa, sw, out_dtype=F32).dtype == F32
    assert ops.matmul_i8(a, w, sa, sw, meta(33, dtype=F16)).dtype == F16
    q, s = ops.rmsnorm_i8(meta(5, 100), meta(100), 1e-5)
    assert q.shape == (5, 100) and q.stride() == (112, 1) and q.dtype == torch.int8
    assert s.shape == (5,) and s.dtype == F32
    q, s, h = ops.add_rmsnorm_i8(meta(5, 128), meta(5, 128), meta(128), 1e-5)
    assert q.is_contiguous() and h.shape == (5, 128) and h.dtype == BF16
    q, s = ops.silu_mul_i8(meta(5, 64, dtype=F16), meta(5, 64, dtype=F16))
    assert q.shape == (5, 64) and s.shape == (5,)
    y, h = ops.mlp_i8(meta(5, 48), meta(5, 48), meta(48), 1e-5, meta(40, 48, dtype=torch.int8), meta(40, dtype=F32),
                      meta(48, 20, dtype=torch.int8), meta(48, dtype=F32))
    assert y.shape == h.shape == (5, 48) and y.dtype == h.dtype == BF16


I8 = torch.int8


@pytest.mark.parametrize("make,error", [
    (lambda: ops.matmul_i8(meta(4, 8), meta(4, 8, dtype=I8), meta(4, dtype=F32), meta(4, dtype=F32)), TypeError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(4, 9, dtype=I8), meta(4, dtype=F32), meta(4, dtype=F32)), ValueError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(2, 4, 8, dtype=I8), meta(4, dtype=F32), meta(4, dtype=F32)), ValueError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(4, 8, dtype=I8), meta(5, dtype=F32), meta(4, dtype=F32)), ValueError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(4, 8, dtype=I8), meta(4, dtype=F32), meta(4)), TypeError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(4, 8, dtype=I8), meta(4, dtype=F32), meta(4, dtype=F32),
                           out_dtype=torch.int8), TypeError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(4, 8, dtype=I8), meta(4, dtype=F32), meta(4, dtype=F32),
                           meta(4), out_dtype=F32), TypeError),
    (lambda: ops.matmul_i8(meta(4, 8, dtype=I8), meta(4, 8, dtype=I8), meta(4, dtype=F32), meta(4, dtype=F32),
                           meta(5)), ValueError),
    (lambda: ops.matmul_i8(meta(1, 131072, dtype=I8), meta(1, 131072, dtype=I8), meta(1, dtype=F32),
                           meta(1, dtype=F32)), ValueError),
    (lambda: ops.rmsnorm_i8(meta(4, 8, dtype=F32), meta(8, dtype=F32), 1e-5), TypeError),
    (lambda: ops.rmsnorm_i8(meta(4, 8), meta(8, dtype=F16), 1e-5), TypeError),
    (lambda: ops.rmsnorm_i8(meta(4, 8), meta(7), 1e-5), ValueError),
    (lambda: ops.rmsnorm_i8(meta(4, 8), meta(8), -1.0), ValueError),
    (lambda: ops.rmsnorm_i8(meta(4, 8), meta(8), float("nan")), ValueError),
    (lambda: ops.rmsnorm_i8(meta(8), meta(8), 1e-5), ValueError),
    (lambda: ops.rmsnorm_i8(meta(4, 0), meta(0), 1e-5), ValueError),
    (lambda: ops.add_rmsnorm_i8(meta(4, 8), meta(1, 8), meta(8), 1e-5), ValueError),
    (lambda: ops.add_rmsnorm_i8(meta(4, 8), meta(4, 8, dtype=F16), meta(8), 1e-5), TypeError),
    (lambda: ops.silu_mul_i8(meta(4, 8), meta(4, 9)), ValueError),
    (lambda: ops.silu_mul_i8(meta(4, 8, dtype=I8), meta(4, 8, dtype=I8)), TypeError),
    (lambda: ops.mlp_i8(meta(5, 48), meta(5, 48), meta(48), 1e-5, meta(40, 48, dtype=I8), meta(40, dtype=F32),
                        meta(48, 21, dtype=I8), meta(48, dtype=F32)), ValueError),
    (lambda: ops.mlp_i8(meta(5, 48), meta(5, 48), meta(48), 1e-5, meta(40, 48), meta(40, dtype=F32),
                        meta(48, 20, dtype=I8), meta(48, dtype=F32)), TypeError),
    (lambda: ops.mlp_i8(meta(5, 48), meta(5, 48), meta(48), 1e-5, meta(40, 48, dtype=I8), meta(39, dtype=F32),
                        meta(48, 20, dtype=I8), meta(48, dtype=F32)), ValueError),
    (lambda: ops.rmsnorm_i8(meta(4, 8).requires_grad_(), meta(8), 1e-5), RuntimeError),
    (lambda: ops.silu_mul_i8(meta(4, 8), meta(4, 8).requires_grad_()), RuntimeError),
    # CPU tensors: there is no CPU implementation
    (lambda: ops.silu_mul_i8(torch.zeros(4, 8, dtype=BF16), torch.zeros(4, 8, dtype=BF16)), NotImplementedError),
])
def test_refusals(make, error):
    with pytest.raises(error):
        make()


def test_gradients_may_be_off():
    x = meta(4, 8).requires_grad_()
    with torch.no_grad():
        assert ops.rmsnorm_i8(x, meta(8), 1e-5)[0].shape == (4, 8)


def calls_with(x):
    """Every operator with `x` ([8, 16] bfloat16, meta) or its rows among the inputs."""
    a, w, f = meta(8, 16, dtype=I8), meta(4, 16, dtype=I8), lambda n: meta(n, dtype=F32)
    return [
        lambda: ops.rmsnorm_i8(x, meta(16), 1e-5)[1],
        lambda: ops.rmsnorm_i8(meta(3, 16), x[0], 1e-5)[1],
        lambda: ops.add_rmsnorm_i8(meta(8, 16), x, meta(16), 1e-5)[2],
        lambda: ops.silu_mul_i8(meta(8, 16), x)[1],
        lambda: ops.matmul_i8(a, w, x[:, 0].float(), f(4)),
        lambda: ops.matmul_i8(a, w, f(8), x[0, :4].float()),
        lambda: ops.matmul_i8(a, w, f(8), f(4), x[0, :4]),
        lambda: ops.mlp_i8(x, meta(8, 16), meta(16), 1e-5, meta(40, 16, dtype=I8), f(40), meta(16, 20, dtype=I8), f(16))[0],
        lambda: ops.mlp_i8(meta(8, 16), meta(8, 16), meta(16), 1e-5, meta(40, 16, dtype=I8), f(40),
                           meta(16, 20, dtype=I8), x[0].float())[0],
    ]


@pytest.mark.parametrize("which", range(9))
def test_derivatives_of_every_kind_are_refused(which):
    import torch.autograd.forward_ad as fwad
    x = meta(8, 16)
    with pytest.raises(RuntimeError, match="no backward"):
        calls_with(x.clone().requires_grad_())[which]()
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            calls_with(fwad.make_dual(x, meta(8, 16)))[which]()
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):  # it does not switch tangents off
            calls_with(fwad.make_dual(x, meta(8, 16)))[which]()
        calls_with(x)[which]()

    def total(v):
        return calls_with(v)[which]().float().sum()
    for transform in (torch.func.grad(total), torch.func.jacfwd(total), torch.func.jacrev(total),
                      lambda v: torch.func.jvp(total, (v,), (v,))):
        with pytest.raises(RuntimeError, match="no backward|tangent"):
            transform(x)
    with torch.no_grad():
        calls_with(x.clone().requires_grad_())[which]()
    with torch.inference_mode():
        calls_with(meta(8, 16))[which]()
    assert torch.func.vmap(lambda v: ops.silu_mul_i8(v, v)[1], in_dims=1)(meta(8, 3, 16)).shape == (3, 8)


def test_a_single_row_has_no_stride():
    """Its address alone says whether it needs a copy, whatever the stride given with it."""
    assert i8.gemm_workspace(1, 8, 33, P, 33, P, 48) == 0
    assert i8.gemm_workspace(4, 1, 33, P, 48, P, 33) == 0
    assert i8.gemm_workspace(1, 1, 33, P, 33, P, 35) == 0
    assert i8.gemm_workspace(1, 8, 33, P + 1, 48, P, 48) == 128 and i8.gemm_workspace(4, 1, 33, P, 48, P + 8, 48) == 128
    assert i8.gemm_workspace(2, 8, 33, P, 33, P, 48) == 2 * 128
    assert i8.mlp_workspace(3, 1, 65, P, 16, P, 65) == i8.mlp_workspace(3, 1, 65, P, 16, P, 80)


@pytest.mark.parametrize("N,K", [(64, 0), (64, 128), (1, 4096), (4096, 16)])
def test_plans_of_the_largest_sizes(N, K):
    """As many tokens as the calls accept are planned as their neighbours are."""
    most = 2 ** 31 - 2 ** 20
    for M in (2 ** 30 - 1, 2 ** 30, most):
        p, q = i8.gemm_plan(M, N, K), i8.gemm_plan(2 ** 29, N, K)
        assert (p["kernel"], p["tile_m"], p["tile_n"], p["splits"]) == (q["kernel"], q["tile_m"], q["tile_n"], q["splits"])
        assert p["tiles"] == -(-M // p["tile_m"]) * -(-N // p["tile_n"])
    for M in (1, 300):
        p = i8.gemm_plan(M, most, K)
        assert p["tiles"] == -(-M // p["tile_m"]) * -(-most // p["tile_n"])


@pytest.mark.parametrize("n,refused", [(2 ** 31 - 2 ** 20, False), (2 ** 31 - 2 ** 20 + 1, True), (2 ** 32 + 4, True)])
def test_sizes_that_the_gpu_refuses_are_refused_as_fakes(n, refused):
    calls = [lambda: ops.matmul_i8(meta(n, 16, dtype=I8), meta(4, 16, dtype=I8), meta(n, dtype=F32), meta(4, dtype=F32)),
             lambda: ops.matmul_i8(meta(4, 16, dtype=I8), meta(n, 16, dtype=I8), meta(4, dtype=F32), meta(n, dtype=F32)),
             lambda: ops.rmsnorm_i8(meta(n, 8), meta(8), 1e-5), lambda: ops.rmsnorm_i8(meta(2, n), meta(n), 1e-5),
             lambda: ops.add_rmsnorm_i8(meta(n, 8), meta(n, 8), meta(8), 1e-5),
             lambda: ops.silu_mul_i8(meta(n, 8), meta(n, 8)),
             lambda: ops.mlp_i8(meta(n, 48), meta(n, 48), meta(48), 1e-5, meta(40, 48, dtype=I8), meta(40, dtype=F32),
                                meta(48, 20, dtype=I8), meta(48, dtype=F32))]
    for call in calls:
        if refused:
            with pytest.raises(ValueError, match="size"):
                call()
        else:
            call()
