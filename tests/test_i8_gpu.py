"""The 8-bit operators on the GPU against their definitions in 64 bits.

Tolerances. A product's sum is a whole number, exact; its conversion to float,
two scalings and the bias round four times (4 * 2^-24 of the values they
round, 5 taken), and the store rounds by half a step of the output type (an
output below the normal range: by half the smallest step). Codes are compared
for equality. A norm's scale takes the sum of the squares in float: at most 40
roundings in a thread's chain at these lengths, 5 in its warp, 32 across the
block, halved by the root, then one: (77 / 2 + 1) * 2^-24. An activation's
scale is rounded once."""
import threading

import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# half the distance of neighbours below the normal range
TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}


@pytest.fixture(scope="module")
def ops(request):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import aegis_torch  # noqa: F401
    yield torch.ops.aegis
    torch.cuda.empty_cache()  # the largest tests take some 15 GB


def gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(torch, g, rows, cols, pad=0, offset=0, lo=-128):
    """Random codes, rows cols + pad apart, starting `offset` bytes into an allocation."""
    buf = torch.randint(lo, 128, (rows * (cols + pad) + offset,), device="cuda", generator=g, dtype=torch.int8)
    return buf[offset:].view(rows, cols + pad)[:, :cols]


def product(torch, a, w, sa, sw, bias=None):
    """(exact, sum of the magnitudes that were rounded) in 64 bits."""
    p = (a.double() @ w.double().t()) * sa.double()[:, None] * sw.double()[None, :]
    mag = p.abs()
    if bias is not None:
        p = p + bias.double()
        mag = mag + bias.double().abs()
    return p, mag


def assert_product(torch, c, a, w, sa, sw, bias=None):
    name = str(c.dtype).split(".")[1]
    exact, mag = product(torch, a, w, sa, sw, bias)
    tol = HALF[name] * exact.abs() * (1 + 2.0 ** -10) + 5 * 2.0 ** -24 * mag + TINY[name]
    off = (c.double() - exact).abs() - tol
    assert off.max().item() <= 0, f"{name} {tuple(a.shape)} x {tuple(w.shape)}: off by {off.max().item()} more than allowed"


def make(torch, seed, M, N, K, pad=0, offset=0, bias=None, lo=-128):
    g = gen(torch, seed)
    a, w = codes(torch, g, M, K, pad, offset, lo), codes(torch, g, N, K, pad, offset, lo)
    sa = torch.rand(M, device="cuda", generator=g) * 0.02 + 1e-3
    sw = torch.rand(N, device="cuda", generator=g) * 0.02 + 1e-3
    b = torch.randn(N, device="cuda", generator=g).to(bias) if bias is not None else None
    return a, w, sa, sw, b


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (2, 129, 256), (7, 1000, 4864), (16, 14336, 896), (17, 333, 384),
          (33, 257, 512), (64, 4096, 1024), (65, 640, 2048), (100, 130, 128), (128, 896, 896), (129, 300, 2048),
          (200, 4096, 1024), (256, 512, 4096), (300, 1024, 640), (513, 770, 1152), (1024, 2048, 512),
          (2000, 2500, 272), (4096, 1024, 16)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("out,bias", [("bfloat16", False), ("float16", True), ("float32", True)])
def test_product_tma_rows(ops, M, N, K, out, bias):
    import torch
    dt = getattr(torch, out)
    pad = -K % 16
    a, w, sa, sw, b = make(torch, M + N + K, M, N, K, pad, 0, dt if bias else None)
    c = ops.matmul_i8(a, w, sa, sw, b, out_dtype=dt)
    assert c.shape == (M, N) and c.dtype == dt
    assert_product(torch, c, a, w, sa, sw, b)
    assert torch.equal(c, ops.matmul_i8(a, w, sa, sw, b, out_dtype=dt))


@pytest.mark.parametrize("M,N,K,pad,offset", [(1, 1, 1, 0, 1), (1, 130, 15, 0, 0), (1, 4096, 4095, 0, 0),
                                              (3, 100, 17, 3, 5), (16, 1000, 777, 0, 0), (20, 129, 129, 2, 3),
                                              (50, 300, 1001, 0, 7), (77, 1000, 777, 0, 0), (130, 257, 255, 1, 2),
                                              (300, 333, 500, 4, 4), (600, 1025, 1111, 0, 1), (64, 128, 256, 0, 8)])
@pytest.mark.parametrize("out", ["bfloat16", "float32"])
def test_product_any_alignment(ops, M, N, K, pad, offset, out):
    import torch
    dt = getattr(torch, out)
    a, w, sa, sw, b = make(torch, 3 * M + N + K, M, N, K, pad, offset, dt)
    c = ops.matmul_i8(a, w, sa, sw, b, out_dtype=dt)
    assert_product(torch, c, a, w, sa, sw, b)
    # The same codes in rows that TMA can read, alone and beside misaligned ones: the same bits.
    p = -K % 16
    a2, w2 = (torch.nn.functional.pad(t, (0, p))[:, :K] for t in (a, w))
    assert torch.equal(c, ops.matmul_i8(a2, w2, sa, sw, b, out_dtype=dt))
    assert torch.equal(c, ops.matmul_i8(a2, w, sa, sw, b, out_dtype=dt))
    assert torch.equal(c, ops.matmul_i8(a, w2, sa, sw, b, out_dtype=dt))


@pytest.mark.parametrize("M,N,K,aligned", [(1, 128, 131071, False), (2, 64, 131056, True), (300, 256, 131056, True)])
@pytest.mark.parametrize("sign", [1, -1])
def test_longest_sums_do_not_overflow(ops, M, N, K, aligned, sign):
    import torch
    a = torch.full((M, K), -128, device="cuda", dtype=torch.int8)
    w = torch.full((N, K), -128 if sign > 0 else 127, device="cuda", dtype=torch.int8)
    one = torch.ones(max(M, N), device="cuda")
    c = ops.matmul_i8(a, w, one[:M], one[:N], out_dtype=torch.float32)
    want = float(K * 128 * (128 if sign > 0 else -127))
    assert (c.double() - want).abs().max().item() <= 2.0 ** -24 * abs(want)


def test_empty_sums_and_sizes(ops):
    import torch
    one = torch.ones(8, device="cuda")
    e = torch.empty(8, 0, device="cuda", dtype=torch.int8)
    bias = torch.arange(8, device="cuda", dtype=torch.float32)
    assert torch.equal(ops.matmul_i8(e, e, one, one, bias), bias.expand(8, 8))
    assert torch.equal(ops.matmul_i8(e, e, one, one, out_dtype=torch.float16), torch.zeros(8, 8, device="cuda").half())
    z = torch.empty(0, 16, device="cuda", dtype=torch.int8)
    k = torch.ones(8, 16, device="cuda", dtype=torch.int8)
    assert ops.matmul_i8(z, k, one[:0], one).shape == (0, 8)
    assert ops.matmul_i8(k, z, one, one[:0]).shape == (8, 0)
    for q, s in (ops.rmsnorm_i8(torch.empty(0, 16, device="cuda").half(), torch.ones(16, device="cuda").half(), 0.0),
                 ops.silu_mul_i8(torch.empty(0, 16, device="cuda").half(), torch.empty(0, 16, device="cuda").half())):
        assert q.shape == (0, 16) and s.shape == (0,)


@pytest.mark.parametrize("M,N,ldc,out", [(3, 130, 140, 1), (300, 700, 701, 0), (600, 512, 520, 2), (17, 64, 96, 2)])
def test_product_leaves_what_is_between_the_rows(ops, M, N, ldc, out):
    import torch
    import aegis_i8 as i8
    dt = {0: torch.float16, 1: torch.bfloat16, 2: torch.float32}[out]
    a, w, sa, sw, b = make(torch, 5, M, N, 256, 0, 0, dt)
    c = torch.full((M + 2, ldc), 7.0, device="cuda", dtype=dt)
    st = i8.load().aegis_i8_gemm(0, torch.cuda.current_stream().cuda_stream, out, M, N, 256, a.data_ptr(), 256,
                                 w.data_ptr(), 256, sa.data_ptr(), sw.data_ptr(), b.data_ptr(),
                                 c.data_ptr() + ldc * c.element_size(), ldc, None, 0)
    assert st == 0
    assert torch.equal(c[1:-1, :N], ops.matmul_i8(a, w, sa, sw, b, out_dtype=dt))
    c[1:-1, :N] = 7.0
    assert (c == 7.0).all()


def test_strides_of_every_kind(ops):
    """Rows of a larger tensor are read in place; other patterns are copied; vectors may be strided."""
    import torch
    a, w, sa, sw, b = make(torch, 21, 33, 130, 200, 0, 0, torch.bfloat16)
    want = ops.matmul_i8(a, w, sa, sw, b)
    wide = torch.zeros(33, 512, device="cuda", dtype=torch.int8)
    wide[:, 16:216], wide[:, 300:500] = a, a
    every2 = torch.zeros(260, 400, device="cuda", dtype=torch.int8)
    every2[::2, ::2] = w
    strided = torch.zeros(130, 3, device="cuda")
    strided[:, 1] = sw
    for x in (wide[:, 16:216], wide[:, 300:500], a.t().contiguous().t()):
        for y in (w, w.t().contiguous().t(), every2[::2, ::2]):
            assert torch.equal(ops.matmul_i8(x, y, sa, strided[:, 1], b), want)
    row = a[:1].expand(33, 200)
    assert torch.equal(ops.matmul_i8(row, w, sa[:1].expand(33), sw, b),
                       ops.matmul_i8(a[:1], w, sa[:1], sw, b).expand(33, 130))
    x = torch.randn(40, 64, device="cuda").half()
    g = torch.randn(64, 2, device="cuda").half()
    q, s, h = ops.add_rmsnorm_i8(x.t(), x.t().contiguous(), g[:40, 0], 1e-5)
    q2, s2, h2 = ops.add_rmsnorm_i8(x.t().contiguous(), x.t().contiguous(), g[:40, 0].contiguous(), 1e-5)
    assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(h, h2)


@pytest.mark.parametrize("M,N,ldc,offset", [(1100, 4099, 4099, 0), (1100, 4099, 4100, 3), (1030, 6401, 6403, 1),
                                            (1100, 4099, 4101, 5), (1100, 4352, 4353, 7), (1100, 4352, 4368, 8),
                                            (1300, 4133, 4144, 0), (1030, 6401, 6402, 2)])
@pytest.mark.parametrize("out", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("bias", [True, False])
def test_large_products_into_rows_of_any_alignment(ops, M, N, ldc, offset, out, bias):
    import torch
    import aegis_i8 as i8
    assert i8.gemm_plan(M, N, 512)["kernel"] == "pair"
    dt = getattr(torch, out)
    a, w, sa, sw, b = make(torch, M + N, M, N, 512, 0, 0, dt if bias else None)
    buf = torch.full((offset + (M + 1) * ldc,), 7.0, device="cuda", dtype=dt)
    st = i8.load().aegis_i8_gemm(0, torch.cuda.current_stream().cuda_stream, {"float16": 0, "bfloat16": 1, "float32": 2}[out],
                                 M, N, 512, a.data_ptr(), 512, w.data_ptr(), 512, sa.data_ptr(), sw.data_ptr(),
                                 b.data_ptr() if bias else None, buf.data_ptr() + offset * buf.element_size(), ldc, None, 0)
    assert st == 0
    c = buf[offset:].view(M + 1, ldc)
    assert_product(torch, c[:M, :N], a, w, sa, sw, b)
    c[:M, :N] = 7.0
    assert (buf == 7.0).all()


def test_product_scales_that_are_not_finite(ops):
    import torch
    a, w, sa, sw, _ = make(torch, 9, 20, 40, 128)
    sa[3], sw[5] = float("nan"), float("inf")
    c = ops.matmul_i8(a, w, sa, sw)
    assert c[3].isnan().all() and not c[:, :5][torch.arange(20, device="cuda") != 3].isnan().any()
    assert c[4, 5].isinf()


# ---------------------------------------------------------------- row operations
def check_codes(torch, q, t):
    """q against 127 t / max |t| of the rows of t (64 bits), to the nearest whole number."""
    m = t.abs().amax(dim=1, keepdim=True)
    want = torch.where(m > 0, torch.round(127.0 * t / m), torch.zeros_like(t))
    assert torch.equal(q.double(), want), f"{(q.double() != want).sum().item()} codes differ"
    return m[:, 0]


def check_norm(torch, q, s, h, w, eps):
    hd = h.double()
    m = check_codes(torch, q, hd * w.double())
    want = m / torch.sqrt(hd.square().mean(dim=1) + eps) / 127.0
    assert ((s.double() - want).abs() <= (77 / 2 + 1) * 2.0 ** -24 * want).all()


ROWS = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 1000), (4, 1024), (3, 1025), (2, 2048), (5, 4096), (3, 4097), (2, 8192),
        (2, 14336), (2, 16385), (1, 28672), (3, 32768), (2, 32769), (2, 40001), (700, 896),
        # more rows than blocks
        (9000, 100), (4800, 1031), (2500, 4096), (700, 3001), (700, 4105), (700, 9000), (400, 17000)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 1)])
def test_norm(ops, dtype, rows, cols, pad, offset):
    import torch
    dt = getattr(torch, dtype)
    g = gen(torch, rows * 31 + cols)

    def stream():
        buf = torch.randn(rows * (cols + pad) + offset, device="cuda", generator=g) * 3
        return buf.to(dt)[offset:].view(rows, cols + pad)[:, :cols]
    x, r = stream(), stream()
    w = (torch.randn(cols + offset, device="cuda", generator=g) + 1).to(dt)[offset:]
    q, s = ops.rmsnorm_i8(x, w, 1e-5)
    check_norm(torch, q, s, x, w, 1e-5)
    q, s, h = ops.add_rmsnorm_i8(x, r, w, 1e-6)
    assert torch.equal(h, (x.float() + r.float()).to(dt))
    check_norm(torch, q, s, h, w, 1e-6)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("halves", [True, False])
def test_silu_mul(ops, dtype, rows, cols, halves):
    import torch
    dt = getattr(torch, dtype)
    g = gen(torch, rows * 37 + cols)
    gu = (torch.randn(rows, 2 * cols, device="cuda", generator=g) * 2).to(dt)
    gate, up = (gu[:, :cols], gu[:, cols:]) if halves else (gu[:, :cols].contiguous(), gu[:, cols:].contiguous())
    q, s = ops.silu_mul_i8(gate, up)
    gd = gate.double()
    m = check_codes(torch, q, gd / (1 + torch.exp(-gd)) * up.double())
    assert ((s.double() - m / 127).abs() <= 2.0 ** -24 * m / 127 * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("cols", [40, 4096, 40000])
def test_codes_at_the_borders(ops, cols):
    """Values that lie exactly between two codes go to the even one."""
    import torch
    half = (torch.arange(cols, device="cuda") % 254 - 127).double() + 0.5  # -126.5 .. 126.5
    x = half.clone()
    x[-1] = 127.0
    x = x.bfloat16()  # 8 bits hold n + 1/2 up to 64; above, the neighbours are whole
    w = torch.ones(cols, device="cuda").bfloat16()
    q, s = ops.rmsnorm_i8(x[None], w, 0.0)
    check_norm(torch, q, s, x[None], w, 0.0)
    x = half.half()
    x[-1] = 127.0
    q, s = ops.rmsnorm_i8(x[None], w.half(), 0.0)
    check_norm(torch, q, s, x[None], w.half(), 0.0)
    # One gate, so t is up times a constant, rounded to 64 bits: that rounding puts
    # 127 t / m on one side of the border or the other, and the codes follow it.
    g, u = torch.ones(2, cols, device="cuda").half(), x.expand(2, cols).contiguous()
    q, s = ops.silu_mul_i8(g, u)
    check_codes(torch, q, g.double() / (1 + torch.exp(-g.double())) * u.double())


@pytest.mark.parametrize("cols", [64, 4097, 40000])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_rows_that_are_zero_or_not_finite(ops, dtype, cols):
    zero_or_not_finite(ops, dtype, cols, 8)


@pytest.mark.parametrize("rows,cols", [(6000, 64), (5000, 1024), (3000, 4096), (800, 12000)])
def test_zero_and_not_finite_rows_among_many(ops, rows, cols):
    zero_or_not_finite(ops, "bfloat16", cols, rows)


def zero_or_not_finite(ops, dtype, cols, rows):
    import torch
    dt = getattr(torch, dtype)
    g = gen(torch, cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dt)
    w = torch.ones(cols, device="cuda").to(dt)
    w[0] = 0
    x[1::8] = 0
    x[2::8, cols // 2] = float("nan")
    x[3::8, cols - 1] = float("inf")
    x[4::8, 0] = -float("inf")  # times a weight of 0
    kind = torch.arange(rows, device="cuda") % 8
    for q, s in (ops.rmsnorm_i8(x, w, 1e-5), ops.silu_mul_i8(x, torch.ones_like(x)),
                 ops.silu_mul_i8(torch.ones_like(x), x), ops.add_rmsnorm_i8(x, torch.zeros_like(x), w, 1e-5)[:2]):
        assert (q[kind == 1] == 0).all() and (s[kind == 1] == 0).all()
        bad = (kind >= 2) & (kind <= 4)
        assert (q[bad] == 0).all() and s[bad].isnan().all()
        rest = (kind == 0) | (kind >= 5)
        assert s[rest].isfinite().all() and (q[rest].abs().amax(dim=1) == 127).all()
    q, s = ops.silu_mul_i8(x, torch.ones_like(x))
    xd = x[rest].double()
    check_codes(torch, q[rest], xd / (1 + torch.exp(-xd)))
    q, s = ops.rmsnorm_i8(x, w, 1e-5)
    check_norm(torch, q[rest], s[rest], x[rest], w, 1e-5)
    big = torch.full((1, cols), 6e4, device="cuda").half()  # the sum leaves f16's range
    q, s, h = ops.add_rmsnorm_i8(big, big, torch.ones(cols, device="cuda").half(), 1e-5)
    assert h.isinf().all() and s.isnan().all() and (q == 0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", [(7, 72), (7, 1001), (7, 40000), (3000, 64), (700, 12000)])
def test_not_finite_next_to_zero(ops, dtype, rows, cols):
    """NaN and infinity in one half do not vanish where the other half is 0."""
    import torch
    dt = getattr(torch, dtype)
    g = gen(torch, rows + cols)
    gate, up = (torch.randn(rows, cols, device="cuda", generator=g).to(dt) for _ in range(2))
    nan, inf = float("nan"), float("inf")
    for i, (a, b) in enumerate([(nan, 0), (inf, 0), (-inf, 0), (0, inf), (0, nan), (-0.0, -inf), (0, 0)]):
        gate[i::7, (5 * i) % cols], up[i::7, (5 * i) % cols] = a, b
    q, s = ops.silu_mul_i8(gate, up)
    gd = gate.double()
    t = gd / (1 + torch.exp(-gd)) * up.double()
    bad = t.isnan().any(dim=1)
    assert bad.sum() == rows - rows // 7
    assert torch.equal(s.isnan(), bad) and (q[bad] == 0).all()
    check_codes(torch, q[~bad], t[~bad])


@pytest.mark.parametrize("cols", [100, 4096, 40000])
@pytest.mark.parametrize("size", [1e30, 1e19, 1e-15, 1e-22, 1e-30, 1e-36])
def test_norm_of_very_large_and_small_rows(ops, cols, size):
    """Squares leave float's range at 1e19 and below 1e-22; bf16 values do not."""
    import torch
    x = (torch.randn(3, cols, device="cuda", generator=gen(torch, cols)) * size).bfloat16()
    w = (torch.randn(cols, device="cuda", generator=gen(torch, 1)) + 1).bfloat16()
    q, s = ops.rmsnorm_i8(x, w, 0.0)
    check_norm(torch, q, s, x, w, 0.0)


@pytest.mark.parametrize("rows,cols", [(8, 72), (8, 4097), (8, 40000), (2400, 1000), (700, 12000)])
def test_silu_where_gate_times_up_leaves_the_range(ops, rows, cols):
    """bf16: gate * up above float's range with a finite result, far below it, and subnormal gates."""
    import torch
    g = gen(torch, rows + cols)
    gate, up = (torch.randn(rows, cols, device="cuda", generator=g) for _ in range(2))
    gate[0::4, 3], up[0::4, 3] = -70.0, 2.0 ** 127
    gate[1::4, cols - 1], up[1::4, cols - 1] = 3e38, 2.0  # the result itself is beyond it
    gate[2::4] *= 1e-25
    up[2::4] *= 1e-25
    gate[2::4, 5], up[2::4, 5] = 1e-10, 1e-5
    gate[3::4] *= 1e-39
    up[3::4] *= 1e35
    gate, up = gate.bfloat16(), up.bfloat16()
    q, s = ops.silu_mul_i8(gate, up)
    gd = gate.double()
    t = gd / (1 + torch.exp(-gd)) * up.double()
    beyond = torch.arange(rows, device="cuda") % 4 == 1
    assert s[beyond].isnan().all() and (q[beyond] == 0).all()
    m = check_codes(torch, q[~beyond], t[~beyond])
    assert ((s[~beyond].double() - m / 127).abs() <= 2.0 ** -24 * m / 127 * (1 + 2.0 ** -20)).all()


def test_silu_of_rows_below_the_range_of_exp(ops):
    import torch
    g = torch.full((2, 300), -95.0, device="cuda").bfloat16()
    g[1] = torch.linspace(-100, -90, 300, device="cuda").bfloat16()
    u = torch.linspace(-3, 3, 300, device="cuda").bfloat16().expand(2, 300).contiguous()
    q, s = ops.silu_mul_i8(g, u)
    gd = g.double()
    m = check_codes(torch, q, gd / (1 + torch.exp(-gd)) * u.double())
    assert ((s.double() - m / 127).abs() <= 2.0 ** -150).all()  # below the normal range: half the smallest step


@pytest.mark.parametrize("cols", [1000, 4096, 40001])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_norm_in_place(ops, cols, place):
    """The C call may put h where x or the residual was; what lies between rows stays."""
    import torch
    import aegis_i8 as i8
    g = gen(torch, cols)
    x, r = (torch.randn(5, cols + 5, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = torch.ones(cols, device="cuda").bfloat16()
    q0, s0, h0 = ops.add_rmsnorm_i8(x[:, :cols], r[:, :cols], w, 1e-5)
    q = torch.full((5, cols + 3), 99, device="cuda", dtype=torch.int8)
    s = torch.empty(5, device="cuda")
    h = x if place == "x" else r
    edge = h[:, cols:].clone()
    st = i8.load().aegis_i8_rmsnorm(0, torch.cuda.current_stream().cuda_stream, 1, 5, cols, x.data_ptr(), cols + 5,
                                    r.data_ptr(), cols + 5, w.data_ptr(), 1e-5, h.data_ptr(), cols + 5, q.data_ptr(),
                                    cols + 3, s.data_ptr())
    assert st == 0
    assert torch.equal(q[:, :cols], q0) and torch.equal(s, s0) and torch.equal(h[:, :cols], h0)
    assert (q[:, cols:] == 99).all() and torch.equal(h[:, cols:], edge)


# ---------------------------------------------------------------- offsets beyond 32 bits
def test_product_with_an_output_beyond_2_31_elements(ops):
    import torch
    M, N, K = 70001, 32771, 48
    a, w, sa, sw, _ = make(torch, 31, M, N, K)
    c = ops.matmul_i8(a, w, sa, sw)
    rows = torch.tensor([0, 1, 32768, 65535, 65537, M - 2, M - 1], device="cuda")
    assert_product(torch, c[rows], a[rows], w, sa[rows], sw)
    cols = torch.tensor([0, 32767, N - 1], device="cuda")
    assert_product(torch, c[:, cols], a, w[cols], sa, sw[cols])


@pytest.mark.parametrize("cols", [16392, 16391])
def test_rows_beyond_2_31_elements(ops, cols):
    import torch
    rows = 140000
    g = gen(torch, cols)
    x = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    x[:1000] = torch.randn(1000, cols, device="cuda", generator=g).bfloat16()
    for i in range(1000, rows, 1000):
        x[i:i + 1000] = x[:1000]
    w = (torch.randn(cols, device="cuda", generator=g) + 1).bfloat16()
    pick = torch.tensor([0, 999, 131000, 131072, rows - 1], device="cuda")
    q, s, h = ops.add_rmsnorm_i8(x, x, w, 1e-5)
    assert torch.equal(h[pick], x[pick] * 2)
    check_norm(torch, q[pick], s[pick], h[pick], w, 1e-5)
    assert torch.equal(q[rows - 1000:], q[:1000]) and torch.equal(s[rows - 1000:], s[:1000])
    del q, s, h
    q, s = ops.silu_mul_i8(x, x)
    xd = x[pick].double()
    check_codes(torch, q[pick], xd / (1 + torch.exp(-xd)) * xd)
    assert torch.equal(q[rows - 1000:], q[:1000])


def test_codes_of_a_matrix_beyond_2_31_bytes(ops):
    import torch
    K, N = 4096, 530001
    w = torch.empty(N, K, device="cuda", dtype=torch.int8)
    w[:1000] = torch.randint(-128, 128, (1000, K), device="cuda", generator=gen(torch, 3), dtype=torch.int8)
    for i in range(1000, N, 1000):
        w[i:i + 1000] = w[:min(1000, N - i)]
    sw = torch.rand(N, device="cuda") * 0.01 + 1e-3
    pick = torch.tensor([0, 524287, 524288, N - 1], device="cuda")
    for M in (1, 16):
        a, _, sa, _, _ = make(torch, M, M, 8, K)
        assert_product(torch, ops.matmul_i8(a, w, sa, sw)[:, pick], a, w[pick], sa, sw[pick])
    a, _, sa, _, _ = make(torch, 5, 3, 8, K - 1)
    assert_product(torch, ops.matmul_i8(a, w[:, 1:], sa, sw)[:, pick], a, w[pick, 1:], sa, sw[pick])


# ---------------------------------------------------------------- the block
def block(torch, seed, M, K, F, dt, w_pad=0):
    g = gen(torch, seed)
    x, r = (torch.randn(M, K, device="cuda", generator=g).to(dt) for _ in range(2))
    nw = (torch.randn(K, device="cuda", generator=g) * 0.2 + 1).to(dt)
    w1, w2 = codes(torch, g, 2 * F, K, w_pad), codes(torch, g, K, F, w_pad)
    s1 = (torch.rand(2 * F, device="cuda", generator=g) + 0.5) / (74 * K ** 0.5)
    s2 = (torch.rand(K, device="cuda", generator=g) + 0.5) / (74 * F ** 0.5)
    return x, r, nw, 1e-5, w1, s1, w2, s2


def composed(torch, ops, x, r, nw, eps, w1, s1, w2, s2):
    F = w2.shape[1]
    q, s, h = ops.add_rmsnorm_i8(x, r, nw, eps)
    gu = ops.matmul_i8(q, w1, s, s1, out_dtype=x.dtype)
    q, s = ops.silu_mul_i8(gu[:, :F], gu[:, F:])
    return ops.matmul_i8(q, w2, s, s2, out_dtype=x.dtype), h, q, s


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("M,K,F,pad", [(1, 896, 4864, 0), (1, 1, 1, 0), (7, 896, 4864, 0), (16, 4096, 1024, 0),
                                       (33, 257, 333, 0), (33, 257, 333, 15), (130, 640, 1000, 8),
                                       (600, 1024, 2048, 0), (1, 4096, 14336, 0)])
def test_block_equals_its_parts(ops, dtype, M, K, F, pad):
    import torch
    b = block(torch, M + K + F, M, K, F, getattr(torch, dtype), pad)
    y, h = ops.mlp_i8(*b)
    y2, h2, q, s = composed(torch, ops, *b)
    assert torch.equal(h, h2) and torch.equal(y, y2)
    assert_product(torch, y, q, b[6], s, b[7])


def test_block_repeats_and_overlaps(ops):
    """Back-to-back calls, two threads on two streams, and replays of a captured graph give the same bits."""
    import torch
    b = block(torch, 1, 4, 2048, 4096, torch.bfloat16)
    c = block(torch, 2, 64, 2048, 4096, torch.bfloat16)
    want_b, want_c = ops.mlp_i8(*b)[0], ops.mlp_i8(*c)[0]
    for _ in range(20):
        got = [ops.mlp_i8(*b)[0], ops.mlp_i8(*c)[0]]
    assert torch.equal(got[0], want_b) and torch.equal(got[1], want_c)
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(name, args):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(30):
                    y = ops.mlp_i8(*args)[0]
                results[name] = y.clone()
            st.synchronize()
        except Exception as e:  # reported by the main thread
            errors.append(e)
    ts = [threading.Thread(target=work, args=("b", b)), threading.Thread(target=work, args=("c", c))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors
    assert torch.equal(results["b"], want_b) and torch.equal(results["c"], want_c)


def test_captured_graphs(ops):
    """Two graphs captured on one stream and replayed on two at once do not share anything; new inputs are seen."""
    import torch
    b = block(torch, 3, 1, 1024, 2048, torch.float16)
    c = block(torch, 4, 40, 1024, 2048, torch.float16)
    ops.mlp_i8(*b), ops.mlp_i8(*c)
    torch.cuda.synchronize()
    graphs = []
    for args in (b, c):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, h = ops.mlp_i8(*args)
        graphs.append((g, y, h))
    fresh = [block(torch, 5, 1, 1024, 2048, torch.float16), block(torch, 6, 40, 1024, 2048, torch.float16)]
    want = [ops.mlp_i8(f[0], f[1], *a[2:]) for f, a in zip(fresh, (b, c))]
    for f, a in zip(fresh, (b, c)):
        a[0].copy_(f[0])
        a[1].copy_(f[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for st, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (g, y, h), (wy, wh) in zip(graphs, want):
        assert torch.equal(y, wy) and torch.equal(h, wh)


def test_weights_written_just_before_the_call(ops):
    """The block starts to read its weights early: not before the kernels that write them have ended."""
    import torch
    b = list(block(torch, 7, 2, 1024, 4096, torch.bfloat16))
    w1, w2 = b[4].clone(), b[6].clone()
    want = ops.mlp_i8(*b)[0]
    filler = torch.empty(1 << 26, device="cuda")
    for _ in range(10):
        b[4].zero_(), b[6].zero_()
        ops.mlp_i8(*b)
        filler.fill_(1.0)
        b[4].copy_(w1)
        b[6].copy_(w2)
        assert torch.equal(ops.mlp_i8(*b)[0], want)


def test_no_watchdog_fired(ops):
    import torch
    import aegis_i8 as i8
    i8.synchronize(0, torch.cuda.current_stream().cuda_stream)


def test_gradients_are_refused(ops):
    import torch
    x = torch.randn(2, 64, device="cuda").half().requires_grad_()
    w = torch.ones(64, device="cuda").half()
    with pytest.raises(RuntimeError, match="no backward"):
        ops.rmsnorm_i8(x, w, 1e-5)
    with torch.no_grad():
        ops.rmsnorm_i8(x, w, 1e-5)
    a, wq, sa, sw, _ = make(torch, 1, 2, 8, 16)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.matmul_i8(a, wq, sa.requires_grad_(), sw)
    with pytest.raises(ValueError, match="different devices"):
        ops.matmul_i8(a, wq, sa.detach(), sw.cpu())
