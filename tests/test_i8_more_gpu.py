"""Calls of the 8-bit operators that their documents allow and that reach code of their own."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import aegis_torch  # noqa: F401
    yield torch.ops.aegis
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,N,K,lda,ldw", [(1, 4096, 777, 777, 784), (1, 300, 5001, 5001, 5008), (1, 64, 33, 1 << 40, 48),
                                           (40, 1, 777, 784, 777), (300, 1, 777, 784, 779), (1, 1, 100, 101, 103)])
def test_single_rows_with_any_stride_need_no_workspace(ops, M, N, K, lda, ldw):
    import torch
    import aegis_i8 as i8
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, w = (torch.randint(-128, 128, (r, (K + 15) // 16 * 16), device="cuda", generator=g, dtype=torch.int8) for r in (M, N))
    sa, sw = (torch.rand(n, device="cuda", generator=g) for n in (M, N))
    assert i8.gemm_workspace(M, N, K, a.data_ptr(), lda, w.data_ptr(), ldw) == 0
    c = torch.empty(M, N, device="cuda")
    st = i8.load().aegis_i8_gemm(0, torch.cuda.current_stream().cuda_stream, 2, M, N, K, a.data_ptr(), lda, w.data_ptr(),
                                 ldw, sa.data_ptr(), sw.data_ptr(), None, c.data_ptr(), N, None, 0)
    assert st == 0, i8.last_error_string()
    assert torch.equal(c, ops.matmul_i8(a[:, :K].contiguous(), w[:, :K].contiguous(), sa, sw, out_dtype=torch.float32))


# A shape for every way a row operation is launched (148 SMs): rows x columns, and whether rows start on 16-byte boundaries.
LAUNCHES = [
    # blocks that walk over many aligned rows, by threads a block
    (400, 2048, True), (3000, 4096, True), (400, 4104, True), (400, 5120, True), (1300, 6144, True), (700, 7168, True),
    (400, 7176, True), (400, 9216, True), (400, 12288, True), (300, 14336, True), (300, 16384, True), (300, 32768, True),
    # a block a row: many rows that are not aligned
    (700, 1024, False), (700, 2048, False), (700, 4096, False), (700, 8192, False), (700, 16384, False), (600, 32768, False),
    # fewer rows, aligned or not
    (16, 4096, True), (64, 4099, False), (16, 5120, True), (100, 8192, True), (9, 8192, False), (8, 8192, True),
    (5, 6144, False), (8, 16384, True), (9, 16384, True), (200, 9000, True), (20, 16383, False), (3, 20000, True),
    (30, 32767, False), (2, 40960, True), (300, 40961, False),
]


def rows_of(torch, g, rows, cols, aligned, dt, scale):
    pad, offset = (-cols % 8, 0) if aligned else (-cols % 8 + 3, 1)
    buf = (torch.randn(rows * (cols + pad) + offset, device="cuda", generator=g) * scale).to(dt)
    return buf[offset:].view(rows, cols + pad)[:, :cols]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols,aligned", LAUNCHES)
def test_every_launch_of_the_row_operations(ops, dtype, rows, cols, aligned):
    import torch
    from test_i8_exact_gpu import assert_scale
    from test_i8_gpu import check_codes
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, r = (rows_of(torch, g, rows, cols, aligned, dt, 2.0) for _ in range(2))
    w = (torch.randn(cols, device="cuda", generator=g) * 0.2 + 1).to(dt)
    w[0] = 0
    kind = torch.arange(rows, device="cuda") % 8  # rows of zeros and rows that are not finite, among the others
    x[1::8], r[1::8] = 0, 0
    x[3::8, cols // 2] = float("nan")
    x[5::8, cols - 1] = float("inf")
    bad, fine = (kind == 3) | (kind == 5), (kind != 3) & (kind != 5)
    some = fine & (kind != 1)

    def check(q, s, t):
        assert (q[bad] == 0).all() and s[bad].isnan().all() and (s[kind == 1] == 0).all()
        return check_codes(torch, q[fine], t[fine])

    q, s = ops.rmsnorm_i8(x, w, 1e-5)
    check(q, s, x.double() * w.double())
    assert_scale(torch, s[some], x[some], w, 1e-5)
    q, s, h = ops.add_rmsnorm_i8(x, r, w, 1e-6)
    assert torch.equal(h[fine], (x.float() + r.float()).to(dt)[fine])
    check(q, s, h.double() * w.double())
    assert_scale(torch, s[some], h[some], w, 1e-6)
    q, s = ops.silu_mul_i8(x, r)
    xd = x.double()
    m = check(q, s, xd / (1 + torch.exp(-xd)) * r.double())
    assert ((s[fine].double() - m / 127).abs() <= 2.0 ** -24 * m / 127 * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("M,K,F,kernels", [(16, 4095, 14335, "stream"), (40, 1023, 8191, "stream"), (2, 1023, 2047, "dot"),
                                           (300, 1023, 4095, "pair")])
def test_block_reads_the_weights_that_the_call_itself_copies(ops, M, K, F, kernels):
    """Unaligned weights are copied into the workspace by a kernel that lets its dependents start before it
    has written anything; the products ask for them before their own wait. What was in the workspace must
    not be seen."""
    import torch
    import aegis_i8 as i8
    plans = {i8.gemm_plan(M, 2 * F, K)["kernel"], i8.gemm_plan(M, K, F)["kernel"]}
    assert kernels in plans
    g = torch.Generator(device="cuda").manual_seed(M + K + F)
    x, r = (torch.randn(M, K, device="cuda", generator=g).bfloat16() for _ in range(2))
    nw = torch.ones(K, device="cuda").bfloat16()
    w1, w2 = (torch.randint(-127, 128, s, device="cuda", generator=g, dtype=torch.int8) for s in ((2 * F, K), (K, F)))
    s1 = (torch.rand(2 * F, device="cuda", generator=g) + 0.5) / (74 * K ** 0.5)
    s2 = (torch.rand(K, device="cuda", generator=g) + 0.5) / (74 * F ** 0.5)
    q, s, h_want = ops.add_rmsnorm_i8(x, r, nw, 1e-5)
    gu = ops.matmul_i8(q, w1, s, s1)
    q, s = ops.silu_mul_i8(gu[:, :F], gu[:, F:])
    want = ops.matmul_i8(q, w2, s, s2)
    n = i8.mlp_workspace(M, K, F, w1.data_ptr(), K, w2.data_ptr(), F)
    assert n > w1.numel() + w2.numel()  # both matrices are copied
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    stream = torch.cuda.current_stream().cuda_stream
    for i in range(20):
        ws.fill_(0x55 if i % 2 else 0x81)
        h, y = torch.empty_like(x), torch.empty_like(x)
        st = i8.load().aegis_i8_mlp(0, stream, 1, M, K, F, x.data_ptr(), K, r.data_ptr(), K, nw.data_ptr(), 1e-5,
                                    w1.data_ptr(), K, s1.data_ptr(), w2.data_ptr(), F, s2.data_ptr(), h.data_ptr(), K,
                                    y.data_ptr(), K, ws.data_ptr(), n)
        assert st == 0, i8.last_error_string()
        assert torch.equal(y, want) and torch.equal(h, h_want)


@pytest.mark.parametrize("M,K,F", [(1, 512, 1024), (20, 333, 1001)])
def test_block_in_place_through_the_c_call(ops, M, K, F):
    """h may stand in the place of x or of the residual, as in aegis_i8_rmsnorm; calls on another stream and thread agree."""
    import torch
    import aegis_i8 as i8
    g = torch.Generator(device="cuda").manual_seed(K)
    x, r = (torch.randn(M, K, device="cuda", generator=g).half() for _ in range(2))
    nw = torch.ones(K, device="cuda").half()
    w1, w2 = (torch.randint(-127, 128, s, device="cuda", generator=g, dtype=torch.int8) for s in ((2 * F, K), (K, F)))
    s1, s2 = torch.full((2 * F,), 1e-3, device="cuda"), torch.full((K,), 1e-3, device="cuda")
    want, h_want = ops.mlp_i8(x, r, nw, 1e-5, w1, s1, w2, s2)
    n = i8.mlp_workspace(M, K, F, w1.data_ptr(), K, w2.data_ptr(), F)
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    side = torch.cuda.Stream()
    for place in (0, 1):
        xs = [x.clone(), r.clone()]
        y = torch.empty_like(x)
        side.wait_stream(torch.cuda.current_stream())
        st = i8.load().aegis_i8_mlp(0, side.cuda_stream, 0, M, K, F, xs[0].data_ptr(), K, xs[1].data_ptr(), K,
                                    nw.data_ptr(), 1e-5, w1.data_ptr(), K, s1.data_ptr(), w2.data_ptr(), F, s2.data_ptr(),
                                    xs[place].data_ptr(), K, y.data_ptr(), K, ws.data_ptr(), n)
        assert st == 0
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, want) and torch.equal(xs[place], h_want)
        assert torch.equal(xs[1 - place], (x, r)[1 - place])
