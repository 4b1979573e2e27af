"""Products whose scales are near the ends of float's range.

a_scale * w_scale * sum is in range although the sum times one scale is not. Tolerance:
the sum's conversion, two multiplications and the bias's addition round once each
(4 * 2^-24 of what they round, 5 taken), the store by half a step of its type; below
float's normal range by half its smallest step too (2^-150)."""
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}


@pytest.fixture(scope="module")
def ops():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import aegis_torch  # noqa: F401
    return torch.ops.aegis


# One of every kernel and way to store: dot, stream with and without slices, pairs into aligned and odd rows.
SHAPES = [(1, 300, 1024, "dot"), (7, 130, 777, "dot"), (16, 512, 4096, "stream"), (40, 20000, 128, "stream"),
          (300, 4096, 640, "stream"), (1100, 4352, 512, "pair"), (700, 4099, 384, "pair")]


@pytest.mark.parametrize("M,N,K,kernel", SHAPES)
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("ea,ew", [(100, -100), (126, -126), (126, -148), (96, -90), (97, -90), (-100, 90), (-101, 90),
                                   (-126, 120), (-140, 127), (-148, 127), (-140, -20), (120, 20)])
@pytest.mark.parametrize("bias", [False, True])
def test_scales_at_the_ends_of_the_range(ops, M, N, K, kernel, out, ea, ew, bias):
    import torch
    import aegis_i8 as i8
    assert i8.gemm_plan(M, N, K)["kernel"] == kernel
    dt = getattr(torch, out)
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, w = (torch.randint(-128, 128, s, device="cuda", generator=g, dtype=torch.int8) for s in ((M, K), (N, K)))
    # every third row of each has an ordinary scale
    sa, sw = ((1 + torch.rand(n, device="cuda", generator=g, dtype=torch.float64)) * 2.0 ** e for n, e in ((M, ea), (N, ew)))
    sa[2::3], sw[2::3] = sa[2::3] * 2.0 ** -ea, sw[2::3] * 2.0 ** -ew
    sa, sw = sa.float(), sw.float()
    sw[N // 2] = 0.0
    b = (torch.randn(N, device="cuda", generator=g) * 2.0 ** min(100, ea + ew + 20)).to(dt) if bias else None
    c = ops.matmul_i8(a, w, sa, sw, b, out_dtype=dt)
    exact = (a.double() @ w.double().t()) * (sa.double()[:, None] * sw.double())
    mag = exact.abs()
    if bias:
        exact, mag = exact + b.double(), mag + b.double().abs()
    most = float(torch.finfo(dt).max)
    tol = HALF[out] * exact.abs() * (1 + 2.0 ** -10) + 5 * 2.0 ** -24 * mag + TINY[out] + 2.0 ** -150
    over = exact.abs() - tol > most * (1 + HALF[out])  # rounds to infinity
    under = exact.abs() + tol < most
    assert torch.equal(c[over].double(), torch.sign(exact[over]) * float("inf"))
    off = ((c.double() - exact).abs() - tol)[under]
    assert not c[under].isnan().any() and off.max().item() <= 0, f"off by {off.max().item()}"
