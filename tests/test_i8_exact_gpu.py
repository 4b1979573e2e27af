"""The norm's scale to the last bit, and the block's results that follow from it.

A norm's scale is one rounding of m / sqrt(mean h^2 + eps) / 127: half a step,
2^-24 of the value. Its sum is taken in 64 bits, at most n roundings of 2^-53
for n columns (2^-33 at 2^20 columns, halved by the root), the rest of the
formula 5 more: 2^-20 of that half step is far above both."""
import struct

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


def as_float(x):
    """x rounded to 32 bits, as the C call takes eps."""
    return struct.unpack("f", struct.pack("f", x))[0]


def assert_scale(torch, s, h, w, eps):
    hd = h.double()
    m = (hd * w.double()).abs().amax(dim=1)
    want = m / torch.sqrt(hd.square().mean(dim=1) + as_float(eps)) / 127.0
    assert (want > 2.0 ** -126).all() and (want < 2.0 ** 127).all()
    off = ((s.double() - want).abs() / want).max().item() * 2.0 ** 24
    assert off <= 1 + 2.0 ** -20, f"{tuple(h.shape)}: off by {off} half steps"


# Every way a row is taken: one piece a thread to four, blocks over many rows, rows beyond 32768.
ROWS = [(1, 1), (2, 64), (300, 1000), (5, 4096), (3, 4099), (2, 8192), (12, 5120), (2, 14336), (9, 16384), (2, 32768),
        (2, 32769), (1, 1 << 20), (700, 896), (700, 1501), (700, 3001), (700, 7001), (400, 5120), (2500, 4096),
        (400, 8192), (400, 14336), (400, 32768)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_norm_scale_is_rounded_once(ops, dtype, rows, cols):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, r = ((torch.randn(rows, cols, device="cuda", generator=g) * 2).to(dt) for _ in range(2))
    w = (torch.randn(cols, device="cuda", generator=g) * 0.2 + 1).to(dt)
    _, s = ops.rmsnorm_i8(x, w, 1e-5)
    assert_scale(torch, s, x, w, 1e-5)
    _, s, h = ops.add_rmsnorm_i8(x, r, w, 1e-6)
    assert_scale(torch, s, h, w, 1e-6)


@pytest.mark.parametrize("rows,cols", [(2, 4096), (2, 40000), (1, 1 << 20), (400, 1024)])
def test_norm_scale_of_rows_of_one_value(ops, rows, cols):
    """Every addition of such a row's squares would round the same way."""
    import torch
    w = torch.ones(cols, device="cuda").bfloat16()
    for v in (1.0078125, 1.3359375, 1.9921875, 117.5):
        x = torch.full((rows, cols), v, device="cuda").bfloat16()
        _, s = ops.rmsnorm_i8(x, w, 0.0)
        assert_scale(torch, s, x, w, 0.0)


@pytest.mark.parametrize("rows,cols", [(2, 1), (2, 4096), (400, 1024), (2, 40000)])
def test_norm_scale_with_a_large_eps(ops, rows, cols):
    """mean h^2 + eps beyond float's range has a scale all the same."""
    import torch
    x = torch.full((rows, cols), 2.9e18, device="cuda").bfloat16()
    w = torch.ones(cols, device="cuda").bfloat16()
    _, s = ops.rmsnorm_i8(x, w, 3.39e38)
    assert_scale(torch, s, x, w, 3.39e38)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("M,K,F", [(1, 1024, 2048), (7, 896, 4864), (33, 257, 333), (64, 4096, 1024), (64, 1024, 14336)])
def test_block_has_the_bits_of_its_definition(ops, dtype, M, K, F):
    """Codes and scales are definite, sums exact, and a product's float steps are fixed: so is every bit of y."""
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(M + K + F)
    x, r = (torch.randn(M, K, device="cuda", generator=g).to(dt) for _ in range(2))
    nw = (torch.randn(K, device="cuda", generator=g) * 0.2 + 1).to(dt)
    w1, w2 = (torch.randint(-127, 128, s, device="cuda", generator=g, dtype=torch.int8) for s in ((2 * F, K), (K, F)))
    s1 = (torch.rand(2 * F, device="cuda", generator=g) + 0.5) / (74 * K ** 0.5)
    s2 = (torch.rand(K, device="cuda", generator=g) + 0.5) / (74 * F ** 0.5)
    eps = 2.0 ** -17
    y, h = ops.mlp_i8(x, r, nw, eps, w1, s1, w2, s2)

    def quantise(t, rms):
        m = t.abs().amax(dim=1, keepdim=True)
        return torch.round(127.0 * t / m), (m[:, 0] / rms / 127.0).float()

    def product(q, w, sq, sw):
        return ((q @ w.double().t()).float() * sq[:, None] * sw[None, :]).to(dt)

    hd = (x.float() + r.float()).to(dt).double()
    assert torch.equal(h.double(), hd)
    q, s = quantise(hd * nw.double(), torch.sqrt(hd.square().mean(dim=1) + eps))
    gu = product(q, w1, s, s1).double()
    q, s = quantise(gu[:, :F] / (1 + torch.exp(-gu[:, :F])) * gu[:, F:], 1.0)
    want = product(q, w2, s, s2)
    assert torch.equal(y, want), f"{(y != want).sum().item()} of {y.numel()} values differ"
