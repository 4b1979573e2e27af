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
