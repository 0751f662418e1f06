"""The 4-bit rows and their product through the tensor calls: matrices without rows."""
import pytest
import torch

from mignon_ai_amd import MignonError, mx4_dequantize_device, mx4_gemm_device, mx4_quantize_device

pytestmark = pytest.mark.gpu


def _device4(M, K):
    Kp = -(-K // 128) * 128
    return tuple(torch.zeros((M, Kp // d), dtype=torch.uint8, device="cuda") for d in (2, 32))


def test_matrices_without_rows():
    x, rows, w = torch.empty((0, 200), device="cuda"), _device4(0, 200), _device4(5, 200)
    mx4_quantize_device(x, *rows)
    mx4_dequantize_device(*rows, x)
    mx4_gemm_device(*rows, *w, torch.empty((0, 5), device="cuda"))
    with pytest.raises(MignonError):
        mx4_gemm_device(*rows, *_device4(5, 300), torch.empty((0, 5), device="cuda"))
    with pytest.raises(MignonError):
        mx4_quantize_device(x, *_device4(0, 300))


def test_product_of_more_than_four_million_tiles():
    """2^28 rows of one step by one tile's channels: the last rows' products in their place, and nothing behind them."""
    M, K, N = (1 << 28) + 70, 128, 64
    A, As = torch.zeros((M, K // 2), dtype=torch.uint8, device="cuda"), torch.full((M, K // 32), 127, dtype=torch.uint8, device="cuda")
    W, Ws = torch.full((N, K // 2), 0x22, dtype=torch.uint8, device="cuda"), torch.full((N, K // 32), 127, dtype=torch.uint8, device="cuda")
    Ws += torch.arange(N, dtype=torch.uint8, device="cuda")[:, None] % 8
    A[-3:] = 0x24  # pairs of 2 and 1
    C = torch.full((M + 1, N), 9.0, dtype=torch.bfloat16, device="cuda")
    mx4_gemm_device(A, As, W, Ws, C[:M])
    want = 192 * 2.0 ** (torch.arange(N, device="cuda") % 8)
    assert bool((C[M - 3:M].float() == want).all()) and bool((C[M] == 9.0).all())
    assert all(not bool(c.any()) for c in C[:M - 3].split(1 << 26))


@pytest.mark.parametrize("K", [1 << 24, (1 << 24) - 3])
def test_the_longest_rows(K):
    """Rows of as many elements as a call takes, nearly all zeros: the values and the product of what is not."""
    M, N, Kp = 3, 5, 1 << 24
    g = torch.Generator("cuda").manual_seed(1)
    at = torch.randint(0, K, (200,), generator=g, device="cuda")
    at[:3] = torch.tensor([0, K - 1, K - 40], device="cuda")
    values = torch.tensor([0.5, 1.0, 2.0, 3.0, 4.0, 6.0, -1.5], device="cuda")
    x = torch.zeros((M + N, K), device="cuda")
    x[:, at] = values[torch.randint(0, 7, (M + N, 200), generator=g, device="cuda")]
    codes, scales = _device4(M + N, K)
    assert codes.shape[1] == Kp // 2
    mx4_quantize_device(x, codes, scales)
    y = torch.full_like(x, 9.0)
    mx4_dequantize_device(codes, scales, y)
    # (a value next to a larger one may be rounded)
    assert int((y != 0).sum()) <= int((x != 0).sum()) and bool(((y - x).abs() <= 1).all())
    C = torch.empty((M, N), device="cuda")
    mx4_gemm_device(codes[:M], scales[:M], codes[M:], scales[M:], C)
    assert torch.equal(C.double(), y[:M].double() @ y[M:].double().t().contiguous())
