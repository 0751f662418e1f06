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
