"""The 4-bit calls' C ABI on a machine without a GPU: calls without rows, and sizes that no launch takes."""
import ctypes

from mignon_ai_amd import _lib

INVALID = _lib.MG_ERR_INVALID


def test_matrices_without_rows_need_no_memory():
    """An empty tensor has no address. What such a call says about types and shapes is checked all the same."""
    L = _lib.lib()
    q = lambda M=0, K=64, ty=0: L.mg_mx4_quantize(None, ty, M, K, K, None, None, _lib.MG_PTR_DEVICE, None)  # noqa: E731
    d = lambda M=0, K=64, ty=0: L.mg_mx4_dequantize(None, None, M, K, None, ty, K, _lib.MG_PTR_DEVICE, None)  # noqa: E731
    g = lambda M=0, K=64, ty=0: L.mg_mx4_gemm(None, None, M, K, None, None, 8, None, ty, _lib.MG_PTR_DEVICE, None)  # noqa: E731
    for f in (q, d, g):
        assert f() == 0
        for bad in (dict(K=0), dict(ty=7), dict(M=-1), dict(M=1)):
            assert f(**bad) == INVALID, bad


def test_products_of_more_tiles_than_a_launch_has_lanes():
    """The refusal names its cause and comes before the device is touched."""
    L, p = _lib.lib(), 1 << 20
    for M, N in (((1 << 30) + 1, 64), ((1 << 31) - 1, 8), ((1 << 31) - 1, 1 << 12), (1 << 27, 1 << 24)):
        assert L.mg_mx4_gemm(p, p, M, 128, p, p, N, p, 0, _lib.MG_PTR_DEVICE, None) == INVALID, (M, N)
        assert b"mg_mx4_gemm: too many" in L.mg_last_error()


def test_attention_of_nearly_two_to_the_31_rows():
    """A last tile of rows that would pass 2^31 is refused like any call of too many."""
    c = _lib.KvCache(1, 1, 32, 64, 0, *(4 * (1 << 20,)))
    ws = lambda T, heads: _lib.lib().mg_kv_attention_workspace(ctypes.addressof(c), heads, T, 0)  # noqa: E731
    assert ws((1 << 30) - 1, 2) == INVALID      # 2^31 - 2 rows
    assert ws((1 << 30) - 64, 2) == 0           # one launch
    assert ws((1 << 30) - 63, 2) == INVALID
    assert ws(((1 << 31) - 1) // 7, 7) == INVALID
