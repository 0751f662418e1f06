"""The 4-bit operators on a machine without a GPU: the reference restatement's format, and the C ABI's refusals, which come
before the device is touched."""
import ctypes

import numpy as np
import pytest

import mx4_ref as R
from mignon_ai_amd import _lib

INVALID = _lib.MG_ERR_INVALID


def test_reference_format():
    x = np.zeros((1, 32))
    x[0, :9] = [4, 5, 5.1, 7, 0.25, 0.26, 0.75, -1.25, -1.75]
    code, s = R.quantize_blocks(x)
    assert s[0, 0] == 127 and list(code[0, :9]) == [6, 6, 7, 7, 0, 1, 2, 10, 12]
    assert R.quantize_blocks(np.zeros((1, 32)))[1][0, 0] == 0
    assert np.isnan(R.rounded(np.full((1, 32), np.inf))).all()
    assert R.quantize_blocks(np.full((1, 32), np.float32(3e38)))[1][0, 0] == 252
    assert R.quantize_blocks(np.full((1, 32), 2.0 ** -149))[1][0, 0] == 0


def test_rows_refusals():
    L, p = _lib.lib(), 1 << 20  # an address that is never touched
    q = lambda **k: L.mg_mx4_quantize(*{**dict(x=p, type=0, M=4, K=64, ld=64, c=p, s=p, f=1, st=None), **k}.values())  # noqa: E731
    for k in (dict(x=None), dict(c=None), dict(s=None), dict(type=3), dict(type=-1), dict(M=-1), dict(K=0), dict(ld=63),
              dict(K=(1 << 24) + 1, ld=1 << 25), dict(x=p + 2), dict(c=p + 4), dict(s=p + 2)):
        assert q(**k) == INVALID, k
        assert b"mg_mx4_quantize" in L.mg_last_error()
        assert L.mg_mx4_dequantize(*[{**dict(c=p, s=p, M=4, K=64, x=p, type=0, ld=64, f=1, st=None), **k}[n]
                                     for n in ("c", "s", "M", "K", "x", "type", "ld", "f", "st")]) == INVALID, k
    assert q(M=0) == 0
    g = lambda **k: L.mg_mx4_gemm(*{**dict(A=p, As=p, M=4, K=64, W=p, Ws=p, N=4, C=p, type=0, f=1, st=None), **k}.values())  # noqa: E731
    for k in (dict(A=None), dict(As=None), dict(W=None), dict(Ws=None), dict(C=None), dict(M=-1), dict(K=0), dict(N=0), dict(type=9),
              dict(A=p + 8), dict(W=p + 1), dict(As=p + 1), dict(Ws=p + 2), dict(C=p + 1), dict(K=(1 << 24) + 1)):
        assert g(**k) == INVALID, k
    assert g(M=0) == 0


def _cache(**k):
    p = 1 << 20
    return _lib.KvCache(*{**dict(n=2, heads=4, head_dim=64, capacity=64, sinks=0, k=p, ks=p, v=p, vs=p), **k}.values())


@pytest.mark.parametrize("bad", [dict(n=-1), dict(heads=0), dict(head_dim=16), dict(head_dim=48), dict(head_dim=256), dict(capacity=0),
                                 dict(capacity=40), dict(sinks=-1), dict(sinks=64), dict(k=None), dict(ks=None), dict(v=None),
                                 dict(vs=None), dict(k=(1 << 20) + 8), dict(vs=(1 << 20) + 1), dict(n=1 << 30)])
def test_cache_refusals(bad):
    L, p = _lib.lib(), 1 << 20
    c, r = _cache(**bad), _lib.KvRows(p, 256, 256, 64)
    a = ctypes.addressof
    assert L.mg_kv_write(a(c), a(r), a(r), 0, 1, p, None, None) == INVALID
    assert L.mg_kv_read(a(c), a(r), a(r), 0, 1, p, None, None, None) == INVALID
    assert L.mg_kv_attention(a(c), a(r), a(r), 0, 4, 1, p, None, 0, 1.0, None, 0, None) == INVALID
    assert L.mg_kv_attention_workspace(a(c), 4, 1, 0) == INVALID
    assert b"mg_kv_attention_workspace" in L.mg_last_error()


def test_call_refusals():
    L, p = _lib.lib(), 1 << 20
    c, r, a = _cache(), _lib.KvRows(p, 256, 256, 64), ctypes.addressof
    null, odd = _lib.KvRows(None, 256, 256, 64), _lib.KvRows(p + 2, 256, 256, 64)
    for k, v, ty, T, pos in ((null, r, 0, 1, p), (r, null, 0, 1, p), (r, r, 5, 1, p), (r, r, 0, -1, p), (r, r, 0, 1, None),
                             (odd, r, 0, 1, p), (r, odd, 0, 1, p), (r, r, 0, 1 << 30, p)):
        assert L.mg_kv_write(a(c), a(k), a(v), ty, T, pos, None, None) == INVALID
        assert L.mg_kv_read(a(c), a(k), a(v), ty, T, pos, None, None, None) == INVALID
        assert L.mg_kv_attention(a(c), a(k), a(v), ty, 4, T, pos, None, 0, 1.0, None, 0, None) == INVALID
    for heads in (0, -4, 6, 65536 + 4):
        assert L.mg_kv_attention(a(c), a(r), a(r), 0, heads, 1, p, None, 0, 1.0, None, 0, None) == INVALID
    assert L.mg_kv_write(None, a(r), a(r), 0, 1, p, None, None) == INVALID
    # a long cache of one sequence is split, and the parts need memory
    long = _cache(n=1, capacity=1 << 16)
    need = L.mg_kv_attention_workspace(a(long), 4, 1, 0)
    assert need > 0
    for ws, size in ((None, need), (p, need - 1), (p, -1), (p + 4, need)):
        assert L.mg_kv_attention(a(long), a(r), a(r), 0, 4, 1, p, None, 0, 1.0, ws, size, None) == INVALID
    # nothing to do
    assert L.mg_kv_write(a(_cache(n=0)), a(r), a(r), 0, 1, p, None, None) == 0
    assert L.mg_kv_attention(a(c), a(r), a(r), 0, 4, 0, p, None, 0, 1.0, None, 0, None) == 0


def test_calls_of_more_rows_than_a_launch_has_lanes():
    L, a = _lib.lib(), ctypes.addressof
    assert L.mg_kv_attention_workspace(a(_cache(n=1 << 25, heads=1)), 1, 1, 0) == 0  # a wave a sequence, four a workgroup
    assert L.mg_kv_attention_workspace(a(_cache(n=1 << 26, heads=1)), 1, 1, 0) == INVALID
    assert L.mg_kv_attention_workspace(a(_cache(n=(1 << 24) - 1, heads=1, capacity=4096)), 1, 1, 0) == 0  # a workgroup a sequence
    assert L.mg_kv_attention_workspace(a(_cache(n=1 << 24, heads=1, capacity=4096)), 1, 1, 0) == INVALID
