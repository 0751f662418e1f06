"""Refusals of the operators for many continuations of one prompt (cache sequences gathered, attention over shared prefixes, log
probabilities): every bad call is an error before anything touches a device."""
import ctypes

import numpy as np
import pytest

import mignon_ai_amd as M
from mignon_ai_amd import _lib

I = ctypes.c_int32 * 64
F = ctypes.c_float * 64


class Plane:
    """Sixteen-byte aligned host memory: never read by a refused call."""

    def __init__(self, size=1 << 16):
        self.m = (ctypes.c_uint8 * (size + 16))()
        self.at = (ctypes.addressof(self.m) + 15) // 16 * 16


def cache(n=2, heads=2, dh=32, cap=64, sinks=0, planes=None, **change):
    planes = planes or [Plane() for _ in range(4)]
    c = _lib.KvCache(n, heads, dh, cap, sinks, *[p.at for p in planes])
    for k, v in change.items():
        setattr(c, k, v)
    c.keep = planes
    return c


def refused(rc, word):
    assert rc == _lib.MG_ERR_INVALID
    assert word in _lib.lib().mg_last_error().decode(), _lib.lib().mg_last_error()


def gather(to, frm, parents=True, lens=True):
    i = I()
    p = ctypes.addressof(i)
    return _lib.lib().mg_kv_gather(ctypes.addressof(to) if to else None, ctypes.addressof(frm) if frm else None, p if parents else None,
                                   p if lens else None, None, None)


def test_gather_refusals():
    a, b = cache(), cache()
    refused(gather(None, a), "null")
    refused(gather(a, b, parents=False), "null")
    refused(gather(a, b, lens=False), "null")
    refused(gather(cache(dh=48), b), "head_dim")
    refused(gather(a, cache(dh=48)), "head_dim")
    refused(gather(a, cache(heads=1)), "heads")
    refused(gather(a, cache(dh=64)), "heads")
    refused(gather(cache(cap=60), b), "capacity")
    refused(gather(cache(sinks=64), b), "sinks")
    refused(gather(cache(k=a.k + 8), b), "misaligned")
    refused(gather(cache(v=None), b), "null")
    # the same planes under other sizes, a plane of one in two caches, planes that overlap
    refused(gather(a, cache(cap=32, planes=a.keep)), "share")
    refused(gather(a, cache(sinks=1, planes=a.keep)), "share")
    refused(gather(a, cache(n=1, planes=a.keep)), "share")
    refused(gather(a, cache(v=a.v)), "share")
    refused(gather(a, cache(k=a.v)), "share")
    refused(gather(a, cache(k=a.k + 2 * 2 * 64 * 16 - 16)), "share")
    refused(gather(a, cache(planes=a.keep, v=b.v)), "share")
    # one launch's lanes, and what one workgroup reads
    refused(gather(cache(n=16385), None), "many")
    far = {"k": 1 << 44, "k_scales": 2 << 44, "v": 3 << 44, "v_scales": 4 << 44}  # (as much memory as it takes is nowhere here)
    refused(gather(cache(n=1 << 22, **far), cache()), "many")
    # nothing to do
    assert gather(cache(n=0), a) == 0
    assert gather(a, cache(n=0, k=None, v=None)) == 0


def shared(c, p, q=True, lens=True, starts=True, type=0, q_heads=4, T=1, ws=0, ws_bytes=0, pos=True, at=0):
    i, x = I(), Plane()
    rows = _lib.KvRows(x.at + at, 1, 1, 1)
    r = ctypes.addressof(rows) if q else None
    ip = ctypes.addressof(i)
    return _lib.lib().mg_kv_attention_shared(ctypes.addressof(c) if c else None, ctypes.addressof(p) if p else None, ip if lens else None,
                                             ip if starts else None, r, r, type, q_heads, T, ip if pos else None, None, 0, 1.0, ws or None,
                                             ws_bytes, None)


def test_shared_attention_refusals():
    c, p = cache(), cache(n=3)
    ws = _lib.lib().mg_kv_attention_shared_workspace(ctypes.addressof(c), ctypes.addressof(p), 4, 1, 0)
    assert ws > 0
    room = Plane()
    refused(shared(None, p, ws=room.at, ws_bytes=ws), "null")
    refused(shared(c, None, ws=room.at, ws_bytes=ws), "null")
    refused(shared(c, p, q=False, ws=room.at, ws_bytes=ws), "null")
    refused(shared(c, p, pos=False, ws=room.at, ws_bytes=ws), "null")
    refused(shared(c, p, lens=False, ws=room.at, ws_bytes=ws), "without")
    refused(shared(c, p, starts=False, ws=room.at, ws_bytes=ws), "without")
    refused(shared(c, p, type=3, ws=room.at, ws_bytes=ws), "type")
    refused(shared(c, p, q_heads=3, ws=room.at, ws_bytes=ws), "q_heads")
    refused(shared(c, cache(heads=1), ws=room.at, ws_bytes=ws), "unequal heads")
    refused(shared(c, cache(dh=64), ws=room.at, ws_bytes=ws), "unequal heads")
    refused(shared(c, cache(cap=33), ws=room.at, ws_bytes=ws), "capacity")
    refused(shared(c, p, at=2, ws=room.at, ws_bytes=ws), "misaligned")
    refused(shared(c, p, ws=room.at + 4, ws_bytes=ws), "misaligned")
    refused(shared(c, p, ws=0, ws_bytes=ws), "workspace")
    refused(shared(c, p, ws=room.at, ws_bytes=ws - 1), "workspace")
    refused(shared(c, p, ws=room.at, ws_bytes=-1), "workspace")
    refused(shared(c, p, T=-1, ws=room.at, ws_bytes=ws), "shape")
    big = cache(n=1 << 20)
    refused(shared(big, p, q_heads=2, T=1 << 12), "many")
    refused(shared(c, cache(n=1 << 26, heads=2), T=1), "many")
    assert _lib.lib().mg_kv_attention_shared_workspace(ctypes.addressof(c), None, 4, 1, 0) == _lib.MG_ERR_INVALID
    # nothing to do
    assert shared(cache(n=0), p) == 0
    assert shared(c, p, T=0) == 0
    assert _lib.lib().mg_kv_attention_shared_workspace(ctypes.addressof(c), ctypes.addressof(p), 4, 0, 0) == 0


def logprobs(x=True, type=0, n=2, V=8, ld=8, targets=True, m=1, k=2, logprob=True, ids=True, top=True, ws=None, at=0, flags=1):
    f, i = F(), I()
    fp, ip = ctypes.addressof(f), ctypes.addressof(i)
    return _lib.lib().mg_token_logprobs(fp + at if x else None, type, n, V, ld, ip if targets else None, m, k, fp if logprob else None, fp,
                                        ip if ids else None, fp if top else None, ws, 0, flags, None)


def test_logprobs_refusals():
    refused(logprobs(x=False), "null")
    refused(logprobs(targets=False), "null")
    refused(logprobs(logprob=False), "null")
    refused(logprobs(ids=False, top=False), "null")
    refused(logprobs(type=9), "type")
    refused(logprobs(n=-1), "shape")
    refused(logprobs(V=0), "shape")
    refused(logprobs(V=(1 << 30) + 1, ld=1 << 31), "shape")
    refused(logprobs(ld=7), "shape")
    refused(logprobs(m=-1), "shape")
    refused(logprobs(k=-1), "k is")
    refused(logprobs(k=9), "k is")
    refused(logprobs(V=100, ld=100, k=65), "k is")
    refused(logprobs(at=2), "misaligned")
    assert logprobs(n=0, x=False) == 0
    ws = _lib.lib().mg_token_logprobs_workspace
    assert ws(-1, 8, 0) == ws(1, 0, 0) == ws(1, 8, 9) == ws(1, 100, 65) == ws(1, (1 << 30) + 1, 0) == ws(1, 8, -1) == _lib.MG_ERR_INVALID
    assert ws(0, 8, 8) >= 0 and ws(1 << 20, 1 << 20, 64) >= 0


def test_host_function_refusals():
    for bad in (np.zeros(4, np.float32), np.zeros((2, 0), np.float32)):
        with pytest.raises(M.MignonError, match="matrix"):
            M.token_logprobs(bad)
    for targets in (np.zeros(3, np.int32), np.zeros((3, 1), np.int32), np.zeros((2, 1, 1), np.int32), np.int32(1)):
        with pytest.raises(M.MignonError, match="targets"):
            M.token_logprobs(np.zeros((2, 4), np.float32), targets)
    with pytest.raises(M.MignonError, match="k is"):
        M.token_logprobs(np.zeros((2, 4), np.float32), k=5)


def test_tensor_refusals():
    """What the Python functions look at before the library is called."""
    torch = pytest.importorskip("torch")
    x = torch.zeros((2, 4))
    f = M.token_logprobs_device
    i32 = torch.zeros((2, 1), dtype=torch.int32)
    for kw in (dict(targets=i32), dict(logprob=torch.zeros((2, 1))), dict(targets=i32.long(), logprob=torch.zeros((2, 1))),
               dict(targets=i32, logprob=torch.zeros((2, 2))), dict(targets=i32[:1], logprob=torch.zeros((1, 1))),
               dict(entropy=torch.zeros(3)), dict(entropy=torch.zeros(2, dtype=torch.float64)),
               dict(top_ids=i32, top_logprob=torch.zeros((2, 2))), dict(top_ids=torch.zeros((2, 5), dtype=torch.int32)),
               dict(entropy=torch.zeros(2))):  # (the last: no GPU tensors)
        with pytest.raises(M.MignonError):
            f(x, **kw)
    with pytest.raises(M.MignonError):
        f(torch.zeros((2, 4), dtype=torch.float64))
    with pytest.raises(M.MignonError):
        f(torch.zeros((4, 2)).t())
