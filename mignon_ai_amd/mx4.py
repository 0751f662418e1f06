"""Microscaled 4-bit numbers on the GPU: quantisation and the product (the 4-bit counterparts of quantize_f32 and gemm_i8),
and a key/value cache held in 4 bits with attention over it.

The format (include/mignon_hip.h): blocks of 32 elements along a row, each with a power-of-two scale byte and 16 bytes of
codes. A matrix [M][K] is held as codes [M][Kp / 2] and scales [M][Kp / 32], Kp being K rounded up to a multiple of 128
(zeros in the padding).

The functions without _device take numpy arrays (float32 or float16) on the host; the *_device functions and KVCache take torch
CUDA tensors and enqueue their work, by default on torch's current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._lib import MG_BF16, MG_F16, MG_F32, MG_PTR_DEVICE, KvCache, KvRows, MignonError, check, lib, ptr

_HOST_TYPES = {np.dtype(np.float32): MG_F32, np.dtype(np.float16): MG_F16}
_torch = None     # (imported with the first call on tensors: the host functions do not need it)
_reals, _u8, _i32 = {}, None, None


def _invalid(msg: str):
    raise MignonError(-1, msg)


def padded(K: int) -> int:
    """The elements that a row of K takes."""
    return (K + 127) // 128 * 128


def _tensors():
    global _torch, _u8, _i32
    import torch
    _reals.update({torch.float32: MG_F32, torch.float16: MG_F16, torch.bfloat16: MG_BF16})
    _torch, _u8, _i32 = torch, torch.uint8, torch.int32


def _launch(who, fn, stream, tensors, args):
    """fn(*args, stream) with the tensors' device as the current one, on `stream` (default: torch's current stream there)."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != dev or dev < 0:
            _invalid(f"{who}: tensors on one GPU are needed")
    if _torch.cuda.current_device() != dev:
        with _torch.cuda.device(dev):
            return _launch(who, fn, stream, tensors, args)
    rc = fn(*args, _torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream)
    if rc < 0:
        check(rc)


def _real(who, t, name):
    """The type, shape and row stride of a matrix of reals."""
    if _torch is None:
        _tensors()
    ty = _reals.get(t.dtype)
    if ty is None:
        _invalid(f"{who}: {name} is float32, float16 or bfloat16")
    if t.dim() != 2:
        _invalid(f"{who}: {name} is a matrix")
    M, K = t.shape
    ld, one = t.stride()
    if (K > 1 and one != 1) or M >> 31 or K >> 31:
        _invalid(f"{who}: {name} has neighbouring elements in its rows, and fewer than 2^31 each way")
    return ty, M, K, ld if M > 1 else K


def _rows4(who, codes, scales, name):
    """Rows and padded elements of a 4-bit matrix."""
    if _torch is None:
        _tensors()
    if codes.dtype is not _u8 or scales.dtype is not _u8 or codes.dim() != 2 or scales.dim() != 2:
        _invalid(f"{who}: {name}'s codes and scales are uint8 matrices")
    (M, b), (m, s) = codes.shape, scales.shape
    if M != m or b != 16 * s or b % 64 or b == 0 or M >> 31 or b >> 30 or not codes.is_contiguous() or not scales.is_contiguous():
        _invalid(f"{who}: {name}'s codes are [M][Kp / 2] and its scales [M][Kp / 32], contiguous, Kp a multiple of 128")
    return M, 2 * b


def mx4_quantize(x):
    """mg_mx4_quantize on a host array [M][K] -> (codes [M][Kp / 2], scales [M][Kp / 32]) uint8."""
    x = np.asarray(x)
    if x.dtype not in _HOST_TYPES:
        x = x.astype(np.float32)
    x = np.ascontiguousarray(x)
    if x.ndim != 2 or x.shape[1] == 0:
        _invalid("mx4_quantize: a matrix is needed")
    M, K = x.shape
    codes, scales = np.empty((M, padded(K) // 2), np.uint8), np.empty((M, padded(K) // 32), np.uint8)
    check(lib().mg_mx4_quantize(ptr(x), _HOST_TYPES[x.dtype], M, K, K, ptr(codes), ptr(scales), 0, None))
    return codes, scales


def _host4(who, codes, scales):
    codes, scales = np.ascontiguousarray(codes, np.uint8), np.ascontiguousarray(scales, np.uint8)
    if (codes.ndim != 2 or scales.ndim != 2 or codes.shape[0] != scales.shape[0] or codes.shape[1] != 16 * scales.shape[1]
            or codes.shape[1] % 64 or codes.shape[1] == 0):
        _invalid(f"{who}: codes are [M][Kp / 2] and scales [M][Kp / 32], Kp a multiple of 128")
    return codes, scales


def mx4_dequantize(codes, scales, K=None):
    """mg_mx4_dequantize on host arrays -> float32 [M][K] (K: the padded length if not given)."""
    codes, scales = _host4("mx4_dequantize", codes, scales)
    M = codes.shape[0]
    K = 2 * codes.shape[1] if K is None else int(K)
    if padded(K) != 2 * codes.shape[1]:
        _invalid("mx4_dequantize: K does not go with the codes")
    y = np.empty((M, K), np.float32)
    check(lib().mg_mx4_dequantize(ptr(codes), ptr(scales), M, K, ptr(y), MG_F32, K, 0, None))
    return y


def mx4_gemm(A, As, W, Ws):
    """mg_mx4_gemm on host arrays: codes and scales of A [M][K] and W [N][K] -> C [M][N] float32."""
    A, As = _host4("mx4_gemm", A, As)
    W, Ws = _host4("mx4_gemm", W, Ws)
    if A.shape[1] != W.shape[1] or W.shape[0] == 0:
        _invalid("mx4_gemm: A and W have rows of one length")
    C = np.empty((A.shape[0], W.shape[0]), np.float32)
    check(lib().mg_mx4_gemm(ptr(A), ptr(As), A.shape[0], 2 * A.shape[1], ptr(W), ptr(Ws), W.shape[0], ptr(C), MG_F32, 0, None))
    return C


def mx4_quantize_device(x, codes, scales, stream=None):
    """mg_mx4_quantize on torch CUDA tensors: x [M][K] float32, float16 or bfloat16 (rows may be strided) into codes and
    scales. Enqueued on `stream` (a stream's address; default: torch's current stream)."""
    ty, M, K, ld = _real("mx4_quantize_device", x, "x")
    if _rows4("mx4_quantize_device", codes, scales, "the result") != (M, padded(K)):
        _invalid("mx4_quantize_device: codes and scales do not go with x")
    _launch("mx4_quantize_device", lib().mg_mx4_quantize, stream, (x, codes, scales),
            (x.data_ptr(), ty, M, K, ld, codes.data_ptr(), scales.data_ptr(), MG_PTR_DEVICE))


def mx4_dequantize_device(codes, scales, y, stream=None):
    """mg_mx4_dequantize on torch CUDA tensors: the values into y [M][K] (rows may be strided)."""
    ty, M, K, ld = _real("mx4_dequantize_device", y, "y")
    if _rows4("mx4_dequantize_device", codes, scales, "the operand") != (M, padded(K)):
        _invalid("mx4_dequantize_device: codes and scales do not go with y")
    _launch("mx4_dequantize_device", lib().mg_mx4_dequantize, stream, (y, codes, scales),
            (codes.data_ptr(), scales.data_ptr(), M, K, y.data_ptr(), ty, ld, MG_PTR_DEVICE))


def mx4_gemm_device(A, As, W, Ws, C, stream=None):
    """mg_mx4_gemm on torch CUDA tensors: C [M][N] = A W^T (float32, float16 or bfloat16, contiguous)."""
    M, Kp = _rows4("mx4_gemm_device", A, As, "A")
    N, Kw = _rows4("mx4_gemm_device", W, Ws, "W")
    ty = _reals.get(C.dtype)
    if ty is None or C.shape != (M, N) or Kp != Kw or not C.is_contiguous():
        _invalid("mx4_gemm_device: A [M][K], W [N][K] and a contiguous C [M][N] of reals are needed")
    _launch("mx4_gemm_device", lib().mg_mx4_gemm, stream, (A, As, W, Ws, C),
            (A.data_ptr(), As.data_ptr(), M, Kp, W.data_ptr(), Ws.data_ptr(), N, C.data_ptr(), ty, MG_PTR_DEVICE))


class KVCache:
    """A 4-bit key/value cache (mg_kv_cache_t) over torch CUDA tensors: k and v codes [n][heads][capacity][head_dim / 2], their
    scales [n][heads][capacity][head_dim / 32], uint8. Positions below `sinks` keep their slots, later ones take turns in the
    others. The caller keeps count of the positions, and has the rows written by `write` (the planes' first contents do not
    matter). Calls are enqueued on torch's current stream of the cache's device."""

    def __init__(self, k, k_scales, v, v_scales, sinks: int = 0):
        self.k, self.k_scales, self.v, self.v_scales = k, k_scales, v, v_scales
        if _torch is None:
            _tensors()
        for t in (k, k_scales, v, v_scales):
            if t.dtype is not _u8 or t.dim() != 4 or not t.is_contiguous() or not t.is_cuda or t.device != k.device:
                _invalid("KVCache: planes are contiguous uint8 tensors of four dimensions on one GPU")
        n, heads, cap, half = k.shape
        if max(k.shape) >> 30 or not 0 <= int(sinks) < max(cap, 1):
            _invalid("KVCache: fewer than 2^30 each way, and sinks fewer than the capacity")
        if v.shape != k.shape or k_scales.shape != (n, heads, cap, half // 16) or v_scales.shape != k_scales.shape:
            _invalid("KVCache: codes are [n][heads][capacity][head_dim / 2], scales [n][heads][capacity][head_dim / 32]")
        self.n, self.heads, self.capacity, self.head_dim, self.sinks = n, heads, cap, 2 * half, int(sinks)
        self.device, self._shape = k.device, (n,)
        self._c = KvCache(n, heads, 2 * half, cap, self.sinks, k.data_ptr(), k_scales.data_ptr(), v.data_ptr(),
                          v_scales.data_ptr())
        self._p, self._planes = ctypes.addressof(self._c), (k, k_scales, v, v_scales)
        self._need = {}
        self._workspace(heads, 1, 0)  # refuses what the calls would refuse

    @classmethod
    def empty(cls, n: int, heads: int, head_dim: int, capacity: int, sinks: int = 0, device="cuda") -> "KVCache":
        """A cache of its own memory; capacity is rounded up to a multiple of 32."""
        import torch
        cap = (int(capacity) + 31) // 32 * 32
        planes = [torch.zeros((n, heads, cap, w), dtype=torch.uint8, device=device)
                  for w in (head_dim // 2, head_dim // 32) * 2]
        return cls(*planes, sinks=sinks)

    def _workspace(self, q_heads, T, window):
        key = (q_heads, T, window)
        need = self._need.get(key)
        if need is None:
            need = lib().mg_kv_attention_workspace(self._p, q_heads, T, window)
            check(-1 if need < 0 else 0)
            if len(self._need) >= 256:
                self._need.clear()
            self._need[key] = need
        return need

    def _rows(self, who, t, name, heads):
        ty = _reals.get(t.dtype)
        if ty is not None and t.dim() == 4:
            n, T, h, d = t.shape
            seq, token, head, one = t.stride()
            if n == self.n and d == self.head_dim and one == 1 and (h == heads if heads else h < 1 << 30) and T < 1 << 30:
                return ty, KvRows(t.data_ptr(), seq, token, head)
        _invalid(f"{who}: {name} is [n][T][heads][head_dim] of float32, float16 or bfloat16, channels side by side")

    def _ints(self, who, *arrays):
        for a in arrays:
            if a is not None and (a.dtype is not _i32 or a.shape != self._shape or not a.is_contiguous()):
                _invalid(f"{who}: positions, counts and lengths are int32 [n]")

    def _two(self, who, k, v, pos, *ints):
        (ty, kr), (tv, vr) = self._rows(who, k, "k", self.heads), self._rows(who, v, "v", self.heads)
        if ty != tv or k.shape != v.shape or pos is None:
            _invalid(f"{who}: k and v have one shape and type, and positions are given")
        self._ints(who, pos, *ints)
        return ty, kr, vr

    def write(self, k, v, pos, counts=None):
        """mg_kv_write: new rows k, v [n][T][heads][head_dim] (any strides but the last) at positions pos[s] + t, of which the
        first counts[s] (default T) are there. pos, counts: int32 [n]."""
        ty, kr, vr = self._two("KVCache.write", k, v, pos, counts)
        _launch("KVCache.write", lib().mg_kv_write, None, (self._planes[0], k, v, pos) + (() if counts is None else (counts,)),
                (self._p, ctypes.addressof(kr), ctypes.addressof(vr), ty, k.shape[1], pos.data_ptr(), ptr(counts)))

    def read(self, k, v, pos, counts=None, lens=None):
        """mg_kv_read: the rows at positions pos[s] + t into k, v; lens [n]: the sequences' lengths (default pos + counts)."""
        ty, kr, vr = self._two("KVCache.read", k, v, pos, counts, lens)
        more = tuple(a for a in (counts, lens) if a is not None)
        _launch("KVCache.read", lib().mg_kv_read, None, (self._planes[0], k, v, pos) + more,
                (self._p, ctypes.addressof(kr), ctypes.addressof(vr), ty, k.shape[1], pos.data_ptr(), ptr(counts), ptr(lens)))

    def attention(self, q, out, pos, counts=None, window: int = 0, scale: float | None = None):
        """mg_kv_attention: rows q [n][T][q_heads][head_dim] at positions pos[s] + t over the cache (their own keys written
        already) into out (which may be q), which is returned; scale: head_dim ** -0.5 if not given."""
        ty, qr = self._rows("KVCache.attention", q, "q", None)
        to, orow = self._rows("KVCache.attention", out, "out", None)
        if ty != to or q.shape != out.shape or pos is None:
            _invalid("KVCache.attention: q and out have one shape and type, and positions are given")
        self._ints("KVCache.attention", pos, counts)
        T, q_heads, window = q.shape[1], q.shape[2], min(max(int(window), 0), 1 << 30)
        need = self._workspace(q_heads, T, window)
        ws = self._planes[0].new_empty(need) if need else None
        _launch("KVCache.attention", lib().mg_kv_attention, None, (self._planes[0], q, out, pos) + (() if counts is None else (counts,)),
                (self._p, ctypes.addressof(qr), ctypes.addressof(orow), ty, q_heads, T, pos.data_ptr(), ptr(counts), window,
                 self.head_dim ** -0.5 if scale is None else scale, ptr(ws), need))
        return out

    def gather(self, parents, lens, source: "KVCache | None" = None, source_lens=None):
        """mg_kv_gather: sequence i becomes sequence parents[i] of `source` (default: of this cache, as if from a copy taken before),
        lens[i] positions long; it stays where parents[i] is none of the source's. parents, lens: int32 [n]; source_lens int32
        [source.n]: the lengths of the source's sequences, where they are longer than what is taken of them."""
        src = self if source is None else source
        if parents is None or lens is None:
            _invalid("KVCache.gather: parents and lengths are given")
        self._ints("KVCache.gather", parents, lens)
        src._ints("KVCache.gather", source_lens)
        more = () if source_lens is None else (source_lens,)
        _launch("KVCache.gather", lib().mg_kv_gather, None, (self._planes[0], src._planes[0], parents, lens) + more,
                (self._p, src._p, parents.data_ptr(), lens.data_ptr(), ptr(source_lens)))

    def attention_shared(self, q, out, pos, prefix: "KVCache", prefix_lens, starts=None, counts=None, window: int = 0,
                         scale: float | None = None):
        """mg_kv_attention_shared: `attention` for sequences that go on from prefixes: sequences starts[g] .. starts[g + 1] - 1 from
        sequence g of `prefix`, of whose first prefix_lens[g] positions they see all that it holds. prefix_lens int32 [prefix.n],
        starts int32 [prefix.n + 1] (None: all go on from the only one). pos counts a sequence's own positions."""
        who = "KVCache.attention_shared"
        ty, qr = self._rows(who, q, "q", None)
        to, orow = self._rows(who, out, "out", None)
        if ty != to or q.shape != out.shape or pos is None or prefix_lens is None:
            _invalid(f"{who}: q and out have one shape and type, positions and the prefixes' lengths are given")
        self._ints(who, pos, counts)
        prefix._ints(who, prefix_lens)
        if starts is not None and (starts.dtype is not _i32 or starts.shape != (prefix.n + 1,) or not starts.is_contiguous()):
            _invalid(f"{who}: starts are int32 [prefixes + 1]")
        T, q_heads, window = q.shape[1], q.shape[2], min(max(int(window), 0), 1 << 30)
        key = (q_heads, T, window, prefix.n, prefix.capacity, prefix.heads, prefix.head_dim)
        need = self._need.get(key)
        if need is None:
            need = lib().mg_kv_attention_shared_workspace(self._p, prefix._p, q_heads, T, window)
            check(-1 if need < 0 else 0)
            if len(self._need) >= 256:
                self._need.clear()
            self._need[key] = need
        ws = self._planes[0].new_empty(need) if need else None
        more = tuple(a for a in (starts, counts) if a is not None)
        _launch(who, lib().mg_kv_attention_shared, None, (self._planes[0], prefix._planes[0], q, out, pos, prefix_lens) + more,
                (self._p, prefix._p, prefix_lens.data_ptr(), ptr(starts), ctypes.addressof(qr), ctypes.addressof(orow), ty, q_heads, T,
                 pos.data_ptr(), ptr(counts), window, self.head_dim ** -0.5 if scale is None else scale, ptr(ws), need))
        return out
