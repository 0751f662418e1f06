"""Log probabilities of given tokens, entropies and the likeliest tokens of rows of logits (mg_token_logprobs).

token_logprobs takes numpy arrays on the host, token_logprobs_device torch CUDA tensors.
"""
from __future__ import annotations

import numpy as np

from . import mx4
from ._lib import MG_PTR_DEVICE, check, lib, ptr

_need = {}


def token_logprobs(logits, targets=None, k: int = 0) -> dict:
    """Rows of logits [n][V] (float32 or float16) -> {"entropy" [n], "logprob" [n][m] of targets [n][m] or [n], "top_ids" and
    "top_logprob" [n][k]}, the last two and "logprob" where they are asked for."""
    x = np.asarray(logits)
    if x.dtype not in mx4._HOST_TYPES:
        x = x.astype(np.float32)
    x = np.ascontiguousarray(x)
    if x.ndim != 2 or x.shape[1] == 0:
        mx4._invalid("token_logprobs: a matrix is needed")
    n, V = x.shape
    if n >> 31 or V >> 31:
        mx4._invalid("token_logprobs: rows and logits of a row are fewer than 2^31")
    out = {"entropy": np.empty(n, np.float32)}
    t = None
    if targets is not None:
        targets = np.asarray(targets)
        shape = targets.shape
        if targets.dtype.kind in "iu" and targets.dtype != np.int32:
            # (what is left of an id in 32 bits could be another's)
            targets = np.where((targets >= 0) & (targets < V), targets.astype(np.int32), np.int32(-1))
        t = np.ascontiguousarray(targets, np.int32).reshape(n, -1) if shape[:1] == (n,) and len(shape) <= 2 and n else np.empty((0, 0), np.int32)
        if n and shape not in ((n,), t.shape):
            mx4._invalid("token_logprobs: targets are [n] or [n][m]")
        out["logprob"] = np.empty(shape, np.float32)
    k = min(max(int(k), -1), 65)  # (the library refuses fewer than none and more than 64)
    if k > 0:
        out["top_ids"], out["top_logprob"] = np.empty((n, k), np.int32), np.empty((n, k), np.float32)
    m = 0 if t is None else t.shape[1]
    check(lib().mg_token_logprobs(ptr(x), mx4._HOST_TYPES[x.dtype], n, V, V, ptr(t) if m else None, m, k,
                                  ptr(out["logprob"]) if m else None, ptr(out["entropy"]), ptr(out.get("top_ids")),
                                  ptr(out.get("top_logprob")), None, 0, 0, None))
    return out


def token_logprobs_device(logits, targets=None, logprob=None, entropy=None, top_ids=None, top_logprob=None):
    """The same on torch CUDA tensors, into those of the outputs that are given: logits [n][V] float32, float16 or bfloat16 (rows may be
    strided), targets int32 [n][m] with logprob float32 [n][m], entropy float32 [n], top_ids int32 and top_logprob float32 [n][k], all
    contiguous. Enqueued on torch's current stream."""
    who = "token_logprobs_device"
    ty, n, V, ld = mx4._real(who, logits, "logits")
    torch = mx4._torch
    if (targets is None) != (logprob is None):
        mx4._invalid(f"{who}: targets and logprob are given together")

    def size(a, b, name):
        """The columns of a and b, which are [n][columns] of int32 and float32."""
        shape = None
        for t, dt in ((a, torch.int32), (b, torch.float32)):
            if t is None:
                continue
            if t.dtype is not dt or t.dim() != 2 or t.shape[0] != n or not t.is_contiguous() or (shape and t.shape != shape):
                mx4._invalid(f"{who}: {name} are contiguous int32 and float32 matrices of n rows")
            shape = t.shape
        return shape[1] if shape else 0

    m, k = size(targets, logprob, "targets and logprob"), size(top_ids, top_logprob, "top_ids and top_logprob")
    if entropy is not None and (entropy.dtype is not torch.float32 or entropy.shape != (n,) or not entropy.is_contiguous()):
        mx4._invalid(f"{who}: entropy is contiguous float32 [n]")
    need = _need.get((n, V, k))
    if need is None:
        need = lib().mg_token_logprobs_workspace(n, V, k)
        check(-1 if need < 0 else 0)
        if len(_need) >= 256:
            _need.clear()
        _need[n, V, k] = need
    ws = logits.new_empty(need, dtype=torch.uint8) if need else None
    given = tuple(t for t in (targets, logprob, entropy, top_ids, top_logprob) if t is not None)
    mx4._launch(who, lib().mg_token_logprobs, None, (logits,) + given,
                (logits.data_ptr(), ty, n, V, ld, ptr(targets), m, k, ptr(logprob), ptr(entropy), ptr(top_ids), ptr(top_logprob), ptr(ws),
                 need, MG_PTR_DEVICE))
