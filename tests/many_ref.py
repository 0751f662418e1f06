"""Cache sequences gathered, attention over shared prefixes and log probabilities in numpy float64: what the GPU tests compare against."""
from __future__ import annotations

import numpy as np


def slot(p, cap, sinks):
    return p if p < sinks else sinks + (p - sinks) % (cap - sinks)


def held(length, cap, sinks):
    """The positions that a sequence of this length has in a cache."""
    return [p for p in range(length) if p < sinks or p >= length - (cap - sinks)]


def gathered(to, frm, parents, lens, from_lens=None, sinks=0, from_sinks=0):
    """Planes [n][heads][slots][bytes] after mg_kv_gather; `to` and `frm` are lists of planes, `frm` is read as it was."""
    old = [p.copy() for p in frm]
    new = [p.copy() for p in to]
    cap, from_cap = to[0].shape[2], frm[0].shape[2]
    for i, parent in enumerate(parents):
        if not 0 <= parent < len(frm[0]):
            continue
        there = set(held(lens[i] if from_lens is None else from_lens[parent], from_cap, from_sinks))
        for p in held(lens[i], cap, sinks):
            for a, b in zip(new, old):
                a[i, :, slot(p, cap, sinks)] = b[parent, :, slot(p, from_cap, from_sinks)] if p in there else 0
    return new


def softmax_rows(q, k, v, scale, p_bits):
    """One query [dh] over keys and values [N][dh]: (out, tolerance), as RefCache.attention derives it, with p_bits [N]: the bits that each
    probability is held to for the product with V, and three rescalings (a chunk's, a wave's, the prefix's) of a 2^-21 each."""
    if len(k) == 0:
        return np.zeros(q.shape), np.zeros(q.shape)
    sc = k @ q * scale
    e = np.exp(sc - sc.max())
    w = e / e.sum()
    d = abs(scale) * (len(q) + 4) * 2.0 ** -23 * (np.abs(k) @ np.abs(q)) + np.abs(sc) * 2.0 ** -22 + 2.0 ** -22
    rel = 2 * d.max() + len(k) * 2.0 ** -23 + 3 * 2.0 ** -21
    return w @ v, 2 * rel * (w @ np.abs(v)) + 2 * (w * 2.0 ** -np.asarray(p_bits, float)) @ np.abs(v)


def logprobs(x, targets, k):
    """Rows [n][V] -> dict of float64 results, and of tolerances for fp32 statistics.

    A power e = 2^((x - m) log2 e) is off by a factor of |x - m| 2^-22 (the difference and its product with log2 e are rounded, each by
    at most 2^-24, and log2 e itself is) and 2^-22 (the instruction), their sum by V 2^-24 more; log S is off by as much as S is
    relatively, and by 2^-22 of itself. The entropy has the same of X = sum (x - m) e, whose terms are rounded twice more."""
    x = np.asarray(x, np.float64)
    n, V = x.shape
    m = x.max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        far = x - m
        e = np.where(far == -np.inf, 0.0, np.exp(far))
        S = e.sum(-1, keepdims=True)
        lp = far - np.log(S)
        lp = np.where(lp < -float(np.finfo(np.float32).max), -np.inf, lp)  # as fp32 holds it: 3e38 below 3e38 is past its range
        size = np.where(e > 0, np.abs(far), 0.0)
        rel = (e * (size + 1)).sum(-1, keepdims=True) / S * 2.0 ** -22 + V * 2.0 ** -24
        X = (e * size).sum(-1, keepdims=True) / S
        relx = (e * size * (size + 2)).sum(-1, keepdims=True) / S * 2.0 ** -22 + V * 2.0 ** -24 * X
        tl = np.abs(np.log(S)) * 2.0 ** -22 + rel
        out = {"entropy": (np.log(S) + X)[:, 0]}
        tol = {"entropy": (tl + relx + X * rel + (X + np.abs(np.log(S))) * 2.0 ** -22)[:, 0]}
        row = np.where(np.isfinite(lp), np.abs(lp) + np.abs(far), 0.0) * 2.0 ** -23 + tl
    if targets is not None:
        t = np.asarray(targets)
        fine = (t >= 0) & (t < V)
        at = np.where(fine, t, 0)
        out["logprob"] = np.where(fine, np.take_along_axis(lp, at, 1), np.nan)
        tol["logprob"] = np.take_along_axis(row, at, 1)
    if k:
        # NaN below all; equal numbers in the order of their ids
        key = np.where(np.isnan(x), -np.inf, x)
        ids = np.stack([np.lexsort((np.arange(V), -key[i], np.isnan(x[i])))[:k] for i in range(n)]) if n else np.zeros((0, k), int)
        out["top_ids"], out["top_logprob"] = ids, np.take_along_axis(lp, ids, 1)
        tol["top_logprob"] = np.take_along_axis(row, ids, 1)
    return out, tol
