"""The 4-bit format, the cache and attention over it in numpy float64: what the GPU tests compare against."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def padded(K):
    return -(-K // 128) * 128


def quantize_blocks(x):
    """Rows [..., K], K a multiple of 32 -> (code of every element, scale bytes [..., K / 32])."""
    b = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], -1, 32)
    a = np.abs(b).max(-1)
    fine = np.isfinite(a)
    e = np.frexp(np.where(fine & (a > 0), a, 1.0))[1] - 1
    s = np.where(fine, np.where(a > 0, np.maximum(e - 2 + 127, 0), 0), 255)
    y = np.ldexp(np.where(fine[..., None], b, 0.0), 127 - np.where(fine, s, 127)[..., None])
    m = np.minimum(np.abs(y), 6.0)
    up = np.searchsorted(GRID, m)                 # GRID[up - 1] < m <= GRID[up]
    lo = np.maximum(up - 1, 0)
    mid = (GRID[lo] + GRID[up]) / 2
    code = np.where(m == GRID[up], up, np.where(m > mid, up, np.where(m < mid, lo, np.where(up % 2 == 0, up, lo))))
    code = code + 8 * np.signbit(y)
    return code.reshape(np.shape(x)).astype(np.uint8), s.astype(np.uint8)


def pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def quantize(x):
    """A matrix [M][K] -> codes [M][Kp / 2], scales [M][Kp / 32], as mg_mx4_quantize defines them."""
    x = np.asarray(x)
    code, s = quantize_blocks(np.pad(x, ((0, 0), (0, padded(x.shape[1]) - x.shape[1]))))
    return pack(code), s


def values(codes, scales):
    """The float64 values of packed codes [..., K / 2] and scales [..., K / 32]."""
    code = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.repeat(scales.astype(np.int64), 32, -1)
    return np.where(s == 255, np.nan, np.ldexp(v, s - 127))


def rounded(x):
    """Rows [..., K], K a multiple of 32, as the format holds them (blocks with NaN or infinity: NaN)."""
    code, s = quantize_blocks(x)
    return values(pack(code), s)


class RefCache:
    """Positions of every sequence and head with the rows the format makes of them."""

    def __init__(self, n, heads, dh, cap, sinks):
        self.n, self.heads, self.dh, self.cap, self.sinks = n, heads, dh, cap, sinks
        self.rows = [{} for _ in range(n)]  # position -> (k [heads][dh], v)

    def write(self, k, v, pos, counts):
        k, v = rounded(np.asarray(k, np.float64)), rounded(np.asarray(v, np.float64))
        for s in range(self.n):
            for t in range(int(counts[s])):
                self.rows[s][int(pos[s]) + t] = (k[s, t], v[s, t])

    def held(self, s, p, end):
        return 0 <= p < end and (p < self.sinks or p >= end - (self.cap - self.sinks))

    def read(self, s, p, end):
        if not self.held(s, p, end):
            return np.zeros((2, self.heads, self.dh))
        return np.stack(self.rows[s][p])

    def attention(self, q, pos, counts, window, scale, p_bits):
        """(out, tolerance): float64 rows for the tokens that are there, and how far fp32 sums of any order may be off.

        A score is a sum of dh exact products in fp32, scaled and turned into a power of two: off by at most
        d = scale * (dh + 4) * 2^-23 * sum|q k| + |score| * 2^-22 + 2^-22. Then every probability is off by a factor of e^(2 d)
        at most, against the largest, held to p_bits bits for the product with V, and the sums over N keys are off by
        N * 2^-23 of sum p|v|; joined parts are rescaled once more each (2^-21)."""
        n, T, hq, dh = q.shape
        G = hq // self.heads
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        for s in range(n):
            end = int(pos[s]) + int(counts[s])
            for t in range(int(counts[s])):
                p = int(pos[s]) + t
                js = [j for j in sorted(self.rows[s]) if j <= p and self.held(s, j, end)
                      and (window <= 0 or j > p - window or j < self.sinks)]
                if not js:
                    continue
                k = np.stack([self.rows[s][j][0] for j in js])
                v = np.stack([self.rows[s][j][1] for j in js])
                for h in range(hq):
                    kk, vv, qq = k[:, h // G], v[:, h // G], np.asarray(q[s, t, h], np.float64)
                    sc = kk @ qq * scale
                    e = np.exp(sc - sc.max())
                    w = e / e.sum()
                    out[s, t, h] = w @ vv
                    d = abs(scale) * (dh + 4) * 2.0 ** -23 * (np.abs(kk) @ np.abs(qq)) + np.abs(sc) * 2.0 ** -22 + 2.0 ** -22
                    rel = 2 * d.max() + 2.0 ** -p_bits + len(js) * 2.0 ** -23 + 2.0 ** -21
                    tol[s, t, h] = rel * (w @ np.abs(vv)) * 2  # and the same for the sum that it is divided by
        return out, tol
