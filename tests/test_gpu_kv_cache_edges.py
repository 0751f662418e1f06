"""Attention over the 4-bit cache where its forms differ most from each other: scores far apart, and blocks of NaN.

The forms: a wave alone with its rows, four waves that share the tiles, and more than 32 rows a head on four and on eight waves;
the second and fourth also in several workgroups that are joined."""
import numpy as np
import pytest
import torch

from mignon_ai_amd import KVCache
from test_gpu_kv_cache import P_BITS, Pair, _ints, _np, _rows

pytestmark = pytest.mark.gpu

# tokens a sequence, capacity, length
FORMS = {"wave": (1, 64, 60), "waves": (1, 512, 500), "waves_joined": (1, 8192, 5000), "many": (40, 128, 100),
         "many_halves": (40, 1024, 900), "many_joined": (40, 8192, 5000)}


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("t", list(P_BITS))
@pytest.mark.parametrize("dh,group", [(128, 1), (32, 3)])
@pytest.mark.parametrize("power", [12, 20, 26, 31])
def test_scores_far_apart(form, t, dh, group, power):
    """Scores up to 2^38: one key takes it all. Its probability is the only one that is not zero, so that the output is its value,
    off by the bits that a probability and the output are held to. A row counts where its best key is ahead by more than the
    sums' error (dh + 4 roundings of at most 2^-23 of the sum of magnitudes, two of the score) and fp32's smallest power."""
    T, cap, L = FORMS[form]
    H, scale = 2, 2.0 ** power
    p = Pair(1, H, dh, cap)
    p.write(_rows((1, L, H, dh), 1), _rows((1, L, H, dh), 2), [0])
    q = _rows((1, T, H * group, dh), 3, t, 2.0)
    out = torch.full_like(q, 55.0)
    p.c.attention(q, out, _ints([L - T]), scale=scale)
    k, v = (np.stack([p.r.rows[0][j][i] for j in range(L)]) for i in (0, 1))
    qn, got, sure = _np(q), _np(out), 0
    for i in range(T):
        seen = L - T + i + 1
        for h in range(H * group):
            kk, row = k[:seen, h // group], qn[0, i, h]
            sc = kk @ row
            best, second = np.argsort(sc)[::-1][:2]
            err = (dh + 4) * 2.0 ** -23 * (np.abs(kk) @ np.abs(row)).max() + 2.0 ** -22 * np.abs(sc).max()
            if (sc[best] - sc[second] - 2 * err) * scale * np.log2(np.e) < 150:
                continue
            sure += 1
            want = v[best, h // group]
            tol = np.abs(want) * (2.0 ** -P_BITS[t] + 2.0 ** -21 + torch.finfo(t).eps / 2)
            assert (np.abs(got[0, i, h] - want) <= tol).all(), (i, h, got[0, i, h], want)
    assert sure >= 0.9 * T * H * group


# tokens a sequence, capacity, length, window
SPOILT = {"wave": (1, 64, 60, 20), "waves": (1, 1024, 900, 400), "waves_wrapped": (1, 512, 700, 380), "waves_joined": (1, 8192, 5000, 4000),
          "rows": (9, 256, 200, 70), "many": (40, 128, 100, 30), "many_halves": (40, 1024, 900, 380), "many_wrapped": (40, 512, 700, 380),
          "many_joined": (40, 8192, 5000, 4000)}


@pytest.mark.parametrize("form", list(SPOILT))
@pytest.mark.parametrize("t", list(P_BITS))
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
def test_nan_reaches_only_the_rows_that_see_it(form, t, dh):
    """Blocks of NaN and infinity next to the window's end, where some rows have lost them, further on, and where only the last rows
    have them; slots that were never written are NaN in both caches. What does not see them has the same bits as without."""
    T, cap, L, window = SPOILT[form]
    n, H, G, lo = 3, 2, 2, L - T - window + 1  # the first row's first position
    k, v = _rows((n, L, H, dh), 1), _rows((n, L, H, dh), 2)
    plain, spoilt = Pair(n, H, dh, cap), Pair(n, H, dh, cap)
    plain.c.write(k, v, _ints([0] * n))
    keys = [(0, lo - 1, 0), (1, L - T + T // 2, 0)]  # sequence, position, head
    values = [(0, lo - 1, 1, dh - 1), (0, lo + T // 3, 0, 0), (2, L - T + T // 2, 1, dh - 32), (2, lo + window // 2, 0, dh // 2),
              (2, min(lo + window // 2 + 32, L - 1), 1, 31), (1, L - 1, 1, dh - 1)]  # and channel
    for i, (s, p, h) in enumerate(keys):
        k[s, p, h, 7 * i] = (np.nan, -np.inf)[i]
    for i, (s, p, h, c) in enumerate(values):
        v[s, p, h, c] = (np.inf, np.nan, -np.inf)[i % 3]
    spoilt.c.write(k, v, _ints([0] * n))
    q = _rows((n, T, H * G, dh), 3, t)
    a, b = (x.c.attention(q, torch.full_like(q, 55.0), _ints([L - T] * n), window=window) for x in (plain, spoilt))
    bad = np.zeros(q.shape, bool)
    for i in range(T):
        p = L - T + i
        for s, j, h in keys:
            bad[s, i, h * G:(h + 1) * G] |= p - window < j <= p
        for s, j, h, c in values:
            bad[s, i, h * G:(h + 1) * G, c // 32 * 32:c // 32 * 32 + 32] |= p - window < j <= p
    bad = torch.from_numpy(bad).cuda()
    assert bool(torch.isfinite(a).all())
    assert torch.equal(torch.isnan(b), bad)
    assert torch.equal(b[~bad], a[~bad])


@pytest.mark.parametrize("form", list(SPOILT))
@pytest.mark.parametrize("t", list(P_BITS))
def test_rows_replaced_by_their_outputs(form, t):
    """out may be q itself: a row is read before anything is written in its place."""
    T, cap, L, window = SPOILT[form]
    n, H, G, dh = 5, 4, 2, 64
    p = Pair(n, H, dh, cap)
    lens = np.array([L, T, L // 2, L - 3, max(1, T // 2)])
    counts = np.minimum(lens, T)
    p.c.write(_rows((n, L, H, dh), 1), _rows((n, L, H, dh), 2), _ints([0] * n), _ints(lens))
    q, pos, cnt = _rows((n, T, H * G, dh), 3, t), _ints(lens - counts), _ints(counts)
    want = p.c.attention(q, q.clone(), pos, cnt, window=window)
    assert torch.equal(p.c.attention(q, q, pos, cnt, window=window), want)


def test_counts_outside_the_call_and_sequences_without_tokens():
    """Counts are taken as 0..T; calls on no sequences or no tokens do nothing."""
    p = Pair(3, 2, 64, 64)
    k, v = _rows((3, 10, 2, 64), 1), _rows((3, 10, 2, 64), 2)
    p.c.write(k, v, _ints([0, 0, 0]), _ints([99, -5, 10]))
    q = _rows((3, 10, 4, 64), 3)
    out = p.c.attention(q, torch.full_like(q, 55.0), _ints([0, 0, 0]), _ints([99, -5, 10]))
    whole = p.c.attention(q, torch.full_like(q, 55.0), _ints([0, 0, 0]), _ints([10, 0, 10]))
    assert torch.equal(out, whole) and bool((out[1] == 55.0).all()) and bool(torch.isfinite(out).all())
    none = KVCache.empty(0, 2, 64, 64)
    empty = torch.empty((0, 3, 2, 64), device="cuda")
    none.write(empty, empty, _ints([]))
    none.read(empty, empty, _ints([]))
    assert none.attention(empty, empty, _ints([])).shape == empty.shape
    still = torch.empty((3, 0, 2, 64), device="cuda")
    p.c.write(still, still, _ints([0, 0, 0]))
    p.c.attention(still, still, _ints([0, 0, 0]))
