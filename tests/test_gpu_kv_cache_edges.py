"""Attention over the 4-bit cache where its forms differ most from each other: scores far apart, and blocks of NaN.

The forms: a wave alone with its rows, four waves that share the tiles, and more than 32 rows a head on four and on eight waves;
the second and fourth also in several workgroups that are joined."""
import numpy as np
import pytest
import torch

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
