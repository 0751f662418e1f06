"""Attention over shared prefixes where scores far from zero are followed by ordinary ones within a prefix, against numpy in float64."""
import numpy as np
import pytest
import torch

import many_ref as R
from test_gpu_kv_shared import OWN_BITS, PREFIX_BITS, TYPES, Filled, ints, num, rows

pytestmark = pytest.mark.gpu

# Scores of the first steps of 64 positions, as powers of two: what follows them is ordinary.
STEPS = {"far": (26,), "very_far": (30,), "nearer_and_nearer": (27, 25, 22), "one_step_ordinary": (0, 26, 0, 26)}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh,T,n", [(32, 1, 4), (64, 40, 3), (96, 43, 3), (128, 1, 5), (128, 43, 3)])
@pytest.mark.parametrize("name", list(STEPS))
def test_far_scores_before_ordinary_ones(t, dh, T, n, name):
    """Positions whose scores are some -2^26 (fp32 queries: -2^36) weigh nothing beside ordinary ones, wherever they stand: every row is
    that of the ordinary positions alone. Channel 0 makes the scores far; other positions' keys have 0 there."""
    H, G, L = 2, 2, 64 * len(STEPS[name]) + 70
    more = 10 if t == torch.float32 else 0
    far = np.zeros(L, bool)

    def edit_prefix(k, v):
        k[..., 0] = 0.0
        for i, p in enumerate(STEPS[name]):
            if p:
                far[64 * i:64 * i + 64] = True
                # (query 2^13 to 2^14: the scales of these keys stay among those that fp16 holds)
                k[0, 64 * i:64 * i + 64, :, 0] = -2.0 ** (p + more - 13) * (1 + torch.arange(64.0, device="cuda")[:, None] / 64)

    def edit_own(k, v):
        k[..., 0] = 0.0
    own, prefix = Filled([T + 5] * n, H, dh, 64, 0, 1, edit=edit_own), Filled((L,), H, dh, (L + 31) // 32 * 32, 0, 5, edit=edit_prefix)
    q = rows((n, T, H * G, dh), 3, torch.float32)
    q[..., 0] = 2.0 ** 13 * (1 + torch.rand(q.shape[:3], generator=torch.Generator().manual_seed(1))).cuda()
    q = q.to(t)
    out = own.c.attention_shared(q, torch.full_like(q, 55.0), ints([5] * n), prefix.c, ints([L]), scale=1.0)
    qn, got = num(q), num(out)
    near = np.flatnonzero(~far)
    assert (prefix.k[0, near, :, 0] == 0).all() and (own.k[..., 0] == 0).all()
    for s in range(n):
        for i in range(T):
            for h in range(H * G):
                k = np.concatenate([prefix.k[0, near, h // G], own.k[s, :6 + i, h // G]])
                v = np.concatenate([prefix.v[0, near, h // G], own.v[s, :6 + i, h // G]])
                # (the far ones are at least 2^21 below, which no rounding of theirs, of 2^-22 of them, brings near)
                assert (prefix.k[0, far, h // G] @ qn[s, i, h]).max() < -2.0 ** 21
                want, tol = R.softmax_rows(qn[s, i, h], k, v, 1.0, [PREFIX_BITS[t]] * len(near) + [OWN_BITS[t]] * (6 + i))
                tol = tol + torch.finfo(t).eps / 2 * np.abs(want) + (2.0 ** -25 if t == torch.float16 else 0)
                assert (np.abs(got[s, i, h] - want) <= tol).all(), (s, i, h, np.abs(got[s, i, h] - want).max())

