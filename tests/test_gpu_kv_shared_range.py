"""Attention over shared prefixes where numbers leave the ordinary range within a prefix: scores far from zero that are followed by ordinary
ones, and blocks of the least scale (byte 0), against numpy in float64."""
import numpy as np
import pytest
import torch

import many_ref as R
from test_gpu_kv_shared import OWN_BITS, PREFIX_BITS, TYPES, Filled, check, ints, num, rows

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


LEAST = 2.0 ** -127  # the scale of byte 0


def least(shape, seed):
    """Values of 4 and 6 times the least scale, of either sign: blocks of byte 0, ordinary numbers in fp32 and bf16."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(2, 4, shape, generator=g).float() * torch.sign(torch.rand(shape, generator=g) - 0.5) * 2.0 ** -126).cuda()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dh,T,n", [(32, 1, 4), (64, 40, 3), (96, 43, 3), (128, 1, 5), (128, 43, 3)])
@pytest.mark.parametrize("where", ["all", "some"])
def test_values_of_the_least_scale(t, dh, T, n, where):
    """Prefix values of blocks with scale byte 0 and codes that are not zero. One position of the prefix has all the weight (its score is
    256 above the others: a power of theirs is 0 in fp32), so the result is that position's values."""
    H, G, L, best = 2, 2, 150, 77

    def edit(k, v):
        k[:] = 0.0
        k[0, best, :, 0] = 2.0
        x = least(v.shape, 9)
        if where == "all":
            v[:] = x
        else:
            v[:, 60:90, 1, dh - 32:] = x[:, 60:90, 1, dh - 32:]

    def edit_own(k, v):
        k[:], v[:] = 0.0, 0.0
    own, prefix = Filled([T] * n, H, dh, 64, 0, 1, edit=edit_own), Filled((L,), H, dh, 160, 0, 5, edit=edit)
    assert (prefix.v[0, best, 1, dh - 32:] != 0).all()
    q = torch.zeros((n, T, H * G, dh))
    q[..., 0] = 128.0
    q = q.to(t).cuda()
    out = num(own.c.attention_shared(q, torch.full_like(q, 55.0), ints([0] * n), prefix.c, ints([L]), scale=1.0))
    for h in range(H * G):
        want = prefix.v[0, best, h // G]
        tol = np.abs(want) * (2.0 ** -PREFIX_BITS[t] + 3 * 2.0 ** -21 + torch.finfo(t).eps / 2)
        assert (np.abs(out[:, :, h] - want) <= tol).all(), h


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh,T,n", [(32, 1, 4), (128, 1, 5), (128, 43, 3)])
def test_keys_of_the_least_scale(t, dh, T, n):
    """Prefix keys of scale byte 0 under a factor that makes ordinary scores of them."""
    H, G, L = 2, 2, 150

    def edit(k, v):
        k[:] = least(k.shape, 9)

    def edit_own(k, v):
        k[:] = 0.0
    own, prefix = Filled([T] * n, H, dh, 64, 0, 1, edit=edit_own), Filled((L,), H, dh, 160, 0, 5, edit=edit)
    assert (prefix.k[0] != 0).all()
    q = rows((n, T, H * G, dh), 3, t, 512.0)
    check(own, prefix, (0, n), q, [0] * n, [T] * n, scale=2.0 ** 115)


def test_zeros_of_the_least_scale_cost_nothing_and_count():
    """Blocks of zeros have byte 0 as well: plain zeros among ordinary values."""
    for t in TYPES:
        def edit(k, v):
            k[:, 10:100, 0] = 0.0
            v[:, 20:130, 1] = 0.0
            v[:, 140:, 0] = -0.0
        own, prefix = Filled([3] * 4, 2, 64, 32, 0, 1), Filled((150,), 2, 64, 160, 0, 5, edit=edit)
        check(own, prefix, (0, 4), rows((4, 3, 4, 64), 3, t), [0] * 4, [3] * 4)
