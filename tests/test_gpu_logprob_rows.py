"""Log probabilities of rows in every division among waves and segments, against numpy in float64 (ids exact). The tolerances count the longest
chain of additions that a logit passes, so that a lost stretch of a long row shows."""
import numpy as np
import pytest
import torch

import many_ref as R
from mignon_ai_amd import token_logprobs, token_logprobs_device
from test_gpu_logprob import TYPES, call, rows

pytestmark = pytest.mark.gpu

# A tile of 2048 logits is added by a lane in 11 steps, and to what it has in one more, where a new maximum may put the old sums at
# another reference: by a power (2^-22), a product each (2^-24), and for X the difference of references times S (2^-23). Lanes meet in 6 steps,
# four waves in 2, 64 segments in 6, after three such rescalings. At most `tiles` tiles a wave.
def chain(tiles):
    return (25 + tiles) * 2.0 ** -24 + (tiles + 3) * 3 * 2.0 ** -22


def expected(x, targets, k, tiles):
    """R.logprobs with the additions of a chain for those of the whole row."""
    x = np.asarray(x, np.float64)
    want, tol = R.logprobs(x, targets, k)
    V = x.shape[1]
    with np.errstate(all="ignore"):
        far = x - x.max(-1, keepdims=True)
        e = np.where(far == -np.inf, 0.0, np.exp(far))
        S = e.sum(-1, keepdims=True)
        X = (e * np.where(e > 0, np.abs(far), 0.0)).sum(-1, keepdims=True) / S
        less = V * 2.0 ** -24 - chain(tiles)  # of S, and of X relatively
        for key in ("logprob", "top_logprob"):
            if key in tol:
                tol[key] = tol[key] - less
        tol["entropy"] = tol["entropy"] - (less * (1 + 2 * X))[:, 0]
    return want, tol


def check(got, want, tol, at=slice(None)):
    for key in got:
        if key == "top_ids":
            assert np.array_equal(got[key], want[key][at]), key
            continue
        a, b, c = got[key], want[key][at], tol[key][at]
        with np.errstate(invalid="ignore"):
            fine = (a == b) | (np.isnan(a) & np.isnan(b)) | (np.abs(a - b) <= c)
        assert fine.all(), (key, np.argwhere(~fine)[:3], a[~fine][:3], b[~fine][:3], c[~fine][:3])


def shapes_of_rows(V, t, seed):
    """Rows that bounds and candidates can go wrong at: ordinary ones, ties, stretches of forbidden tokens, steps up and down, NaN."""
    inf = float("inf")
    x = rows(20, V, seed, t)
    r = torch.Generator().manual_seed(seed + 1)
    up = torch.arange(V).float()
    x[4] = torch.randint(0, 4, (V,), generator=r).to(t)      # few different numbers
    x[5] = 2.5                                               # one
    x[6, :V // 2] = -inf                                     # the first half forbidden
    x[7, V // 2:] = -inf                                     # the last
    x[8, :min(2100, V - 1)] = -inf                           # more than a wave's first tile
    x[9] = (up / 64).to(t)                                   # every tile above the one before
    x[10] = (-up / 64).to(t)
    x[11] = (up // 500).to(t)                                # in steps of equal numbers
    x[12] = -inf                                             # nothing allowed
    x[13] = -inf
    x[13, V - 1] = 0.5                                       # the last token alone
    x[14, V // 3] = float("nan")
    x[15, V // 5] = inf
    x[16] = torch.finfo(t).min
    x[17, :V // 2] = torch.finfo(t).min
    x[18, ::3] = -inf
    x[19] = -inf
    x[19, ::97] = 1.0                                        # few allowed, all alike
    return x


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [2047, 2048, 2049, 4095, 4097, 5000, 6143, 8191, 8192, 8193])
@pytest.mark.parametrize("n", [2047, 2048, 2051])
def test_rows_that_a_wave_takes_alone(n, V, t):
    """Around the sizes where rows go from four waves to one: several tiles a wave, a last one that is not full, a last workgroup that
    is not full. Equal rows have equal results, wherever they stand."""
    base = shapes_of_rows(V, t, V)
    at = np.random.default_rng(n).integers(0, len(base), n)
    x = base.cuda()[torch.from_numpy(at).cuda()]
    targets = np.random.default_rng(V).integers(0, V, (len(base), 2))
    targets[3] = (-1, V)
    for k in (0, 1, 20, 64):
        check(call(x, targets[at], k), *expected(base.double().numpy(), targets, k, -(-V // 2048)), at)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,V", [(1, 16384), (1, 16385), (3, 50001), (20, 30000), (20, 100003), (255, 16500), (256, 20000), (600, 12289)])
def test_rows_that_four_waves_or_segments_take(n, V, t):
    base = shapes_of_rows(V, t, V)
    at = np.arange(n) % len(base) if n > 5 else np.array([8, 0, 6])[:n]
    x = base.cuda()[torch.from_numpy(at).cuda()]
    targets = np.random.default_rng(V).integers(0, V, (len(base), 1))
    for k in (0, 5, 64):
        check(call(x, targets[at], k), *expected(base.double().numpy(), targets, k, -(-V // 8192)), at)


@pytest.mark.parametrize("n,V", [(1, 1 << 20), (1, 300007), (2, 131072), (7, 200000), (16, 100000), (512, 65536), (2500, 8192), (2500, 2048)])
def test_a_lost_stretch_shows(n, V):
    """Equal logits: log p is -log V and the entropy log V. Then one likely token at the ends of the stretches that waves and segments
    take (all multiples of 2048 and their neighbours among the targets)."""
    x = torch.full((n, V), 3.25, device="cuda")
    places = sorted({p for a in range(0, V + 1, 2048) for p in (a - 1, a) if 0 <= p < V} | {V - 1})
    got = call(x, np.full((n, 1), V // 2), 1)
    # the reference of equal logits is met by no rescaling; log S by 2^-22 of itself, the power of 0 is 1
    tol = chain(-(-V // 2048)) + (np.log(V) + 1) * 2.0 ** -21
    for key in ("logprob", "top_logprob"):
        assert (np.abs(got[key] + np.log(V)) <= tol).all(), key
    assert (np.abs(got["entropy"] - np.log(V)) <= tol).all() and (got["top_ids"] == 0).all()
    pick = np.random.default_rng(V).permutation(places)
    for a in range(0, len(pick), n):
        some = pick[a:a + n]
        y = x[:len(some)].clone()
        y[torch.arange(len(some)), torch.from_numpy(some)] = 3.25 + 40.0
        if len(some) < n:
            y = torch.cat([y, x[len(some):]])
        got = call(y, np.resize(some, (n, 1)), 1)
        # beside e^40 all others together are V e^-40 < 2^-37
        m = len(some)
        assert (np.abs(got["logprob"][:m]) <= 2.0 ** -20).all() and (got["entropy"][:m] <= 2.0 ** -20).all()
        assert np.array_equal(got["top_ids"][:m, 0], some)


@pytest.mark.parametrize("V", [5000, 20000, 150000])
def test_rows_alone_and_in_company(V):
    """The same rows alone, in a small and in a large call: the same ids, the same sums within the tolerance of either (rows are divided
    among waves by their number, so the last bits may differ); two equal calls: the same bits."""
    x = shapes_of_rows(V, torch.float32, 3).cuda()
    many = x.repeat(2100 // len(x) + 1, 1) if V < 100000 else x.repeat(30, 1)
    _, tol = expected(x.double().cpu().numpy(), None, 16, -(-V // 2048))
    few, all_ = call(x, None, 16), call(many, None, 16)
    again = call(many, None, 16)
    for key in all_:
        assert np.array_equal(all_[key], again[key], equal_nan=key != "top_ids")
    for i in range(len(x)):
        one = call(x[i:i + 1], None, 16)
        for other in (few, all_):
            assert np.array_equal(one["top_ids"][0], other["top_ids"][i])
            for key in ("entropy", "top_logprob"):
                a, b = one[key][0], other[key][i]
                with np.errstate(invalid="ignore"):
                    assert ((a == b) | (np.isnan(a) & np.isnan(b)) | (np.abs(a - b) <= 2 * tol[key][i])).all(), (key, i)


def test_ids_past_32_bits_are_outside_the_vocabulary():
    """Host targets of any integer type: an id is what it says, not what is left of it in 32 bits."""
    x = rows(3, 50, 1).numpy()
    ids = np.array([[7, 2 ** 32 + 7, -2 ** 32 + 7], [3, 2 ** 31, 2 ** 63 - 1], [0, -2 ** 31 - 1, 49]], np.int64)
    got = token_logprobs(x, ids)["logprob"]
    want = token_logprobs(x, np.where((ids >= 0) & (ids < 50), ids, -1).astype(np.int32))["logprob"]
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(np.isnan(got), (ids < 0) | (ids >= 50))
    big = token_logprobs(x, np.array([2 ** 64 - 1, 2 ** 32, 5], np.uint64))["logprob"]
    assert np.isnan(big[:2]).all() and big[2] == token_logprobs(x, [0, 0, 5])["logprob"][2]
    assert token_logprobs(x, np.array([1, 2, 3], np.uint8))["logprob"].tolist() == token_logprobs(x, [1, 2, 3])["logprob"].tolist()


def test_more_rows_than_workgroups():
    """2^24 short rows and more: four a workgroup."""
    n, V = (1 << 24) + 5, 3
    x = torch.randn((n, V), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    entropy, ids = torch.full((n,), 77.0, device="cuda"), torch.full((n, 1), -5, dtype=torch.int32, device="cuda")
    token_logprobs_device(x, entropy=entropy, top_ids=ids)
    assert torch.equal(ids[:, 0].long(), x.argmax(-1))
    p = torch.log_softmax(x.double(), -1)
    # the statistics of three logits (R.logprobs): entropy and its parts are below 2, a logit's distance from the largest below 12
    assert float((entropy + (p.exp() * p).sum(-1)).abs().max()) <= 2 * (chain(1) + 14 * 2.0 ** -22) * 2
