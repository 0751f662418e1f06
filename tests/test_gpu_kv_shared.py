"""Attention over shared prefixes through the C ABI against numpy in float64 (tolerance: many_ref.softmax_rows, plus half a step of the
output's type). Probabilities are held to 24 bits for fp32 queries; for the 16-bit types to 16 bits over a sequence's own positions
and to 11 over a prefix."""
import numpy as np
import pytest
import torch

import many_ref as R
import mx4_ref as X
from mignon_ai_amd import KVCache, MignonError, token_logprobs_device

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
OWN_BITS = {torch.float32: 23, torch.float16: 16, torch.bfloat16: 16}
PREFIX_BITS = {torch.float32: 23, torch.float16: 11, torch.bfloat16: 11}


def ints(a):
    return torch.tensor(np.array(a).tolist(), dtype=torch.int32, device="cuda")


def rows(shape, seed, t=torch.float32, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * size).to(t).cuda()


def num(t):
    return t.double().cpu().numpy()


class Filled:
    """A cache full of garbage with sequences of the given lengths written into it, and what it holds of them."""

    def __init__(self, lens, heads, dh, cap, sinks=0, seed=0, size=1.0, edit=None):
        n, L = len(lens), max(1, max(lens))
        planes = [torch.full((n, heads, cap, w), 255, dtype=torch.uint8, device="cuda") for w in (dh // 2, dh // 32) * 2]
        self.c, self.lens, self.sinks, self.cap = KVCache(*planes, sinks=sinks), list(lens), sinks, cap
        k, v = rows((n, L, heads, dh), seed, size=size), rows((n, L, heads, dh), seed + 1, size=size)
        if edit:
            edit(k, v)
        for a in range(0, L, 256):  # (a call's rows that fall out of the ring at once would not be written)
            cnt = [min(max(x - a, 0), 256) for x in lens]
            self.c.write(k[:, a:a + 256], v[:, a:a + 256], ints([a] * n), ints(cnt))
        self.k, self.v = X.rounded(num(k)), X.rounded(num(v))

    def held(self, s, length=None):
        return R.held(self.lens[s] if length is None else length, self.cap, self.sinks)


def reference(own, prefix, prefix_lens, starts, q, pos, counts, window, scale):
    n, T, hq, dh = q.shape
    qn, G = num(q), hq // own.c.heads
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(n):
        g = [g for g in range(len(prefix_lens)) if starts[g] <= s < starts[g + 1]]
        end = pos[s] + counts[s]
        far = prefix.held(g[0], min(prefix_lens[g[0]], prefix.cap)) if g else []
        for t in range(counts[s]):
            p = pos[s] + t
            js = [j for j in own.held(s, end) if j <= p and (window <= 0 or j > p - window or j < own.sinks)]
            bits = [PREFIX_BITS[q.dtype]] * len(far) + [OWN_BITS[q.dtype]] * len(js)
            for h in range(hq):
                k, v = own.k[s, js, h // G], own.v[s, js, h // G]
                if g:
                    k = np.concatenate([prefix.k[g[0], far, h // G], k])
                    v = np.concatenate([prefix.v[g[0], far, h // G], v])
                out[s, t, h], tol[s, t, h] = R.softmax_rows(qn[s, t, h], k, v, scale, bits)
    return out, tol


def check(own, prefix, starts, q, pos, counts, window=0, scale=None, prefix_lens=None, none=False):
    lens = prefix.lens if prefix_lens is None else prefix_lens
    out = torch.full_like(q, 55.0)
    got = own.c.attention_shared(q, out, ints(pos), prefix.c, ints(lens), starts=None if none else ints(starts), counts=ints(counts),
                                 window=window, scale=scale)
    assert got is out
    want, tol = reference(own, prefix, lens, starts, q, pos, counts, window, q.shape[3] ** -0.5 if scale is None else scale)
    tol = tol + torch.finfo(q.dtype).eps / 2 * np.abs(want) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    got = num(out)
    for s in range(q.shape[0]):
        c = counts[s]
        assert (np.abs(got[s, :c] - want[s, :c]) <= tol[s, :c]).all(), (s, np.abs(got[s, :c] - want[s, :c]).max())
        assert (got[s, c:] == 55.0).all()
    return out


# heads, group, tokens, own capacity, sinks, window, own lengths, the prefixes' capacity and lengths, first sequences
SHAPES = {
    "one": (1, 1, 1, 32, 0, 0, (1,), 32, (1,), (0, 1)),
    "pair": (2, 1, 1, 64, 0, 0, (1, 40), 64, (33,), (0, 2)),
    "empty_prefix": (2, 2, 1, 64, 0, 0, (5, 40, 1), 64, (0, 64), (0, 2, 3)),
    "lengths": (2, 3, 1, 64, 0, 0, (5, 40, 1, 7, 64, 20, 2), 96, (31, 32, 95, 96, 1), (0, 1, 2, 4, 6, 7)),
    "past_capacity": (1, 4, 1, 32, 0, 0, (5, 9), 64, (500,), (0, 2)),
    "without": (2, 2, 1, 64, 0, 0, (5, 40, 1, 7, 64), 160, (70, 9, 3), (1, 3, 3, 4)),
    "ring": (3, 2, 1, 64, 4, 30, (500, 64, 65, 3, 31), 320, (300, 290), (0, 3, 5)),
    "tokens": (2, 4, 5, 96, 3, 40, (5, 40, 7, 200), 320, (129, 310), (0, 1, 4)),
    "wide_group": (1, 20, 3, 64, 0, 0, (5, 60), 640, (600,), (0, 2)),
    "many": (2, 4, 40, 128, 0, 0, (40, 100, 128), 352, (340,), (0, 3)),
    "crowd": (2, 1, 1, 32, 0, 0, tuple(range(1, 151)), 288, (257, 40, 100), (0, 129, 140, 150)),
    "joined": (1, 2, 1, 1024, 0, 0, (1000, 30), 2048, (2000,), (0, 2)),
    "many_joined": (1, 5, 33, 1024, 2, 700, (900, 40), 1024, (1000, 5), (0, 1, 2)),
}


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
def test_against_float64(name, t, dh):
    H, G, T, cap, sinks, window, lens, p_cap, p_lens, starts = SHAPES[name]
    own = Filled(lens, H, dh, cap, sinks, 1)
    prefix = Filled([min(x, p_cap) for x in p_lens], H, dh, p_cap, 0, 11)
    counts = [min(T, x) if s != 1 or len(lens) < 4 else 0 for s, x in enumerate(lens)]
    if T > 1 and len(lens) > 2:
        counts[2] = max(1, counts[2] - 1)
    own_lens = [x - min(T, x) + c for x, c in zip(lens, counts)]  # (rows past the count were written all the same: not seen)
    pos = [x - c for x, c in zip(own_lens, counts)]
    q = rows((len(lens), T, H * G, dh), 21, t)
    check(own, prefix, starts, q, pos, counts, window, prefix_lens=p_lens)
    if len(p_lens) == 1 and starts == (0, len(lens)):
        check(own, prefix, starts, q, pos, counts, window, scale=-0.3, prefix_lens=p_lens, none=True)


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_rows_replaced_by_their_outputs(t):
    """Queries and outputs as slices of wider rows, heads before tokens, every element's alignment; out may be q."""
    own, prefix = Filled((20, 33, 7), 2, 64, 64, 0, 1), Filled((200,), 2, 64, 224, 0, 5)
    counts, pos = [3, 2, 1], [17, 31, 6]
    q = rows((3, 3, 4, 64), 9, t)
    want = check(own, prefix, (0, 3), q, pos, counts)
    wide = torch.zeros((3, 4, 3, 64 * 3 + 1), dtype=t, device="cuda")
    view = wide[..., 65:129].transpose(1, 2)
    view.copy_(q)
    to = torch.full((3, 3, 4 * 64 + 3), 55.0, dtype=t, device="cuda")[:, :, 1:257].unflatten(2, (4, 64))
    lens, cnt, at = ints(prefix.lens), ints(counts), ints(pos)
    assert torch.equal(own.c.attention_shared(view, to, at, prefix.c, lens, counts=cnt), want)
    again = q.clone()
    own.c.attention_shared(again, again, at, prefix.c, lens, counts=cnt)
    for s, c in enumerate(counts):
        assert torch.equal(again[s, :c], want[s, :c]) and torch.equal(again[s, c:], q[s, c:])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh", [32, 96, 128])
@pytest.mark.parametrize("T,n", [(1, 3), (1, 40), (40, 3)])
def test_prefixes_that_wrapped(t, dh, T, n):
    """A prefix longer than its cache: the sinks and the ring's last positions are there, in whatever order."""
    own = Filled([T + 2] * n, 1, dh, 64, 0, 1)
    prefix = Filled((500, 260), 1, dh, 256, 5, 7)
    starts = (0, n // 2, n)
    q = rows((n, T, 3, dh), 3, t)
    out = torch.empty_like(q)
    own.c.attention_shared(q, out, ints([2] * n), prefix.c, ints([500, 260]), starts=ints(starts))
    want, tol = reference(own, Wrapped(prefix), [500, 260], starts, q, [2] * n, [T] * n, 0, dh ** -0.5)
    tol = tol + torch.finfo(t).eps / 2 * np.abs(want) + (2.0 ** -25 if t == torch.float16 else 0)
    assert (np.abs(num(out) - want) <= tol).all()


class Wrapped:
    def __init__(self, f):
        self.k, self.v, self.cap, self.lens, self._f = f.k, f.v, f.cap, f.lens, f

    def held(self, s, length):
        return self._f.held(s)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -24, 2.0 ** -14, 2.0 ** 14, 2.0 ** 40])
@pytest.mark.parametrize("T,n", [(1, 4), (50, 4)])
def test_values_of_all_sizes(t, dh, size, T, n):
    """Prefix values far from one, all or in some blocks: the result is as exact, relative to them. fp16 outputs hold fp16's range only."""
    if t == torch.float16 and size > 2.0 ** 12:
        size = 2.0 ** 10

    def edit(k, v):
        v[0, :, 0] *= size
        v[0, 100:, 1, :32] *= size
    own = Filled([T] * n, 2, dh, 64, 0, 1)
    prefix = Filled((190,), 2, dh, 192, 0, 7, edit=edit)
    check(own, prefix, (0, n), rows((n, T, 4, dh), 3, t), [0] * n, [T] * n)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 18])
def test_keys_of_all_sizes(t, size):
    own = Filled([1] * 4, 2, 64, 64, 0, 1)

    def edit(k, v):
        k[0, :, 0] *= size
        k[0, 50:60, 1, :32] *= size
    prefix = Filled((190,), 2, 64, 192, 0, 7, edit=edit)
    scale = 0.125 if size < 1 else 0.125 / size
    check(own, prefix, (0, 4), rows((4, 1, 4, 64), 3, t), [0] * 4, [1] * 4, scale=scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh,T", [(128, 1), (32, 1), (64, 40)])
@pytest.mark.parametrize("power", [12, 20, 26, 31])
def test_scores_far_apart(t, dh, T, power):
    """Scores up to 2^38: one key takes it all, in the prefix or among the row's own. A row counts where its best key is ahead by more
    than the sums' error (dh + 4 roundings of at most 2^-23 of the sum of magnitudes, two of the score) and fp32's smallest power."""
    n, H, G, scale = 3, 2, 2, 2.0 ** power
    own, prefix = Filled([T + 30] * n, H, dh, 128, 0, 1), Filled((400,), H, dh, 416, 0, 5)
    q = rows((n, T, H * G, dh), 3, t, 2.0)
    out = torch.full_like(q, 55.0)
    own.c.attention_shared(q, out, ints([30] * n), prefix.c, ints([400]), scale=scale)
    qn, got, sure = num(q), num(out), 0
    for s in range(n):
        for i in range(T):
            for h in range(H * G):
                js = list(range(31 + i))
                kk = np.concatenate([prefix.k[0, :, h // G], own.k[s, js, h // G]])
                vv = np.concatenate([prefix.v[0, :, h // G], own.v[s, js, h // G]])
                sc = kk @ qn[s, i, h]
                best, second = np.argsort(sc)[::-1][:2]
                err = (dh + 4) * 2.0 ** -23 * (np.abs(kk) @ np.abs(qn[s, i, h])).max() + 2.0 ** -22 * np.abs(sc).max()
                if (sc[best] - sc[second] - 2 * err) * scale * np.log2(np.e) < 150:
                    continue
                sure += 1
                bits = PREFIX_BITS[t] if best < 400 else OWN_BITS[t]
                tol = np.abs(vv[best]) * (2.0 ** -bits + 3 * 2.0 ** -21 + torch.finfo(t).eps / 2)
                assert (np.abs(got[s, i, h] - vv[best]) <= tol).all(), (s, i, h)
    assert sure >= 0.8 * n * T * H * G


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("T,n", [(1, 4), (1, 90), (40, 4)])
def test_nan_reaches_only_the_rows_that_see_it(t, dh, T, n):
    """A block of NaN in one prefix's keys, one in another's values, and in a sequence's own: other rows keep their bits. What lies
    behind a prefix's length is NaN in every case."""
    H, G, starts = 2, 2, (0, n // 4, n // 2, n)
    key, value, mine = (0, 77, 1), (1, 200, 0, dh - 1), n - 1

    def edit_prefix(k, v):
        k[key[0], key[1], key[2], 5] = np.nan
        v[value[0], value[1], value[2], value[3]] = np.inf

    def edit_own(k, v):
        v[mine, T - 1, 1, 0] = np.nan

    make = [(Filled([T] * n, H, dh, 64, 0, 1, edit=e), Filled((210, 230, 211), H, dh, 256, 0, 5, edit=p))
            for e, p in ((None, None), (edit_own, edit_prefix))]
    q = rows((n, T, H * G, dh), 3, t)
    a, b = (o.c.attention_shared(q, torch.full_like(q, 55.0), ints([0] * n), p.c, ints(p.lens), starts=ints(starts)) for o, p in make)
    bad = np.zeros(q.shape, bool)
    bad[starts[0]:starts[1], :, key[2] * G:(key[2] + 1) * G] = True
    bad[starts[1]:starts[2], :, value[2] * G:(value[2] + 1) * G, value[3] // 32 * 32:] = True
    bad[mine, T - 1, G:, :32] = True
    bad = torch.from_numpy(bad).cuda()
    assert bool(torch.isfinite(a).all())
    assert torch.equal(torch.isnan(b), bad)
    assert torch.equal(b[~bad], a[~bad])


def test_counts_lengths_and_starts_outside_their_range():
    """Counts are taken as 0..T, prefix lengths as 0..capacity, first sequences as 0..n; calls on nothing do nothing."""
    own, prefix = Filled((10, 10, 10), 2, 64, 64, 0, 1), Filled((96, 40), 2, 64, 96, 0, 5)
    q = rows((3, 10, 4, 64), 3)

    def run(lens, starts, counts):
        return own.c.attention_shared(q, torch.full_like(q, 55.0), ints([0] * 3), prefix.c, ints(lens), starts=ints(starts), counts=ints(counts))
    a, b = run([2 ** 31 - 1, -5], [-7, 2, 99], [99, -5, 10]), run([96, 0], [0, 2, 3], [10, 0, 10])
    assert torch.equal(a, b) and bool((a[1] == 55.0).all()) and bool(torch.isfinite(a).all())
    plain = own.c.attention(q, torch.full_like(q, 55.0), ints([0] * 3))
    assert torch.equal(run([0, 0], [0, 2, 3], [10] * 3), plain) and torch.equal(run([96, 40], [0, 0, 0], [10] * 3), plain)
    nothing = KVCache.empty(0, 2, 64, 32)
    assert torch.equal(own.c.attention_shared(q, torch.full_like(q, 55.0), ints([0] * 3), nothing, ints([]), starts=ints([0])), plain)
    e = torch.empty((0, 3, 4, 64), device="cuda")
    assert nothing.attention_shared(e, e, ints([]), prefix.c, ints([96, 40]), starts=ints([0, 0, 0])).shape == e.shape
    e = torch.empty((3, 0, 4, 64), device="cuda")
    own.c.attention_shared(e, e, ints([0] * 3), prefix.c, ints([96, 40]), starts=ints([0, 2, 3]))


def test_a_row_that_sees_nothing_is_zero():
    """An empty prefix and a sequence whose positions are all behind its end."""
    own, prefix = Filled((5, 5), 1, 64, 32, 0, 1), Filled((0,), 1, 64, 32, 0, 5)
    q = rows((2, 1, 2, 64), 3)
    out = own.c.attention_shared(q, torch.full_like(q, 55.0), ints([-1, 4]), prefix.c, ints([0]))
    assert not out[0].any() and out[1].any()


def test_prefix_past_32_bits():
    """A prefix whose codes lie beyond the first 4 GiB of its plane."""
    m, H, dh, cap = 40, 8, 128, 1 << 18
    planes = [torch.empty((m, H, cap, w), dtype=torch.uint8, device="cuda") for w in (dh // 2, dh // 32) * 2]
    far, near = KVCache(*planes), Filled((300,), H, dh, 320, 0, 5)
    far.gather(ints([-1] * (m - 1) + [0]), ints([0] * (m - 1) + [300]), source=near.c)
    own, q = Filled((3, 4), H, dh, 32, 0, 1), rows((2, 1, H, dh), 3, torch.bfloat16)
    out = own.c.attention_shared(q, torch.empty_like(q), ints([2, 3]), far, ints([0] * (m - 1) + [300]), starts=ints([0] * m + [2]))
    want, tol = reference(own, near, [300], (0, 2), q, [2, 3], [1, 1], 0, dh ** -0.5)
    assert (np.abs(num(out) - want) <= tol + 2.0 ** -8 * np.abs(want)).all()


def test_captured_and_replayed():
    """Lengths, starts and queries change between replays; two graphs in turn, eager calls of another shape between."""
    own, prefix = Filled((60, 33, 50, 8), 2, 128, 64, 0, 1), Filled((900, 700), 2, 128, 1024, 0, 5)
    other = Filled((30, 30), 2, 128, 32, 0, 9)
    graphs, outs, args = [], [], []
    side = torch.cuda.Stream()
    for n, f in ((4, own), (2, other)):
        a = dict(q=rows((n, 1, 8, 128), n, torch.bfloat16), pos=ints([7] * n), lens=ints([900, 700]), starts=ints([0, 1, n]))
        out = torch.empty_like(a["q"])

        def call(a=a, out=out, f=f):
            f.c.attention_shared(a["q"], out, a["pos"], prefix.c, a["lens"], starts=a["starts"])
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
        outs.append(out)
        args.append(a)
    for step in range(4):
        for a in args:
            n = a["q"].shape[0]
            a["q"].copy_(rows(a["q"].shape, 30 + step, torch.bfloat16))
            a["lens"].copy_(ints([900 - 250 * step, 1 + 200 * step]))
            a["starts"].copy_(ints([0, step % (n + 1), n]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, out, f in zip(args, outs, (own, other)):
            want = f.c.attention_shared(a["q"], torch.empty_like(out), a["pos"], prefix.c, a["lens"], starts=a["starts"])
            assert torch.equal(out, want)


def test_two_streams_at_once():
    own, prefix = Filled([40] * 6, 2, 64, 64, 0, 1), Filled((3000,), 2, 64, 3008, 0, 5)
    qs = [rows((6, 1, 4, 64), i, torch.float16) for i in range(2)]
    pos, lens = ints([39] * 6), ints([3000])
    want = [own.c.attention_shared(q, torch.empty_like(q), pos, prefix.c, lens) for q in qs]
    outs, streams = [[torch.empty_like(q) for _ in range(5)] for q in qs], [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for r in range(5):
        for q, o, s in zip(qs, outs, streams):
            with torch.cuda.stream(s):
                own.c.attention_shared(q, o[r], pos, prefix.c, lens)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)


def test_refusals_of_tensors():
    own, prefix = Filled((3, 4), 2, 64, 32, 0, 1), Filled((9, 9), 2, 64, 32, 0, 5)
    q, pos, lens, starts = rows((2, 1, 4, 64), 3), ints([2, 3]), ints([9, 9]), ints([0, 1, 2])
    f = own.c.attention_shared
    for bad in (dict(starts=starts[:2]), dict(starts=starts.long()), dict(starts=None), dict(lens=ints([9])), dict(lens=ints([9, 9]).cpu()),
                dict(q=q[:, :, :3]), dict(q=q.double()), dict(pos=None), dict(lens=None), dict(prefix=Filled((9, 9), 1, 64, 32).c),
                dict(prefix=Filled((9, 9), 2, 32, 32).c)):
        a = dict(q=q, pos=pos, lens=lens, starts=starts, prefix=prefix.c)
        a.update(bad)
        with pytest.raises(MignonError):
            f(a["q"], torch.empty_like(a["q"]), a["pos"], a["prefix"], a["lens"], starts=a["starts"])


def test_a_beam_search():
    """The operators together: beams over a shared prompt; their candidates from the logits' likeliest tokens, the cache reordered by
    the beams' parents, the next step's attention over prompt and own tokens. Every beam's score is that of its tokens, recomputed
    from nothing in float64 along its whole path."""
    V, H, dh, W, steps, P = 301, 2, 64, 6, 12, 150
    D = H * dh
    g = torch.Generator().manual_seed(5)
    table, wk, wv, wq, wo = (torch.randn(s, generator=g) * D ** -0.5 for s in ((V, D), (D, D), (D, D), (D, D), (V, D)))
    table, wo = table * D ** 0.5, wo * 3
    prompt = torch.randint(0, V, (P,), generator=g)
    heads = lambda x: x.view(1, -1, H, dh).contiguous().cuda()
    prefix, own = KVCache.empty(1, H, dh, P), KVCache.empty(W, H, dh, 32)
    x = table[prompt]
    prefix.write(heads(x @ wk), heads(x @ wv), ints([0]))
    tokens, score, path, moved = [int(prompt[-1])] * W, np.zeros(W), [[] for _ in range(W)], 0
    for step in range(steps):
        x = table[tokens]
        k, v, q = (y.view(W, 1, H, dh).contiguous().cuda() for y in (x @ wk, x @ wv, x @ wq))
        pos = ints([step] * W)
        own.write(k, v, pos)
        out = own.attention_shared(q, torch.empty_like(q), pos, prefix, ints([P]))
        logits = (out.view(W, D).cpu() + x) @ wo.t()
        ids, lp = torch.empty((W, W), dtype=torch.int32, device="cuda"), torch.empty((W, W), device="cuda")
        token_logprobs_device(logits.cuda(), top_ids=ids, top_logprob=lp)
        total = score[:, None] + num(lp)
        if step == 0:
            total[1:] = -np.inf  # (all beams are one as yet)
        best = np.argsort(-total, axis=None, kind="stable")[:W]
        parents, which = best // W, best % W
        ids = ids.cpu().numpy()
        tokens = [int(ids[p, w]) for p, w in zip(parents, which)]
        path = [path[p] + [t] for p, t in zip(parents, tokens)]
        score = total.reshape(-1)[best]
        own.gather(ints(parents), ints([step + 1] * W))
        moved += step > 0 and int((parents != np.arange(W)).sum())
    assert len(set(map(tuple, path))) == W and moved
    f64 = lambda t: t.double().numpy()
    E, WO = f64(table), f64(wo)
    project = lambda ids, w: f64(table[ids] @ w).reshape(-1, H, dh)
    pk, pv = X.rounded(project(prompt, wk)), X.rounded(project(prompt, wv))
    for b in range(W):
        seq, want = [int(prompt[-1])] + path[b], 0.0
        k, v, q = project(seq, wk), project(seq, wv), project(seq, wq)
        k, v = X.rounded(k), X.rounded(v)
        for i in range(steps):
            o = np.zeros((H, dh))
            for h in range(H):
                o[h] = R.softmax_rows(q[i, h], np.concatenate([pk[:, h], k[:i + 1, h]]), np.concatenate([pv[:, h], v[:i + 1, h]]),
                                      dh ** -0.5, 23)[0]
            z = WO @ (o.reshape(-1) + E[seq[i]])
            want += z[path[b][i]] - z.max() - np.log(np.exp(z - z.max()).sum())
        # fp32 throughout: twelve steps, each with logits of a few tens from sums of D products (D 2^-24 of the sum of magnitudes,
        # which |o + x| |w|, some 128 x 1 x 0.3, bounds by 50): 12 * 2 * 50 * 128 * 2^-24 = 9e-3
        assert abs(want - score[b]) <= 9e-3, (b, want, score[b])


@pytest.mark.parametrize("t", TYPES)
def test_many_prefixes(t):
    """More prefixes than a wave has lanes, most of them of few sequences or none, some longer than a workgroup's rows."""
    r = np.random.default_rng(3)
    m, n = 150, 420
    starts = np.sort(np.concatenate([[2], r.integers(0, n, m - 20), np.full(19, 100)]))
    starts = np.concatenate([starts, [n - 1]])
    starts[-30:-1] = np.minimum(starts[-30:-1], 200)  # (one prefix has the last two hundred)
    starts = np.sort(starts)
    own = Filled(r.integers(1, 20, n).tolist(), 1, 32, 32, 0, 1)
    prefix = Filled(r.integers(0, 70, m).tolist(), 1, 32, 96, 0, 5)
    q = rows((n, 1, 2, 32), 9, t)
    check(own, prefix, starts.tolist(), q, [x - 1 for x in own.lens], [1] * n)


def test_tokens_without_a_count_and_scale_zero():
    """counts None: all rows; a scale of zero: all positions alike; a negative window: none."""
    own, prefix = Filled([9, 5], 2, 32, 64, 0, 1), Filled((40,), 2, 32, 64, 0, 5)
    q = rows((2, 3, 2, 32), 9)
    out = own.c.attention_shared(q, torch.empty_like(q), ints([6, 2]), prefix.c, ints([40]), window=-3, scale=0.0)
    want, tol = reference(own, prefix, [40], (0, 2), q, [6, 2], [3, 3], 0, 0.0)
    assert (np.abs(num(out) - want) <= tol + 2.0 ** -24 * np.abs(want)).all()
