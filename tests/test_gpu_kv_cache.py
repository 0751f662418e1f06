"""The 4-bit key/value cache through the C ABI against numpy in float64: rows written, read back, and attention over them.

What is written is exact (see test_gpu_mx4.py). Attention is held to RefCache.attention's tolerance, the arithmetic of fp32
sums, with the probabilities held to 24 bits for fp32 queries and to 16 for the 16-bit types (two bf16 parts), plus half a
step of the output's type."""
import numpy as np
import pytest
import torch

import mx4_ref as R
from mignon_ai_amd import KVCache, MignonError

pytestmark = pytest.mark.gpu
P_BITS = {torch.float32: 23, torch.float16: 16, torch.bfloat16: 16}


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _rows(shape, seed, t=torch.float32, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * size).to(t).cuda()


def _np(t):
    return t.double().cpu().numpy()


class Pair:
    """A cache on the GPU, its planes full of garbage, and the reference beside it."""

    def __init__(self, n, heads, dh, cap, sinks=0, garbage=255):
        planes = [torch.full((n, heads, cap, w), garbage, dtype=torch.uint8, device="cuda") for w in (dh // 2, dh // 32) * 2]
        self.c, self.r = KVCache(*planes, sinks=sinks), R.RefCache(n, heads, dh, cap, sinks)

    def write(self, k, v, pos, counts=None):
        self.c.write(k, v, _ints(pos), None if counts is None else _ints(counts))
        self.r.write(_np(k), _np(v), pos, [k.shape[1]] * self.r.n if counts is None else counts)

    def fill(self, lens, seed, T=64, t=torch.float32):
        """Sequences grown to their lengths, T tokens a call."""
        done = np.zeros(self.r.n, int)
        while (done < lens).any():
            cnt = np.minimum(np.asarray(lens) - done, T)
            shape = (self.r.n, T, self.r.heads, self.r.dh)
            self.write(_rows(shape, seed + int(done.max()), t), _rows(shape, seed + 500 + int(done.max()), t), done, cnt)
            done = done + cnt

    def check(self, q, pos, counts=None, window=0, scale=None):
        n, T, hq, dh = q.shape
        cnt = [T] * n if counts is None else counts
        out = torch.full_like(q, 55.0)
        self.c.attention(q, out, _ints(pos), None if counts is None else _ints(counts), window=window, scale=scale)
        want, tol = self.r.attention(_np(q), pos, cnt, window, dh ** -0.5 if scale is None else scale, P_BITS[q.dtype])
        tol = tol + torch.finfo(q.dtype).eps / 2 * np.abs(want) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
        got = _np(out)
        for s in range(n):
            assert (np.abs(got[s, :cnt[s]] - want[s, :cnt[s]]) <= tol[s, :cnt[s]]).all(), (s, np.abs(got - want).max())
            assert (got[s, cnt[s]:] == 55.0).all()
        return out


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("t", list(P_BITS))
def test_write_and_read(dh, t):
    """Calls of several sizes from empty to twice around the ring, padded rows, slices of one projection; what is read is the
    held positions' values, zeros elsewhere, and rows past the counts stay."""
    n, H, cap, sinks = 3, 2, 64, 5
    p = Pair(n, H, dh, cap, sinks)
    pos, rng = np.zeros(n, int), np.random.default_rng(dh)
    for step, T in enumerate((1, 7, 40, 64, 200, 1, 33)):
        qkv = _rows((n, T, 3, H, dh), 10 * dh + step, t)
        cnt = np.minimum(rng.integers(0, T + 1, n), T) if step % 2 else np.full(n, T)
        p.write(qkv[:, :, 1], qkv[:, :, 2], pos, cnt if step % 2 else None)
        pos = pos + cnt
    span = int(pos.max()) + 3
    k, v = (torch.full((n, span, H, dh), 77.0, dtype=t, device="cuda") for _ in range(2))
    counts = np.minimum(pos + 1, span - 1)
    p.c.read(k, v, _ints(np.zeros(n)), _ints(counts), _ints(pos))
    for s in range(n):
        want = np.stack([p.r.read(s, i, pos[s]) for i in range(span)], 1)
        for got, w in ((k, want[0]), (v, want[1])):
            w = torch.from_numpy(w).to(t)
            assert torch.equal(got[s, :counts[s]].cpu(), w[:counts[s]])
            assert bool((got[s, counts[s]:] == 77.0).all())


def test_one_call_longer_than_the_ring():
    """Two tokens of a call with one slot: the later one is kept, whatever order the lanes run in."""
    p = Pair(2, 3, 64, 32, 4)
    p.write(_rows((2, 300, 3, 64), 1), _rows((2, 300, 3, 64), 2), [0, 17], [300, 299])
    k, v = (torch.empty((2, 320, 3, 64), device="cuda") for _ in range(2))
    p.c.read(k, v, _ints([0, 0]), None, _ints([300, 316]))
    for s, end in ((0, 300), (1, 316)):
        held = {i: r for i, r in p.r.rows[s].items()}
        for i in range(320):
            fine = p.r.held(s, i, end) and i in held
            if fine:
                assert np.array_equal(_np(k[s, i]), held[i][0]) and np.array_equal(_np(v[s, i]), held[i][1])


SHAPES = [  # heads, group, dh, capacity, sinks, window, lengths
    (2, 1, 32, 64, 0, 0, (1, 2, 31, 64)),
    (1, 1, 32, 64, 0, 64, (150, 64, 65, 1000)),
    (2, 4, 128, 256, 0, 0, (1, 33, 200, 256)),
    (1, 5, 96, 96, 3, 40, (5, 95, 97, 300)),
    (3, 2, 64, 160, 40, 100, (20, 41, 160, 777)),
    (1, 16, 64, 64, 1, 1, (1, 2, 64, 65)),
    (1, 20, 32, 1024, 4, 700, (1, 705, 1024, 1500)),
    (2, 1, 128, 32, 31, 0, (31, 32, 33, 400)),
]


@pytest.mark.parametrize("heads,group,dh,cap,sinks,window,lens", SHAPES)
@pytest.mark.parametrize("t", list(P_BITS))
def test_decode(heads, group, dh, cap, sinks, window, lens, t):
    p = Pair(len(lens), heads, dh, cap, sinks)
    p.fill(lens, 7, t=t)
    q = _rows((len(lens), 1, heads * group, dh), 3, t, 2.0)
    p.check(q, np.asarray(lens) - 1, window=window)
    # an idle sequence, and other scales
    for scale in (0.25, -0.25, 0.0):
        p.check(q, np.asarray(lens) - [1, 0, 1, 0], [1, 0, 1, 0], window, scale)


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("t", list(P_BITS))
@pytest.mark.parametrize("T,group,sinks,window", [(2, 1, 0, 0), (5, 3, 2, 9), (17, 4, 0, 0), (65, 1, 3, 30), (130, 2, 0, 1)])
def test_chunks(dh, t, T, group, sinks, window):
    """Several rows a sequence, as after a prompt's part was written, of unequal numbers."""
    n, heads, cap = 3, 2, 256
    p = Pair(n, heads, dh, cap, sinks)
    lens = np.array([T, T + 3, 200 if T < 200 else T])
    counts = np.array([T, T // 2, T])
    p.fill(lens, 11, t=t)
    q = _rows((n, T, heads * group, dh), 5, t, 2.0)
    for scale in (None, -0.25, 0.0):
        p.check(q, lens - counts, counts, window, scale)


@pytest.mark.parametrize("t", list(P_BITS))
@pytest.mark.parametrize("T", [1, 40])
def test_chunk_over_a_ring_that_lost_what_its_first_rows_saw(t, T):
    """A ring shorter than the window and the call: rows see what is still held, some of them only the sinks or nothing."""
    p = Pair(2, 1, 64, 32, 0)
    p.fill([100, 60], 3, T=T, t=t)
    p.check(_rows((2, 40, 1, 64), 4, t), [60, 20], [40, 40], 5)
    p = Pair(2, 1, 64, 32, 2)
    p.fill([100, 60], 3, T=T, t=t)
    p.check(_rows((2, 40, 1, 64), 4, t), [60, 20], [40, 40], 5)


@pytest.mark.parametrize("t", list(P_BITS))
def test_rows_before_the_first_position_see_nothing(t):
    """Negative positions have no keys: zeros."""
    p = Pair(1, 1, 32, 32)
    p.fill([4], 3, t=t)
    out = p.check(_rows((1, 7, 1, 32), 4, t), [-3], [7])
    assert float(out[0, :3].abs().max()) == 0


@pytest.mark.parametrize("T", [1, 33])
def test_long_history_is_split_and_joined(T):
    p = Pair(2, 2, 128, 8192, 4)
    rng = np.random.default_rng(1)
    k, v = (torch.from_numpy(rng.standard_normal((2, 8000, 2, 128)).astype(np.float32)).cuda() for _ in range(2))
    p.write(k, v, [0, 0], [8000, 3777])
    for t in P_BITS:
        q = _rows((2, T, 8, 128), 6, t, 3.0)
        for window in (0, 3000):
            p.check(q, [8000 - T, 3777 - T], window=window)


@pytest.mark.parametrize("T", [1, 40])
def test_nan_and_infinity_reach_only_the_rows_that_see_them(T):
    """A key and a value block with NaN or infinity, behind the window, in it, and after some of the rows."""
    n, dh, L = 4, 64, 96
    k, v = _rows((n, L, 2, dh), 1), _rows((n, L, 2, dh), 2)
    plain = Pair(n, 2, dh, 128)
    plain.write(k, v, [0] * n)
    k[0, 10, 0, 3], v[0, 11, 1, 40] = np.nan, np.inf      # outside the window of every row
    k[1, 90, 0, 3] = np.inf                               # rows from 90 on see it
    v[2, 90, 1, 40] = np.nan                              # the same, channels 32 to 63 only
    spoilt = Pair(n, 2, dh, 128)
    spoilt.write(k, v, [0] * n)
    q = _rows((n, T, 4, dh), 3)
    a, b = (p.c.attention(q, torch.empty_like(q), _ints([L - T] * n), window=30) for p in (plain, spoilt))
    for s in range(n):
        for i in range(T):
            hit = L - T + i >= 90
            for h in range(4):
                bad = torch.zeros(dh, dtype=torch.bool)
                if s == 1 and hit and h < 2:
                    bad[:] = True
                if s == 2 and hit and h >= 2:
                    bad[32:] = True
                got = b[s, i, h].cpu()
                assert torch.equal(torch.isnan(got), bad), (s, i, h)
                assert torch.equal(got[~bad], a[s, i, h].cpu()[~bad])


def test_large_scores():
    """Scores far apart and of either sign: one key takes it all, no overflow on the way."""
    p = Pair(2, 1, 32, 64)
    k = _rows((2, 50, 1, 32), 1, size=1e4)
    p.write(k, _rows((2, 50, 1, 32), 2), [0, 0])
    q = _rows((2, 1, 2, 32), 3, size=1e4)
    out = p.c.attention(q, torch.empty_like(q), _ints([49, 49]))
    for s in range(2):
        for h in range(2):
            best = max(range(50), key=lambda j: float(p.r.rows[s][j][0][0] @ _np(q[s, 0, h])))
            assert np.array_equal(_np(out[s, 0, h]), p.r.rows[s][best][1][0])


@pytest.mark.parametrize("offset", [0, 1])
def test_strided_rows(offset):
    """q and out as slices of wider rows, at any element offset."""
    n, T, H, dh = 2, 3, 2, 64
    p = Pair(n, H, dh, 64)
    p.fill([30, 64], 1)
    flat = _rows((n * T * 5 * H * dh + 8,), 2)
    wide = flat[offset:offset + n * T * 5 * H * dh].view(n, T, 5, H, dh)
    q = wide[:, :, 1:3].reshape(n, T, 2 * H, dh)
    out = torch.zeros_like(flat)
    o = out[offset:offset + n * T * 5 * H * dh].view(T, n, 5 * H, dh).transpose(0, 1)[:, :, :2 * H]
    p.c.attention(wide.view(n, T, 5 * H, dh)[:, :, H:3 * H], o, _ints([27, 61]))
    want, tol = p.r.attention(_np(q), [27, 61], [T, T], 0, dh ** -0.5, 23)
    assert (np.abs(_np(o) - want) <= tol + 2.0 ** -24 * np.abs(want)).all()
    o.zero_()
    assert float(out.abs().max()) == 0
    k = out[offset:offset + n * T * 2 * H * dh].view(n, T, 2, H, dh)
    k.copy_(_rows(k.shape, 9))
    p.write(k[:, :, 0], k[:, :, 1], [30, 64])
    back = torch.zeros(flat.shape, device="cuda")[offset:offset + k.numel()].view(k.shape)
    p.c.read(back[:, :, 0], back[:, :, 1], _ints([30, 64]))
    assert np.array_equal(_np(back), R.rounded(_np(k)))


def test_planes_beyond_32_bit_offsets():
    """Planes of more than 2^32 bytes: the last sequence's last head."""
    n, H, dh, cap = 2, 17, 128, 1 << 21
    c = KVCache.empty(n, H, dh, cap)
    assert c.k.numel() > 1 << 32
    first = cap - 40
    k, v, q = (_rows((n, 60, H, dh), i) for i in (1, 2, 3))
    c.write(k, v, _ints([first] * n))  # over the ring's end
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    c.read(ko, vo, _ints([first] * n))
    assert np.array_equal(_np(ko), R.rounded(_np(k))) and np.array_equal(_np(vo), R.rounded(_np(v)))
    assert int(c.k[0, 0, 20:-40].max()) == 0 and int(c.k[0, :, 100].max()) == 0
    r = R.RefCache(1, 1, dh, cap, 0)
    r.write(_np(k[-1:, :, -1:]), _np(v[-1:, :, -1:]), [first], [60])
    out = c.attention(q[:, -1:], torch.empty_like(q[:, -1:]), _ints([first + 59] * n), window=50)
    want, tol = r.attention(_np(q[-1:, -1:, -1:]), [first + 59], [1], 50, dh ** -0.5, 23)
    # the reference holds the call's own tokens only: the window reaches no further
    assert (np.abs(_np(out[-1:, :, -1:]) - want) <= tol + 2.0 ** -24 * np.abs(want)).all()


def test_a_step_captured_and_replayed():
    """Write, attend and advance as a decode loop does, captured once and replayed: every replay equals the eager step on a
    second cache; two graphs of one cache have workspaces of their own."""
    n, H, G, dh, cap = 3, 2, 4, 64, 4096
    a, b = KVCache.empty(n, H, dh, cap, sinks=2), KVCache.empty(n, H, dh, cap, sinks=2)
    k, v = _rows((n, 4000, H, dh), 1), _rows((n, 4000, H, dh), 2)
    start = _ints([0, 0, 0])
    for c in (a, b):
        c.write(k, v, start, _ints([4000, 1000, 10]))
    x = torch.empty((n, 1, (G + 2) * H, dh), device="cuda")
    pos = _ints([4000, 1000, 10])
    out, out2 = torch.empty((n, 1, G * H, dh), device="cuda"), torch.empty((n, 1, G * H, dh), device="cuda")

    def step(c, out, window):
        c.write(x[:, :, G * H:(G + 1) * H], x[:, :, (G + 1) * H:], pos)
        c.attention(x[:, :, :G * H], out, pos, window=window)

    x.copy_(_rows(x.shape, 5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, out, 0)
    torch.cuda.current_stream().wait_stream(side)
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(a, out, 0)
    with torch.cuda.graph(g2):
        step(a, out2, 2000)
    for i in range(4):
        x.copy_(_rows(x.shape, 20 + i))
        want, want2 = torch.empty_like(out), torch.empty_like(out)
        step(b, want, 0)
        step(b, want2, 2000)
        g.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want2)
        assert torch.equal(a.k, b.k) and torch.equal(a.v_scales, b.v_scales)
        pos += 1


def test_results_are_the_same_bits_every_time():
    """No sum depends on the order in which workgroups end."""
    n, H, dh = 5, 2, 64
    p = Pair(n, H, dh, 512, 3)
    p.fill([500, 77, 600, 1, 300], 1)
    q = _rows((n, 1, 4, dh), 2)
    pos = _ints([499, 76, 599, 0, 299])
    whole = p.c.attention(q, torch.empty_like(q), pos, window=200)
    again = p.c.attention(q, torch.empty_like(q), pos, window=200)
    assert torch.equal(whole, again)


def test_refusals():
    c = KVCache.empty(2, 2, 64, 64)
    q, pos = torch.zeros((2, 1, 2, 64), device="cuda"), _ints([0, 0])
    for bad in (lambda: KVCache.empty(2, 2, 48, 64), lambda: KVCache.empty(2, 2, 64, 64, sinks=64),
                lambda: KVCache(c.k, c.k_scales, c.v[:1], c.v_scales), lambda: KVCache(c.k[:, :, ::2], c.k_scales, c.v, c.v_scales),
                lambda: KVCache(c.k.cpu(), c.k_scales, c.v, c.v_scales), lambda: KVCache(c.k, c.v, c.v, c.v_scales),
                lambda: c.write(q[:, :, :1], q[:, :, :1], pos), lambda: c.write(q, q.half(), pos), lambda: c.write(q[:1], q[:1], pos),
                lambda: c.write(q, q, pos.long()), lambda: c.write(q, q, pos[:1]), lambda: c.write(q, q, pos.cpu()),
                lambda: c.write(q, q, None), lambda: c.write(q.cpu(), q.cpu(), pos), lambda: c.write(q.transpose(2, 3), q, pos),
                lambda: c.read(q, q, pos, pos.float()), lambda: c.read(q, q, pos, None, pos.long()),
                lambda: c.attention(q[:, :, :1], q[:, :, :1].clone(), pos), lambda: c.attention(q, q.half(), pos),
                lambda: c.attention(q.double(), q.double(), pos), lambda: c.attention(q, torch.zeros((2, 1, 4, 64), device="cuda"), pos)):
        with pytest.raises(MignonError):
            bad()


def test_sizes_that_the_interface_cannot_hold_are_refused():
    """Shapes of tensors that stand for more elements than they have, and windows past 32 bits."""
    c = KVCache.empty(1, 2, 32, 64)
    wide = torch.zeros(1, 1, 2, 32, device="cuda").expand(1, (1 << 32) + 1, 2, 32)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for call in (lambda: c.write(wide, wide, pos), lambda: c.read(wide, wide, pos), lambda: c.attention(wide, wide, pos)):
        with pytest.raises(MignonError):
            call()
    for sinks in (-1, 64, (1 << 32) + 1):
        with pytest.raises(MignonError):
            KVCache.empty(1, 2, 32, 64, sinks=sinks)
    x = torch.randn(1, 40, 2, 32, device="cuda")
    c.write(x, x, pos)
    q = torch.randn(1, 40, 2, 32, device="cuda")
    whole = c.attention(q, torch.empty_like(q), pos)
    for window in ((1 << 32) + 1, 1 << 31, -(1 << 33), np.int64(40)):
        assert torch.equal(c.attention(q, torch.empty_like(q), pos, window=window), whole)


def test_a_cache_keeps_its_planes():
    """The tensors a cache was made of live as long as it, whatever becomes of its attributes."""
    c, d = KVCache.empty(1, 2, 32, 64), KVCache.empty(1, 2, 32, 64)
    x = torch.randn(1, 3, 2, 32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.write(x, x, pos)
    d.write(x, x, pos)
    c.k = c.v = None
    junk = [torch.full((1, 2, 64, 16), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    assert torch.equal(c.attention(x, torch.empty_like(x), pos), d.attention(x, torch.empty_like(x), pos))
    del junk


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("t", list(P_BITS))
@pytest.mark.parametrize("L,cap,window,sinks", [(481, 512, 0, 0), (700, 1152, 90, 5), (1100, 1152, 520, 33), (1300, 1152, 0, 7)])
def test_many_rows_over_long_histories(dh, t, L, cap, window, sinks):
    """Tiles shared by the two halves of a workgroup, odd and even numbers of them, one of them with nothing to see for some rows;
    lengths apart, one of them of a single token."""
    n, T, H, G = 3, 35, 2, 2
    lens = np.array([L, 31, 1])
    p = Pair(n, H, dh, cap, sinks)
    p.fill(lens, dh, T=256, t=t)
    counts = np.minimum(lens, T)
    p.check(_rows((n, T, H * G, dh), 9, t, 2.0), lens - counts, counts, window)


def test_two_streams_at_once():
    """Calls that need workspaces, on two streams at the same time, over one cache: each gives what it gives alone."""
    c = KVCache.empty(2, 2, 64, 8192)
    for p in (c.k, c.v):
        p.random_(0, 256)
    for p in (c.k_scales, c.v_scales):
        p.random_(120, 126)
    qs = [_rows((2, T, 4, 64), T, torch.float16) for T in (1, 1, 40, 40)]
    pos = [_ints([8192 - q.shape[1], 5000]) for q in qs]
    alone = [c.attention(q, torch.empty_like(q), p) for q, p in zip(qs, pos)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        outs = [torch.empty_like(q) for q in qs]
        torch.cuda.synchronize()
        for s, q, o, p in zip(streams, qs, outs, pos):
            with torch.cuda.stream(s):
                c.attention(q, o, p)
        torch.cuda.synchronize()
        for a, b in zip(alone, outs):
            assert torch.equal(a, b)
