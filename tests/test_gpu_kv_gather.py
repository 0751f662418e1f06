"""Sequences of a 4-bit cache gathered, through the C ABI: every byte of every plane as many_ref.gathered says, those that no position asks
for as they were."""
import numpy as np
import pytest
import torch

import many_ref as R
from mignon_ai_amd import KVCache, MignonError

pytestmark = pytest.mark.gpu


def make(n, heads, dh, cap, sinks=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    planes = [torch.randint(0, 256, (n, heads, cap, w), dtype=torch.uint8, generator=g).cuda() for w in (dh // 2, dh // 32) * 2]
    return KVCache(*planes, sinks=sinks)


def planes(c):
    return [t.cpu().numpy() for t in (c.k, c.k_scales, c.v, c.v_scales)]


def ints(a):
    return torch.tensor(np.array(a).tolist(), dtype=torch.int32, device="cuda")


def check(c, parents, lens, source=None, source_lens=None):
    src = c if source is None else source
    want = R.gathered(planes(c), planes(src), parents, lens, source_lens, c.sinks, src.sinks)
    c.gather(ints(parents), ints(lens), source=source, source_lens=None if source_lens is None else ints(source_lens))
    for got, w in zip(planes(c), want):
        assert np.array_equal(got, w)


MAPS = {"cycle": lambda n, r: np.roll(np.arange(n), 1), "back": lambda n, r: np.roll(np.arange(n), -1), "reverse": lambda n, r: np.arange(n)[::-1],
        "fork": lambda n, r: np.zeros(n, int), "last": lambda n, r: np.full(n, n - 1), "any": lambda n, r: r.integers(0, n, n),
        "permuted": lambda n, r: r.permutation(n), "some": lambda n, r: np.where(r.random(n) < 0.4, r.integers(0, n, n), -1),
        "halves": lambda n, r: np.arange(n) // 2, "outside": lambda n, r: r.integers(-3, n + 3, n), "same": lambda n, r: np.arange(n)}


@pytest.mark.parametrize("name", list(MAPS))
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
def test_in_place(name, dh):
    """Forks, swaps, cycles: as if from a copy. Lengths from nothing to twice around the ring."""
    for n, heads, cap, sinks in ((1, 1, 32, 0), (2, 3, 64, 5), (7, 2, 96, 0), (33, 1, 64, 1)):
        r = np.random.default_rng(n * dh)
        c = make(n, heads, dh, cap, sinks, n)
        lens = r.integers(0, 2 * cap, n)
        lens[0] = (0, 1, cap, cap - 1)[n % 4]
        check(c, MAPS[name](n, r), lens)


@pytest.mark.parametrize("n", [1025, 3000, 16384])
def test_in_place_many_sequences(n):
    r = np.random.default_rng(n)
    c = make(n, 1, 32, 32, 0, 1)
    check(c, r.permutation(n), np.full(n, 32))
    check(c, np.roll(np.arange(n), 1), r.integers(0, 40, n))


def test_in_place_shortened():
    """Less is taken than the parents hold, also of rings that have wrapped: what they lost becomes zeros."""
    c = make(5, 2, 96, 64, 3, 2)
    check(c, [1, 0, 3, 4, 4], [20, 61, 70, 5, 200], source_lens=[64, 63, 75, 500, 201])


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("cap,sinks,from_cap,from_sinks", [(64, 0, 64, 0), (96, 4, 64, 0), (32, 0, 160, 7), (64, 8, 64, 3), (32, 31, 96, 0)])
def test_from_another_cache(dh, cap, sinks, from_cap, from_sinks):
    r = np.random.default_rng(dh + cap)
    for n, m, heads in ((1, 1, 1), (6, 2, 3), (3, 9, 2)):
        c, src = make(n, heads, dh, cap, sinks, 1), make(m, heads, dh, from_cap, from_sinks, 2)
        for step in range(3):
            there = r.integers(0, 2 * from_cap, m)
            parents = r.integers(-1, m + 1, n)
            lens = np.array([r.integers(0, there[p] + 2) if 0 <= p < m else 40 for p in parents])
            check(c, parents, lens, source=src, source_lens=there)
            check(c, parents, np.minimum(lens, min(cap - sinks, from_cap - from_sinks)), source=src)
            check(c, parents, r.integers(0, 300, n), source=src)


def test_long_sequences_and_many_heads():
    r = np.random.default_rng(0)
    c = make(3, 70, 64, 1024, 4, 1)
    check(c, [2, 0, 0], [1024, 700, 3000])
    big, small = make(2, 2, 128, 20000 // 32 * 32, 0, 2), make(4, 2, 128, 4096, 4, 3)
    check(small, [1, 0, -1, 1], [15000, 3000, 9, 4097], source=big, source_lens=[3000, 15000])
    check(big, [3, 3], [4000, 4096], source=small)


def test_planes_past_32_bits():
    """Sequences whose codes lie beyond the first 4 GiB of a plane."""
    n, heads, dh, cap = 40, 8, 128, 1 << 18
    a = [torch.empty((n, heads, cap, w), dtype=torch.uint8, device="cuda") for w in (dh // 2, dh // 32) * 2]
    assert a[0].numel() > 1 << 32
    c = KVCache(*a)
    for t in a:
        for s in (0, n - 1):
            t[s, :, :2100] = torch.randint(0, 256, t[s, :, :2100].shape, dtype=torch.uint8, device="cuda")
    old = [t[n - 1].clone() for t in a]
    first = [t[0, :, :64].clone() for t in a]
    parents = np.full(n, -1)
    parents[n - 2], parents[n - 1], parents[1] = n - 1, 0, n - 1
    lens = np.full(n, 0)
    lens[n - 2], lens[n - 1], lens[1] = 2100, 64, 1999
    c.gather(ints(parents), ints(lens))
    for t, o, f in zip(a, old, first):
        assert torch.equal(t[n - 2, :, :2100], o[:, :2100]) and torch.equal(t[1, :, :1999], o[:, :1999])
        assert torch.equal(t[n - 1, :, :64], f) and torch.equal(t[n - 1, :, 64:2100], o[:, 64:2100])
    d = KVCache.empty(2, heads, dh, 2112)
    d.gather(ints([n - 2, 1]), ints([2100, 1999]), source=c)
    assert torch.equal(d.k[0, :, :2100], old[0][:, :2100]) and torch.equal(d.v_scales[1, :, :1999], old[3][:, :1999])
    assert not d.k[1, :, 1999:].any()


def test_what_was_copied_is_seen():
    """Forked sequences go on by themselves: attention over a copy is that over its parent, and writes to one leave the other."""
    c = make(4, 2, 64, 64, 2, 3)
    g = torch.Generator().manual_seed(1)
    rows = [torch.randn((4, 50, 2, 64), generator=g).cuda() for _ in range(2)]
    c.write(*rows, ints([0] * 4))
    c.gather(ints([-1, 0, 0, 2]), ints([50, 50, 30, 50]))
    q = torch.randn((1, 1, 4, 64), generator=g).cuda().expand(4, 1, 4, 64).contiguous()
    out = torch.empty_like(q)
    c.attention(q, out, ints([49, 49, 29, 49]))
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])
    before = planes(c)
    c.write(rows[0][:, :1], rows[1][:, :1], ints([50, 50, 30, 50]), ints([0, 1, 0, 0]))
    after = planes(c)
    for a, b in zip(before, after):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[2:], b[2:]) and not np.array_equal(a[1], b[1])


def test_captured_and_replayed():
    """A rotation in a graph: every replay moves on by one, eager work between."""
    n = 5
    c = make(n, 2, 96, 64, 0, 1)
    twin = KVCache(*[t.clone() for t in (c.k, c.k_scales, c.v, c.v_scales)])
    parents, lens = ints(np.roll(np.arange(n), 1)), ints([64] * n)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        make(n, 2, 96, 64).gather(parents, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.gather(parents, lens)
    for step in range(4):
        g.replay()
        twin.gather(parents, lens)
        torch.cuda.synchronize()
        for a, b in zip(planes(c), planes(twin)):
            assert np.array_equal(a, b)


def test_refusals_of_tensors():
    c, d = make(3, 2, 64, 64), make(2, 2, 64, 64)
    i = ints([0, 0, 0])
    for bad in (i.long(), i[:2], i.cpu(), ints([0, 0, 0, 0, 0, 0])[::2]):
        with pytest.raises(MignonError):
            c.gather(bad, i)
        with pytest.raises(MignonError):
            c.gather(i, bad)
    with pytest.raises(MignonError):
        c.gather(i, i, source=d, source_lens=i)
    with pytest.raises(MignonError):
        c.gather(i, i, source=make(2, 1, 64, 64))
    with pytest.raises(MignonError):
        c.gather(i, i, source=KVCache(c.k[:2], c.k_scales[:2], c.v[:2], c.v_scales[:2]))
    with pytest.raises(MignonError):
        c.gather(i, i, source=KVCache(c.k, c.k_scales, d.v.repeat(2, 1, 1, 1)[:3].contiguous(), c.v_scales))
    with pytest.raises(MignonError):
        c.gather(None, i)


def test_in_place_past_2_to_28_pieces():
    """A head's plane of more than 2^28 pieces of 16 bytes: byte offsets within it pass 32 bits."""
    cap = (1 << 28) + 64
    a = [torch.empty((2, 1, cap, w), dtype=torch.uint8, device="cuda") for w in (16, 1) * 2]
    c = KVCache(*a)
    tails = []
    for t in a:
        t[:, :, :1000] = torch.randint(0, 256, t[:, :, :1000].shape, dtype=torch.uint8, device="cuda")
        t[:, :, -1000:] = torch.randint(0, 256, t[:, :, -1000:].shape, dtype=torch.uint8, device="cuda")
        tails.append((t[:, :, :1000].clone(), t[:, :, -1000:].clone()))
    c.gather(ints([1, 0]), ints([cap, cap - 3]))
    for t, (first, last) in zip(a, tails):
        assert torch.equal(t[:, :, :1000], first.flip(0))
        assert torch.equal(t[0, :, -1000:], last[1]) and torch.equal(t[1, :, -1000:-3], last[0, :, :-3]) and torch.equal(t[1, :, -3:], last[1, :, -3:])
