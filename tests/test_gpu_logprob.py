"""Log probabilities, entropies and the likeliest tokens through the C ABI against numpy in float64 (tolerances: many_ref.logprobs; ids exact)."""
import numpy as np
import pytest
import torch

import many_ref as R
from mignon_ai_amd import MignonError, token_logprobs, token_logprobs_device

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rows(n, V, seed, t=torch.float32, size=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((n, V), generator=g) * size).to(t)


def call(x, targets=None, k=0, entropy=True):
    n = x.shape[0]
    d = {"targets": None if targets is None else torch.as_tensor(np.asarray(targets), dtype=torch.int32).cuda()}
    if targets is not None:
        d["logprob"] = torch.full(d["targets"].shape, 77.0, device="cuda")
    if entropy:
        d["entropy"] = torch.full((n,), 77.0, device="cuda")
    if k:
        d["top_ids"] = torch.full((n, k), -5, dtype=torch.int32, device="cuda")
        d["top_logprob"] = torch.full((n, k), 77.0, device="cuda")
    token_logprobs_device(x, **d)
    return {key: v.cpu().numpy() for key, v in d.items() if key != "targets" and v is not None}


def check(got, x, targets=None, k=0):
    want, tol = R.logprobs(x.double().cpu().numpy(), targets, k)
    for key in got:
        if key == "top_ids":
            assert np.array_equal(got[key], want[key]), key
            continue
        a, b = got[key], want[key]
        same = (a == b) | (np.isnan(a) & np.isnan(b))
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(a - b) <= tol[key])).all(), (key, np.nanmax(np.abs(a - b)))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 255, 1000, 1025, 4096, 8191, 32768, 32771, 50001, 131072, 300007])
def test_rows_of_all_lengths(V, t):
    """Several rows of each length, one and many alternatives and targets, targets outside the vocabulary."""
    for n, m, k in ((1, 1, min(V, 1)), (3, 2, min(V, 20)), (2, 0, min(V, 64)), (5, 3, 0)):
        x = rows(n, V, V + n, t)
        targets = np.random.default_rng(V).integers(0, V, (n, m)) if m else None
        if m > 1:
            targets[0, 0], targets[-1, -1] = -1, V
            targets[1, 0] = -2 ** 31
        check(call(x.cuda(), targets, k), x, targets, k)


@pytest.mark.parametrize("n,V", [(1, 1 << 20), (300, 8192), (4099, 257), (70000, 33)])
def test_many_rows_and_long_ones(n, V):
    x = rows(n, V, n)
    targets = np.random.default_rng(n).integers(0, V, (n, 1))
    check(call(x.cuda(), targets, 7), x, targets, 7)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,pad,offset", [(1000, 1, 0), (1001, 7, 3), (8192, 8, 1), (40000, 3, 5)])
def test_strided_rows_at_any_alignment(V, pad, offset, t):
    """Rows inside a wider buffer; what lies between them is not read as logits."""
    wide = torch.full((4, V + pad + offset), 1e4).to(t)
    x = rows(4, V, 3, t)
    wide[:, offset:offset + V] = x
    targets = [[0], [V - 1], [V // 2], [5]]
    check(call(wide.cuda()[:, offset:offset + V], targets, 9), x, targets, 9)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [70, 5000, 60000])
def test_equal_logits_go_by_id(V, t):
    """Everything equal; few different values; both zeros; the largest ones all at one place of every lane's share or side by side."""
    k = 64
    few = torch.randint(0, 4, (1, V), generator=torch.Generator().manual_seed(1)).to(t)
    zeros = torch.zeros((1, V), dtype=t)
    zeros[0, ::3] = -0.0
    up, down = torch.zeros((1, V)), torch.zeros((1, V))
    up[0, V - 70:] = torch.arange(70.0)
    down[0, :70] = 70 - torch.arange(70.0)
    stride = torch.zeros((1, V))
    stride[0, ::64] = 5.0 + (torch.arange(len(range(0, V, 64))) % 7)
    ramp = torch.arange(V).float()[None] / 64
    x = torch.cat([torch.full((1, V), 2.5).to(t), few, zeros, up.to(t), down.to(t), stride.to(t), ramp.to(t), -ramp.to(t)])
    check(call(x.cuda(), None, k), x, None, k)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [5, 3000, 70001])
def test_infinities_and_nan(V, t):
    """Forbidden tokens, rows with nothing allowed or one token allowed, the type's lowest value as a mask, positive infinity, NaN."""
    low, inf, nan = torch.finfo(t).min, float("inf"), float("nan")
    x = rows(8, V, 5, t)
    x[0, ::2] = -inf
    x[1] = -inf
    x[2] = -inf
    x[2, V // 2] = 1.0
    x[3, 1:] = low
    x[4] = low
    x[5, V - 1] = inf
    x[6, 2] = nan
    x[7] = nan
    targets = np.array([[0, 1]] * 7 + [[1, 4]])
    k = min(V, 5)
    got = call(x.cuda(), targets, k)
    check(got, x, targets, k)
    assert np.isnan(got["entropy"][[1, 5, 6, 7]]).all() and np.isnan(got["logprob"][[1, 5, 6, 7]]).all()
    assert got["entropy"][2] == 0.0 and got["logprob"][0, 0] == -np.inf


def test_far_apart_and_large_logits():
    """One token takes it all; logits near the type's largest; all nearly equal."""
    x = rows(4, 4001, 9)
    x[0, 77] = 1e30
    x[1] *= 1e30
    x[2] = 3e38
    x[2, 5] = -3e38
    x[3] = 1000.0 + x[3] * 1e-3
    targets = [[77], [0], [5], [9]]
    check(call(x.cuda(), targets, 20), x, targets, 20)


def test_outputs_are_optional_and_host_arrays():
    x = rows(3, 999, 2)
    every = call(x.cuda(), [[1], [2], [3]], 4)
    one = call(x.cuda(), None, 4, entropy=False)
    assert np.array_equal(one["top_ids"], every["top_ids"]) and np.array_equal(one["top_logprob"], every["top_logprob"])
    ids = torch.empty((3, 4), dtype=torch.int32, device="cuda")
    token_logprobs_device(x.cuda(), top_ids=ids)
    assert np.array_equal(ids.cpu().numpy(), every["top_ids"])
    host = token_logprobs(x.numpy(), np.array([1, 2, 3]), 4)
    assert host["logprob"].shape == (3,)
    for key, v in every.items():
        assert np.array_equal(host[key].reshape(v.shape), v), key
    half = token_logprobs(x.half().numpy(), np.array([[1, 2]] * 3))
    assert set(half) == {"entropy", "logprob"}
    check(half, x.half(), np.array([[1, 2]] * 3))
    assert token_logprobs(np.zeros((0, 5), np.float32), np.zeros(0, np.int32), 2)["top_ids"].shape == (0, 2)
    token_logprobs_device(torch.empty((0, 5), device="cuda"), entropy=torch.empty(0, device="cuda"))


def test_the_same_bits_again_and_in_any_company():
    """A row's results do not depend on the call it is in, nor on the run."""
    x = rows(40, 20000, 4).cuda()
    a, b = call(x, None, 16), call(x, None, 16)
    for key in a:
        assert np.array_equal(a[key], b[key])


def test_captured_and_replayed():
    """A graph replayed on new logits between eager calls of other shapes, and two graphs replayed in turn."""
    xs = [rows(2, 131072, i).cuda() for i in range(4)]
    x, y = xs[0].clone(), rows(1, 200000, 8).cuda()
    outs, graphs = [], []
    side = torch.cuda.Stream()
    for z in (x, y):
        o = {"entropy": torch.empty(len(z), device="cuda"), "top_ids": torch.empty((len(z), 20), dtype=torch.int32, device="cuda"),
             "top_logprob": torch.empty((len(z), 20), device="cuda")}
        with torch.cuda.stream(side):
            token_logprobs_device(z, **o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            token_logprobs_device(z, **o)
        outs.append(o)
        graphs.append(g)
    for new in xs:
        x.copy_(new)
        call(rows(3, 5000, 1).cuda(), None, 3)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, z in zip(outs, (x, y)):
            want = call(z, None, 20)
            for key in want:
                assert np.array_equal(o[key].cpu().numpy(), want[key])


def test_two_streams_at_once():
    xs = [rows(4, 150000, i).cuda() for i in range(2)]
    want = [call(x, None, 20) for x in xs]
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in xs]
    for x, s in zip(xs, streams):
        o = [{"top_ids": torch.empty((4, 20), dtype=torch.int32, device="cuda"), "top_logprob": torch.empty((4, 20), device="cuda"),
              "entropy": torch.empty(4, device="cuda")} for _ in range(5)]
        outs.append(o)
    torch.cuda.synchronize()
    for r in range(5):
        for x, s, o in zip(xs, streams, outs):
            with torch.cuda.stream(s):
                token_logprobs_device(x, **o[r])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        for r in range(5):
            for key in w:
                assert np.array_equal(o[r][key].cpu().numpy(), w[key])


def test_refusals_of_tensors():
    x = rows(2, 10, 1).cuda()
    with pytest.raises(MignonError):
        token_logprobs_device(x, entropy=torch.empty(2))
    with pytest.raises(MignonError):
        token_logprobs_device(x, top_ids=torch.empty((2, 11), dtype=torch.int32, device="cuda"))
    with pytest.raises(MignonError):
        token_logprobs_device(x[:, ::2], entropy=torch.empty(2, device="cuda"))
