"""Sets of sessions with 4-bit key and value rings (mg_sessions_create_mx4): a model of one attention block against a float64
restatement that rounds the keys and values a step attends over, past the point where the rings wrap; every way to step gives
the same bits; refusals."""
import numpy as np
import pytest

import mx4_ref
from helpers import RTOL, assert_close, model_bytes, uniform_model_bytes
from mignon_ai_amd import MignonError, Model, engine_option, synth
from oracle import oracle as O
from ref_f64 import latch_base, rmsnorm, sig

pytestmark = pytest.mark.gpu


@pytest.fixture
def restore():
    prev = engine_option("kv_rings", "auto"), engine_option("step_kernel", "auto"), engine_option("step_graph", "auto")
    yield
    for name, v in zip(("kv_rings", "step_kernel", "step_graph"), prev):
        engine_option(name, v)


def _spec(dh, heads, window, context):
    return synth.ModelSpec(V=64, D=dh * heads, H=dh * heads, blocks=[synth.BlockSpec(1, 2, 1)], heads=heads, window=window,
                           context=context)


class Ref:
    """One sequence through a model of one block of one step (step-major, float64): what attention adds at each position."""

    def __init__(self, rm, ids, max_context):
        self.rm, self.T = rm, len(ids)
        D, H, blk = rm.D, rm.H, rm.blocks[0]
        f = lambda a, *shape: np.asarray(a, np.float64).reshape(shape)
        self.emb = f(rm.embed, rm.V, D)
        cur = self.emb[ids] * float(rm.embed_scale)
        n = rmsnorm(cur, f(blk.gamma, D))
        lam = sig(n @ f(blk.wsel, D, D).T * float(blk.ssel) + latch_base(D))
        G, g = np.empty_like(n), np.zeros(D)
        for t in range(self.T):
            g = lam[t] * g + (1 - lam[t]) * n[t]
            G[t] = g
        left = np.zeros_like(n)
        left[blk.initial_dilation:] = n[:self.T - blk.initial_dilation]
        hid = np.concatenate([n, left, G], 1) @ f(blk.w1, 2 * H, 3 * D).T * float(blk.s1) + f(blk.b1, 2 * H)
        o = (hid[:, :H] * sig(hid[:, H:])) @ f(blk.w2, 2 * D, H).T * float(blk.s2) + f(blk.b2, 2 * D)
        gate = sig(o[:, D:])
        self.cur = (1 - gate) * cur + gate * o[:, :D]
        a = blk.attn
        qkv = rmsnorm(self.cur, f(a["norm"], D)) @ f(a["qkv"], 3 * D, D).T * float(a["sqkv"])
        self.q, self.k, self.v = (np.ascontiguousarray(x) for x in np.split(qkv, 3, 1))
        self.wo = f(a["wo"], D, D) * float(a["so"])
        self.cap = rm.window if rm.window > 0 else max_context

    def logits(self, t, k, v):
        rm, dh = self.rm, self.rm.D // self.rm.heads
        lo = max(0, t - self.cap + 1)
        att = np.empty(rm.D)
        for h in range(rm.heads):
            sl = slice(h * dh, (h + 1) * dh)
            s = k[lo:t + 1, sl] @ self.q[t, sl] / np.sqrt(dh)
            p = np.exp(s - s.max())
            att[sl] = p / p.sum() @ v[lo:t + 1, sl]
        fn = rmsnorm(self.cur[t] + self.wo @ att, np.asarray(rm.final_norm, np.float64))
        return self.emb @ fn * float(rm.embed_scale) + (np.asarray(rm.head_b, np.float64) if len(rm.head_b) else 0.0)


def _unsure(x):
    """What the format holds of x (rows [T][D]), and the elements that an error of the product's 1e-5 of a row's largest could
    round another way: a list of (t, column, other value)."""
    r = mx4_ref.rounded(x)
    d = 1e-5 * np.abs(x).max(1, keepdims=True)
    other = {}
    for y in (mx4_ref.rounded(x + d), mx4_ref.rounded(x - d), mx4_ref.rounded(x + d * np.sign(x)), mx4_ref.rounded(x - d * np.sign(x))):
        for t, c in zip(*np.nonzero(y != r)):
            other[t, c] = y[t, c]
    return r, [(t, c, y) for (t, c), y in other.items()]


def _against_ref(spec, S, P, lens, n):
    data = uniform_model_bytes(spec, 5, 0.1)
    rm, m = O.read_model(data), Model(data)
    context = O.OracleModel(rm).max_context  # (a context of less than 64 tokens counts as 128)
    lens = np.array(lens, np.int32)
    prompts = synth.token_ids(7, "mx4:p", (S, P), spec.V)
    steps = synth.token_ids(7, "mx4:s", (n, S), spec.V)
    ss = m.sessions(S, kv="mx4")
    first = ss.prefill(prompts, lens)[0]
    got = [ss.step(steps[i])[0] for i in range(n)]
    for s in range(S):
        ids = np.concatenate([prompts[s, :lens[s]], steps[:, s]])
        ref = Ref(rm, ids, context)
        assert_close(first[s], ref.logits(lens[s] - 1, ref.k, ref.v), what=f"session {s}, prompt")
        (k, ku), (v, vu) = _unsure(ref.k), _unsure(ref.v)
        for i in range(n):
            t = lens[s] + i
            want = ref.logits(t, k, v)
            # the parity bar, and what each element that may have been rounded the other way would change
            tol = RTOL * np.maximum(np.abs(want), np.sqrt(np.mean(want ** 2)))
            for rows, unsure, which in ((k, ku, 0), (v, vu, 1)):
                for tt, c, y in unsure:
                    if t - ref.cap < tt <= t:
                        alt = rows.copy()
                        alt[tt, c] = y
                        tol = tol + np.abs(ref.logits(t, alt, v) - want if which == 0 else ref.logits(t, k, alt) - want)
            worst = (np.abs(got[i][s] - want) / tol).max()
            assert worst <= 1, f"session {s}, step {i}: {worst} of the tolerance"


@pytest.mark.parametrize("dh,heads,window,context", [(32, 2, 16, 48), (64, 3, 0, 40), (96, 2, 33, 64), (128, 1, 5, 32),
                                                     (32, 2, 0, 64)])
def test_steps_attend_over_the_rounded_rows(restore, dh, heads, window, context):
    _against_ref(_spec(dh, heads, window, context), 3, 11, [11, 4, 1], 60)


@pytest.mark.parametrize("dh,heads,window,context", [(32, 2, 16, 64), (64, 1, 33, 100), (96, 1, 3, 64), (128, 1, 64, 96)])
def test_prompts_longer_than_the_ring(restore, dh, heads, window, context):
    """Of a prompt's rows that share a slot the later one is kept."""
    _against_ref(_spec(dh, heads, window, context), 4, 70 if context > 64 else 60, [60, 35, 33, 5], 12)


@pytest.mark.parametrize("cfg,S", [("c3", 5), ("c4", 37), ("c5", 300)])
def test_every_way_to_step_gives_the_same(restore, cfg, S):
    """Layered and tiled, from graphs or one launch at a time, and greedy decoding against single steps; past the ring's end."""
    m, V = Model(model_bytes(cfg)), synth.CONFIGS[cfg]["spec"].V
    prompts = synth.token_ids(3, "mx4:p", (S, 60), V)
    lens = 1 + np.arange(S, dtype=np.int32) * 7 % 60
    runs = {}
    for mode in ("auto", "layered", "tiled"):
        for graph in ("auto", "off"):
            engine_option("step_kernel", mode)
            engine_option("step_graph", graph)
            ss = m.sessions(S, kv="mx4")
            outs = [ss.prefill(prompts, lens)]
            for _ in range(12):
                outs.append(ss.step(np.asarray(outs[-1][1], np.int32)))
            runs[mode, graph] = outs
    engine_option("step_kernel", "auto")
    engine_option("step_graph", "auto")
    want = runs["layered", "off"]
    for key, outs in runs.items():
        for i, (x, y) in enumerate(zip(want, outs)):
            for a, b in zip(x, y):
                assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), (key, i)
    ids, _ = m.sessions(S, kv="mx4").decode_greedy(prompts, 13, lens)
    assert np.array_equal(ids, np.stack([np.asarray(o[1]) for o in want], 1))


def test_a_set_taken_again_and_its_memory(restore):
    """A prefill starts a set over: what the last conversation left is not seen. And the bytes a conversation holds."""
    m, V = Model(model_bytes("c3")), synth.CONFIGS["c3"]["spec"].V
    S = 9
    p = synth.token_ids(4, "mx4:again", (S, 20), V)
    ss, fresh = m.sessions(S, kv="mx4"), m.sessions(S, kv="mx4")
    ss.prefill(p[::-1].copy())
    for i in range(70):
        ss.step(p[:, i % 20])
    x, y = ss.prefill(p), fresh.prefill(p)
    assert np.array_equal(x[0], y[0])
    for i in range(3):
        assert np.array_equal(ss.step(p[:, i])[0], fresh.step(p[:, i])[0])
    engine_option("kv_rings", "fp32")
    plain = m.sessions(S)
    saved = 2 * 2 * 64 * 128 * 4 - 2 * 2 * 64 * (128 // 2 + 128 // 32)
    assert plain.device_bytes() - ss.device_bytes() == saved
    # the prompt's own logits are those of any set
    assert_close(x[0], plain.prefill(p)[0])


def test_models_without_attention_and_refusals(restore):
    m = Model(model_bytes("c1"))
    p = synth.token_ids(2, "mx4:c1", (4, 9), 512)
    a, b = m.sessions(4, kv="mx4"), m.sessions(4)
    assert np.array_equal(a.prefill(p)[0], b.prefill(p)[0])
    assert np.array_equal(a.step(p[:, 0])[0], b.step(p[:, 0])[0])
    with pytest.raises(ValueError):
        m.sessions(4, kv="int4")
    with pytest.raises(MignonError):
        m.sessions(0, kv="mx4")
    with pytest.raises(MignonError, match="width 24"):
        Model(uniform_model_bytes(_spec(24, 2, 8, 32), 5, 0.1)).sessions(2, kv="mx4")


def test_steps_without_allocation(restore):
    """step_noalloc, its workspace in the library's own memory, gives what a step gives."""
    import torch
    m, V = Model(model_bytes("c3")), synth.CONFIGS["c3"]["spec"].V
    S = 21
    p = synth.token_ids(6, "mx4:na", (S, 30), V)
    a, b = m.sessions(S, kv="mx4"), m.sessions(S, kv="mx4")
    a.prefill(p)
    b.prefill(p)
    for i in range(3):
        ids = torch.from_numpy(p[:, i].copy()).cuda()
        lg, am, pb = (torch.empty(s, dtype=t, device="cuda") for s, t in (((S, V), torch.float32), (S, torch.int32), (S, torch.float64)))
        b.step_noalloc(ids, lg, am, pb)
        m.sync()
        want = a.step(p[:, i])
        for x, y in zip(want, (lg, am, pb)):
            assert np.array_equal(x, y.cpu().numpy())
