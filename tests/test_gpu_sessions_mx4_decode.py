"""Sets of sessions with 4-bit rings in batched decodes whose sessions end one after another: stop tokens, sampling, and what the
set holds."""
import numpy as np
import pytest

from helpers import model_bytes, uniform_model_bytes
from mignon_ai_amd import Model, _lib, engine_option, synth
from test_gpu_sampling import _replay

pytestmark = pytest.mark.gpu


class Mx4:
    """A model whose sets have 4-bit rings."""

    def __init__(self, m):
        self.sessions = lambda n: m.sessions(n, kv="mx4")


@pytest.fixture
def restore():
    prev = {k: engine_option(k, "auto") for k in ("step_kernel", "step_graph")}
    yield
    for k, v in prev.items():
        engine_option(k, v)


@pytest.mark.parametrize("kernel", ["layered", "tiled"])
@pytest.mark.parametrize("graph", ["off", "on"])
def test_stop_tokens(restore, kernel, graph):
    """A reply with stop tokens is the reply without them up to the first one, past the point where the rings wrap: 16 sessions of a
    tile end at different steps, and whole tiles before the others."""
    engine_option("step_kernel", kernel)
    engine_option("step_graph", graph)
    m, V, S, G = Model(model_bytes("c3")), synth.CONFIGS["c3"]["spec"].V, 70, 60
    prompts = synth.token_ids(8, "mx4:until", (S, 40), V)
    prompts[16:32] = prompts[16]
    lens = (np.arange(S) * 7 % 40 + 1).astype(np.int32)
    lens[16:32] = 40
    full, probs = m.sessions(S, kv="mx4").decode_greedy(prompts, G, lens)
    for stops in ([int(full[16, 3])], [int(x) for x in full[::9, 30]], [V + 5]):
        ids, pr, counts = m.sessions(S, kv="mx4").decode_greedy_until(prompts, G, stops, lens)
        for i in range(S):
            k = next((j for j, x in enumerate(full[i]) if int(x) in stops), G)
            assert counts[i] == k
            assert np.array_equal(ids[i, :k], full[i, :k]) and np.array_equal(pr[i, :k], probs[i, :k])


@pytest.mark.parametrize("kernel", ["layered", "tiled"])
def test_sampled_replies(restore, kernel):
    """Every token of a sampled decode is what the restated sampler picks from the logits of single steps of such a set."""
    engine_option("step_kernel", kernel)
    m, V, S, G = Model(model_bytes("c3")), synth.CONFIGS["c3"]["spec"].V, 20, 30
    prompts = synth.token_ids(5, "mx4:sample", (S, 50), V)
    lens = (np.arange(S) * 11 % 50 + 1).astype(np.int32)
    seeds = [1000 + 7 * i for i in range(S)]
    args = 0.8, 40, 0.9, 1.3, True
    free = _replay(Mx4(m), prompts, lens, G, seeds, *args, set())
    stops = [int(free[0][4]), int(free[3][11])]
    want = _replay(Mx4(m), prompts, lens, G, seeds, *args, set(stops))
    ids, counts = m.sessions(S, kv="mx4").decode_sample(prompts, G, seeds, *args, stops, lens)
    assert [ids[i, :counts[i]].tolist() for i in range(S)] == want and counts.min() < G


def test_device_bytes_count_the_attention_workspace():
    """Few sessions of a long window split their histories, for which the set holds memory: a share of it is each session's."""
    import ctypes
    heads, dh, context = 2, 32, 4096
    m = Model(uniform_model_bytes(synth.ModelSpec(V=64, D=heads * dh, H=64, blocks=[synth.BlockSpec(1, 2, 1)], heads=heads, window=0,
                                                  context=context), 5, 0.1))

    def workspace(n):
        c = _lib.KvCache(n, heads, dh, context, 0, *(4 * (1 << 20,)))
        return _lib.lib().mg_kv_attention_workspace(ctypes.addressof(c), heads, 1, context)

    assert workspace(3) > 0 and workspace(600) == 0
    a, b = (m.sessions(n, kv="mx4").device_bytes() for n in (3, 600))
    assert a - b == -(-workspace(3) // 3)
