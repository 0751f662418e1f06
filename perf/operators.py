"""The 4-bit operators, timed over their public entry points and in plain form.

Numbers are held in the microscaled 4-bit format: blocks of 32 neighbouring elements, each element one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (code = sign bit 8 + index of the magnitude; element 2i in the low half of byte i),
each block with a power of two 2^(s - 127), s one byte, taken from its largest magnitude a: 2^(floor(log2 a) - 2), at least
2^-127. An element is rounded to the nearest value, ties to the even code, and beyond 6 to 6.

kinds
  quantize   mx4_quantize_device and mx4_dequantize_device: rows into 4 bits and back; returns the values they stand for
  product    mx4_gemm_device: C = A W^T of two 4-bit matrices, both with K along the rows (padded with zeros to a multiple
             of 128)
  write      KVCache.write and KVCache.read: new key and value rows into a 4-bit cache, at their positions; returns the
             values the cache then holds for them
  attention  KVCache.attention: queries over a 4-bit cache, causal, with a sliding window and a few first positions
             (sinks) that stay visible

A cache holds n sequences of H key/value heads: positions below `sinks` have slots of their own, later ones take turns in
the other slots (a ring). Query t of a sequence sits at position pos + t; `counts` says how many of the T rows are there.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def _kv(name, kind, n, T, H, G, dh, L, cap, type, window=0, sinks=0, ragged=True):
    return {"name": name, "kind": kind, "n": n, "T": T, "H": H, "G": G, "dh": dh, "L": L, "cap": cap, "type": type,
            "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # the activations of a few decoding sessions before a product: one short launch each way
        {"name": "quantize_rows", "kind": "quantize", "M": 16, "K": 384, "type": "f32"},
        # a long batch's activations
        {"name": "quantize_batch", "kind": "quantize", "M": 16384, "K": 4096, "type": "bf16"},
        # the vocabulary's logits for one token of the largest benchmark model
        {"name": "product_token", "kind": "product", "M": 1, "K": 384, "N": 8192, "type": "f32"},
        # the rule's product (three state rows in, two hidden rows out) over a prompt of odd length
        {"name": "product_ragged", "kind": "product", "M": 1001, "K": 1152, "N": 2048, "type": "f32"},
        # a large layer over a long batch
        {"name": "product_batch", "kind": "product", "M": 16384, "K": 4096, "N": 4096, "type": "bf16"},
        # a decode step of the benchmark's session set writes its token
        _kv("write_step", "write", 4096, 1, 8, 1, 32, 64, 64, "f32", ragged=False),
        # prompts of unequal length are taken in
        _kv("write_prompts", "write", 16, 2048, 8, 1, 128, 2048, 2048, "bf16"),
        # the decode step of the benchmark's session set: many short windows
        _kv("attention_set", "attention", 4096, 1, 8, 1, 32, 150, 64, "f32", window=64),
        # one conversation with a long history
        _kv("attention_one", "attention", 1, 1, 8, 4, 128, 30000, 30016, "f16", ragged=False),
        # a batch of long histories, grouped heads
        _kv("attention_long", "attention", 32, 1, 8, 4, 128, 16384, 16384, "bf16"),
        # endless streams in constant memory: a window and four sinks, the ring long since wrapped
        _kv("attention_stream", "attention", 256, 1, 8, 2, 64, 5000, 1056, "f16", window=1000, sinks=4),
        # a prompt's next thousand tokens over what the cache holds
        _kv("attention_chunk", "attention", 2, 1024, 8, 4, 128, 8192, 8192, "bf16", sinks=4, window=6000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "write", "attention", "attention", "attention"))
    c = {"kind": kind, "type": rng.choice(("f32", "f16", "bf16"))}
    if kind == "quantize":
        c.update(M=_log(rng, 1, 65536), K=_log(rng, 1, 8192))
        while c["M"] * c["K"] > 1 << 24:
            c["M"] = max(1, c["M"] // 2)
        return c
    if kind == "product":
        c.update(M=rng.choice((_log(rng, 1, 32), _log(rng, 1, 16384))), K=_log(rng, 16, 8192), N=_log(rng, 16, 16384))
        while c["M"] * c["K"] * c["N"] > 1 << 37:
            c["M"] = max(1, c["M"] // 2)
        return c
    H, dh, T = rng.choice((1, 2, 4, 6, 8)), rng.choice((32, 64, 96, 128)), 1
    G = 1 if kind == "write" else rng.choice((1, 1, 2, 4, 5, 8))
    sinks = rng.choice((0, 0, 1, 4, 40))
    if kind == "write":
        T, L = rng.choice((1, _log(rng, 2, 2048))), _log(rng, 2, 4096)
        window, cap = 0, -(-(sinks + rng.choice((max(L // 2, T), L)) + 1) // 32) * 32
        n = _log(rng, 1, max(1, min(4096, (1 << 25) // (max(T, 32) * H * dh), (1 << 28) // (cap * H * dh))))
    else:
        T, L = rng.choice((1, 1, _log(rng, 2, 1024))), _log(rng, 1, 32768)
        window = rng.choice((0, _log(rng, 1, L)))
        cap = -(-(sinks + (min(window + T, L) if window else L) + 1) // 32) * 32
        n = _log(rng, 1, max(1, min(4096, (1 << 28) // (cap * H * dh))))
        n = max(1, min(n, (1 << 28) // (H * G * T * cap)))
    c.update(n=n, T=T, H=H, G=G, dh=dh, L=L, cap=cap, window=window, sinks=sinks, ragged=rng.random() < 0.7)
    return c


def _lengths(c):
    """Every sequence's length after the call's tokens, and how many of its T rows are there: lengths are even or spread
    from one to L, and one in eight of the spread sequences has nothing to do in this call."""
    rng = random.Random(repr((c["n"], c["T"], c["L"])))
    lens = [c["L"]] * c["n"]
    if c["ragged"]:
        lens = [rng.randint(1, c["L"]) for _ in lens]
        lens[0] = c["L"]
    counts = [min(c["T"], n) for n in lens]
    if c["ragged"]:
        counts = [0 if i and rng.random() < 0.125 else k for i, k in enumerate(counts)]
    return np.array(lens), np.array(counts)


# ---- the format ----------------------------------------------------------------------------------------------------
def _codes(x):
    """float32 rows [..., K], K a multiple of 32 -> codes uint8 [..., K] (one element each), scale bytes [..., K / 32]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = b.abs().amax(-1)
    s = ((a.view(torch.int32) >> 23) - 2).clamp(min=0)  # the exponent's bits are floor(log2 a) + 127
    up = ((254 - s) << 23).view(torch.float32)          # 2^(127 - s), exact
    y = b * up[..., None]
    m = y.abs()
    # the borders between the eight magnitudes; a tie goes to the even code
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code += (y < 0).to(torch.uint8) * 8
    return code.reshape(x.shape), s.to(torch.uint8)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


_tables = {}


def _table(device):
    if device not in _tables:
        v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        _tables[device] = torch.tensor(v + [-x for x in v], dtype=torch.float32, device=device)
    return _tables[device]


def _values(packed, scales):
    """Packed codes [..., K / 2] and scale bytes [..., K / 32] -> the float32 values they stand for, [..., K]."""
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(*scales.shape, 32)
    s = scales.to(torch.int32)
    size = torch.where(s > 0, s << 23, 1 << 22).view(torch.float32)  # 2^(s - 127); 2^-127 has no exponent bits
    v = _table(packed.device)[code.int()] * size[..., None]
    return v.reshape(*packed.shape[:-1], -1)


def _padded(x, to):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % to))


# ---- inputs --------------------------------------------------------------------------------------------------------
def _normal(shape, seed, k, spread=0.0):
    """Normal values; with spread, columns of unequal size, as activations and keys have them."""
    g = torch.Generator("cuda").manual_seed(1000 * int(seed) + k)
    x = torch.randn(shape, generator=g, device="cuda")
    if spread:
        x *= torch.exp(spread * torch.randn(shape[-1:], generator=g, device="cuda"))
    return x


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, s = case, dict(case)
    kind, t = c["kind"], TYPES[c["type"]]
    if kind == "quantize":
        M, K = c["M"], c["K"]
        s["x"] = _normal((M, K), seed, 1, 0.7).to(t)
        Kp = -(-K // 128) * 128
        s["codes"] = torch.empty((M, Kp // 2), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((M, Kp // 32), dtype=torch.uint8, device="cuda")
        s["y"] = torch.empty((M, K), dtype=t, device="cuda")
        return s
    if kind == "product":
        for name, rows, k, size in (("A", c["M"], 1, 1.0), ("W", c["N"], 2, c["K"] ** -0.5)):
            code, s[name + "s"] = _codes(_padded(_normal((rows, c["K"]), seed, k, 0.3) * size, 128))
            s[name] = _pack(code)
        s["C"] = torch.empty((c["M"], c["N"]), dtype=t, device="cuda")
        return s
    n, T, H, dh, cap = c["n"], c["T"], c["H"], c["dh"], c["cap"]
    lens, counts = _lengths(c)
    s["pos"], s["counts"] = _ints(lens - counts), _ints(counts)
    held = _ints(np.minimum(lens if kind == "attention" else lens - counts, cap))
    there = (torch.arange(cap, device="cuda") < held[:, None])[:, None, :, None]
    for name, k in (("k", 1), ("v", 2)):
        s[name + "_codes"] = torch.zeros((n, H, cap, dh // 2), dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.zeros((n, H, cap, dh // 32), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (H * cap * dh))
        for i in range(0, n, step):
            shape = (min(step, n - i), H, cap, dh)
            code, scale = _codes(_normal(shape, seed, 10 * i + k, 0.5 if name == "k" else 0.0))
            s[name + "_codes"][i:i + step] = _pack(code) * there[i:i + step]
            s[name + "_scales"][i:i + step] = scale * there[i:i + step]
    if kind == "write":
        # keys and values as the projection leaves them: one row of both for each token
        s["kv"] = _normal((n, T, 2, H, dh), seed, 3, 0.5).to(t)
        s["k_out"], s["v_out"] = (torch.zeros((n, T, H, dh), dtype=t, device="cuda") for _ in range(2))
    else:
        s["q"] = _normal((n, T, H * c["G"], dh), seed, 3, 0.3).to(t)
        s["out"] = torch.zeros((n, T, H * c["G"], dh), dtype=t, device="cuda")
    return s


# ---- the operators in plain form -----------------------------------------------------------------------------------
def _slots(p, c):
    """The slot of position p."""
    return torch.where(p < c["sinks"], p, c["sinks"] + (p - c["sinks"]) % (c["cap"] - c["sinks"]))


def _quantize(s):
    code, scale = _codes(_padded(s["x"].float(), 128))
    s["codes"].copy_(_pack(code))
    s["scales"].copy_(scale)
    s["y"].copy_(_values(s["codes"], s["scales"])[:, :s["K"]])
    return s["y"]


def _product(s):
    s["C"].copy_(torch.matmul(_values(s["A"], s["As"]), _values(s["W"], s["Ws"]).t()))
    return s["C"]


def _store(codes, scales, out, seq, slot, tok, code, scale):
    codes[seq, :, slot] = code
    scales[seq, :, slot] = scale
    out[seq, tok] = _values(codes[seq, :, slot], scales[seq, :, slot]).to(out.dtype)


def _write(s):
    t = torch.arange(s["T"], device="cuda")
    p = s["pos"][:, None] + t
    end = (s["pos"] + s["counts"])[:, None]
    kept = (t < s["counts"][:, None]) & ((p < s["sinks"]) | (p >= end - (s["cap"] - s["sinks"])))
    seq, tok = kept.nonzero(as_tuple=True)
    slot = _slots(p[seq, tok], s)
    code, scale = _codes(s["kv"][seq, tok].float())
    code = _pack(code)
    _store(s["k_codes"], s["k_scales"], s["k_out"], seq, slot, tok, code[:, 0], scale[:, 0])
    _store(s["v_codes"], s["v_scales"], s["v_out"], seq, slot, tok, code[:, 1], scale[:, 1])
    return {"k": s["k_out"], "v": s["v_out"]}


def _attention(s):
    n, T, H, G, dh, cap, sinks = (s[k] for k in ("n", "T", "H", "G", "dh", "cap", "sinks"))
    k, v = _values(s["k_codes"], s["k_scales"]), _values(s["v_codes"], s["v_scales"])
    q = s["q"].float().view(n, T, H, G, dh).permute(0, 2, 3, 1, 4).reshape(n, H, G * T, dh)
    score = torch.matmul(q, k.transpose(-1, -2)).view(n, H, G, T, cap) * dh ** -0.5
    # which position each slot holds, and who sees it
    j, last = torch.arange(cap, device="cuda"), (s["pos"] + s["counts"] - 1)[:, None]
    held = torch.where(j < sinks, j, last - (last - j) % (cap - sinks))
    fine = (held <= last) & (held >= torch.where(j < sinks, 0, sinks))
    t = torch.arange(T, device="cuda")
    at = (s["pos"][:, None] + t)[:, :, None]
    sees = fine[:, None] & (held[:, None] <= at)
    if s["window"]:
        sees &= (held[:, None] > at - s["window"]) | (held[:, None] < sinks)
    sees = sees[:, None, None]
    score.masked_fill_(~sees, -math.inf)
    most = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(most > -math.inf, most, 0.0))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(n, H, G * T, cap), v).view(n, H, G, T, dh) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, T, H * G, dh).to(s["out"].dtype)
    rows = (t < s["counts"][:, None])[:, :, None, None]
    s["out"].copy_(torch.where(rows, o, s["out"]))
    return s["out"]


def _cache(s):
    """The cache object over the state's planes, which a program keeps."""
    if "cache" not in s:
        from mignon_ai_amd import KVCache
        s["cache"] = KVCache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], sinks=s["sinks"])
    return s["cache"]


def run(s):
    kind = s["kind"]
    if not own:
        return {"quantize": _quantize, "product": _product, "write": _write, "attention": _attention}[kind](s)
    from mignon_ai_amd import mx4_dequantize_device, mx4_gemm_device, mx4_quantize_device
    if kind == "quantize":
        mx4_quantize_device(s["x"], s["codes"], s["scales"])
        mx4_dequantize_device(s["codes"], s["scales"], s["y"])
        return s["y"]
    if kind == "product":
        mx4_gemm_device(s["A"], s["As"], s["W"], s["Ws"], s["C"])
        return s["C"]
    if kind == "write":
        kv = s["kv"]
        _cache(s).write(kv[:, :, 0], kv[:, :, 1], s["pos"], s["counts"])
        _cache(s).read(s["k_out"], s["v_out"], s["pos"], s["counts"])
        return {"k": s["k_out"], "v": s["v_out"]}
    return _cache(s).attention(s["q"], s["out"], s["pos"], s["counts"], window=s["window"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def _seen(c):
    """Pairs of a query row and a position it sees, and positions that some row sees, over all sequences."""
    lens, counts = _lengths(c)
    pairs = seen = 0
    ring = c["cap"] - c["sinks"]
    for n, k in zip(lens.tolist(), counts.tolist()):
        if not k:
            continue
        p = np.arange(n - k, n)
        low = np.maximum(n - ring, p - c["window"] + 1 if c["window"] else 0)
        low = np.minimum(np.maximum(low, c["sinks"]), p + 1)
        pairs += int((np.minimum(c["sinks"], p + 1) + np.where(p >= c["sinks"], p + 1 - low, 0)).sum())
        seen += int(min(c["sinks"], n) + max(0, n - max(int(low.min()), c["sinks"])))
    return pairs, seen


def work(case):
    c = case
    size = SIZES[c["type"]]
    if c["kind"] == "quantize":
        return {"bytes": c["M"] * c["K"] * (2 * size + 17 / 32), "flops": 0}
    if c["kind"] == "product":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": (M + N) * K * 17 / 32 + M * N * size, "flops": 2 * M * N * K}
    row = c["H"] * c["dh"]
    tokens = int(_lengths(c)[1].sum())
    if c["kind"] == "write":
        return {"bytes": tokens * row * 2 * (2 * size + 17 / 32), "flops": 0}
    pairs, seen = _seen(c)
    return {"bytes": seen * row * 2 * 17 / 32 + 2 * tokens * row * c["G"] * size, "flops": 4 * pairs * row * c["G"]}


# ---- 64-bit results ------------------------------------------------------------------------------------------------
def _nearest(x):
    """What the format makes of float64 rows [..., K]: the values, by the spacing of the 4-bit numbers around each."""
    K = x.shape[-1]
    b = _padded(x, 32)
    b = b.reshape(*b.shape[:-1], -1, 32)
    a = b.abs().amax(-1, keepdim=True)
    size = torch.exp2(torch.where(a > 0, torch.floor(torch.log2(a)) - 2, -127.0).clamp(min=-127.0))
    y = (b / size).abs()
    gap = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = torch.clamp(torch.round(y / gap) * gap, max=6.0) * torch.sign(b) * size
    return y.reshape(*x.shape[:-1], -1)[..., :K]


def _read64(packed, scales):
    """The float64 values of packed codes: sign, exponent and mantissa bits of each."""
    code = torch.stack((packed % 16, packed // 16), -1).reshape(*packed.shape[:-1], -1).double()
    sign = torch.where(code >= 8, -1.0, 1.0).double()
    m = code - torch.where(code >= 8, 8.0, 0.0)
    e = torch.floor(m / 2)
    v = torch.where(e == 0, m / 2, (1 + (m - 2 * e) / 2) * torch.exp2(e - 1))
    return sign * v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quantize":
        return torch.cat([_nearest(x.double()) for x in s["x"].split(max(1, (1 << 24) // s["K"]))])
    if kind == "product":
        w = _read64(s["W"], s["Ws"]).t().contiguous()
        return torch.cat([torch.matmul(_read64(a, e), w) for a, e in zip(s["A"].split(4096), s["As"].split(4096))])
    lens, counts = _lengths(s)
    sinks, ring, T = s["sinks"], s["cap"] - s["sinks"], s["T"]
    if kind == "write":
        out = [_nearest(s["kv"][:, :, i].double()) for i in range(2)]
        p = torch.tensor(lens - counts, device="cuda")[:, None] + torch.arange(T, device="cuda")
        n = torch.tensor(lens, device="cuda")[:, None]
        kept = (p < n) & ((p < sinks) | (p >= n - ring))
        return {name: o * kept[:, :, None, None] for name, o in zip(("k", "v"), out)}
    H, G, dh = s["H"], s["G"], s["dh"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for i, (n, c) in enumerate(zip(lens.tolist(), counts.tolist())):
        if not c:
            continue
        # the positions that some row sees, in their order
        first = max(sinks, n - ring, n - c - s["window"] + 1 if s["window"] else 0)
        where = np.concatenate([np.arange(min(sinks, n)), np.arange(first, max(first, n))])
        slot = torch.tensor(np.where(where < sinks, where, sinks + (where - sinks) % ring), device="cuda")
        k, v = (_read64(s[m + "_codes"][i, :, slot], s[m + "_scales"][i, :, slot]) for m in ("k", "v"))
        where = torch.tensor(where, device="cuda")
        for t in range(0, c, 256):
            q = s["q"][i, t:min(t + 256, c)].double()
            rows = q.shape[0]
            at = n - c + t + torch.arange(rows, device="cuda")[:, None]
            sees = where <= at
            if s["window"]:
                sees &= (where > at - s["window"]) | (where < sinks)
            q = q.view(rows, H, G, dh).permute(1, 2, 0, 3).reshape(H, G * rows, dh)
            x = torch.matmul(q, k.transpose(1, 2).contiguous()).view(H, G, rows, -1) / math.sqrt(dh)
            x = torch.softmax(x.masked_fill(~sees, -math.inf), -1).view(H, G * rows, -1)
            o = torch.matmul(x, v).view(H, G, rows, dh).permute(2, 0, 1, 3)
            out[i, t:t + rows] = o.reshape(rows, H * G, dh)
    return out
