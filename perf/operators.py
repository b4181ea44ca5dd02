"""The serving operators over packed rows and paged caches, as cases that can be timed.

Four operators: rotary positions of packed rows, the round trip of rows through
a paged cache (written, quantised where the cache has 8 bits, and read back),
attention of new tokens over a paged cache, and attention of packed prompts.
Shapes are Gemma-3-1B's (4 query heads over 1 KV head of 256, window 512), which
this repository's benchmark and tests use, and generic ones of 128 and 64 dims.

`own` false: the plain form, elementary torch operations in 32 bits (angles and
roundings to 8 bits in 64), rounded once at the end. `own` true: the calls a
program makes of the C ABI, with torch tensors as device memory.
"""
import math
import random

import torch

own = False

DEV = "cuda"
F32, F64 = torch.float32, torch.float64
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
      "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}


def listed():
    return [
        # a decode step of 16 sequences deep in their contexts: all latency
        {"name": "rope_16", "op": "rope", "tokens": 16, "heads": 4, "kv_heads": 1, "dim": 256, "rot": 256,
         "type": "f32", "layout": "half", "scaling": "none", "theta": 1e6, "reach": 4096},
        # a long prompt's chunk in a model of interleaved pairs over half of
        # the head, its context extended eightfold
        {"name": "rope_8192", "op": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "type": "bf16", "layout": "interleaved", "scaling": "bands", "theta": 5e5, "reach": 131072},
        # the new rows of a decode step of 16 sequences, through an 8-bit cache
        {"name": "kv_16", "op": "kv", "seqs": 16, "new": 1, "past": 4096, "kv_heads": 1, "dim": 256, "type": "f32",
         "cache": "i8", "page": 64, "ragged": True},
        # prompts of eight sequences at once, as they enter an 8-bit cache
        {"name": "kv_8192", "op": "kv", "seqs": 8, "new": 1024, "past": 1000, "kv_heads": 8, "dim": 128,
         "type": "bf16", "cache": "e4m3", "page": 16, "ragged": True},
        # the same for one long document in a cache of 16 bits
        {"name": "kv_32000", "op": "kv", "seqs": 1, "new": 32000, "past": 0, "kv_heads": 4, "dim": 64,
         "type": "f16", "cache": "f16", "page": 128, "ragged": False},
        # the benchmark's decode attention (one sequence at 4096), on pages
        {"name": "decode_1", "op": "paged", "seqs": 1, "new": 1, "past": 4095, "heads": 4, "kv_heads": 1, "dim": 256,
         "type": "f32", "cache": "f16", "page": 64, "window": 0, "ragged": False},
        # a server's decode step: many sequences of all lengths
        {"name": "decode_64", "op": "paged", "seqs": 64, "new": 1, "past": 8000, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "bf16", "cache": "bf16", "page": 16, "window": 0, "ragged": True},
        # long contexts in an 8-bit cache
        {"name": "decode_16_long", "op": "paged", "seqs": 16, "new": 1, "past": 32767, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "bf16", "cache": "i8", "page": 64, "window": 0, "ragged": False},
        # chunks of long prompts over what the cache holds of them
        {"name": "chunk_512", "op": "paged", "seqs": 4, "new": 512, "past": 15000, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "f16", "cache": "e4m3", "page": 64, "window": 0, "ragged": True},
        # a prompt in a sliding-window layer
        {"name": "prompt_2000", "op": "packed", "seqs": 1, "new": 2000, "heads": 4, "kv_heads": 1, "dim": 256,
         "type": "f16", "window": 512, "ragged": False},
        # prompts of different lengths in one call
        {"name": "prompts_16", "op": "packed", "seqs": 16, "new": 1000, "heads": 16, "kv_heads": 4, "dim": 64,
         "type": "f16", "window": 0, "ragged": True},
        # one long prompt
        {"name": "prompt_16384", "op": "packed", "seqs": 1, "new": 16384, "heads": 16, "kv_heads": 2, "dim": 128,
         "type": "bf16", "window": 0, "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_SHAPES = [(4, 1, 256), (32, 8, 128), (16, 2, 128), (16, 4, 64), (8, 8, 64), (10, 2, 96), (6, 2, 80), (12, 4, 192)]


def draw(rng):
    op = rng.choice(["rope", "kv", "paged", "paged", "paged", "packed", "packed"])
    heads, kv_heads, dim = rng.choice(_SHAPES)
    shape = {"heads": heads, "kv_heads": kv_heads, "dim": dim}
    if op == "rope":
        return {"op": op, "tokens": _log(rng, 1, 8192), **shape, "rot": rng.choice([dim, dim, dim // 2, dim - 16]),
                "type": rng.choice(["f32", "f16", "bf16"]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "bands", "parts"]), "theta": rng.choice([1e4, 5e5, 1e6]),
                "reach": _log(rng, 16, 1 << 20)}
    if op == "kv":
        seqs = _log(rng, 1, 64)
        return {"op": op, "seqs": seqs, "new": rng.choice([1, _log(rng, 2, 16384 // seqs)]),
                "past": rng.choice([0, _log(rng, 1, 4096)]), "kv_heads": kv_heads, "dim": dim,
                "type": rng.choice(["f32", "f16", "bf16"]), "cache": rng.choice(["f16", "bf16", "i8", "e4m3"]),
                "page": rng.choice([16, 32, 64, 128, 256]), "ragged": rng.random() < 0.7}
    window = rng.choice([0, 0, 0, _log(rng, 16, 2000)])
    ragged = rng.random() < 0.7
    if op == "paged":
        cache = rng.choice(["f16", "bf16", "i8", "e4m3"])
        kind = {"f16": ["f16", "f32"], "bf16": ["bf16"]}.get(cache, ["f16", "bf16", "f32"])
        new = rng.choice([1, 1, 1, _log(rng, 2, 512)])
        seqs = _log(rng, 1, 64 if new == 1 else 8)
        past = rng.choice([0, _log(rng, 16, (1 << 19) // seqs if new == 1 else 1 << 13)])
        return {"op": op, "seqs": seqs, "new": new, "past": min(past, 32768), **shape, "type": rng.choice(kind),
                "cache": cache, "page": rng.choice([16, 32, 64, 128, 256]), "window": window, "ragged": ragged}
    seqs = _log(rng, 1, 32)
    return {"op": op, "seqs": seqs, "new": _log(rng, 1, 8192 // seqs), **shape, "type": rng.choice(["f16", "bf16"]),
            "window": window, "ragged": ragged}


# ---- inputs ----------------------------------------------------------------

def _lengths(c):
    """(new, past) of each sequence: the case's own, or spread below them (the first keeps them)."""
    n, new, past = c["seqs"], c["new"], c.get("past", 0)
    if not c["ragged"]:
        return [new] * n, [past] * n
    r = random.Random("%d %d %d" % (n, new, past))
    return [new] + [r.randint(max(1, new // 8), new) for _ in range(n - 1)], \
           [past] + [r.randint(past // 8, past) for _ in range(n - 1)]


def _cum(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def _normal(g, *shape, std=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=F32) * std).to(dtype)


def _pool(g, c, pages):
    """A cache of so many pages, all of it rows of N(0, 1), in the cache's type, and its scales."""
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    if SIZE[c["cache"]] == 2:
        return _normal(g, *shape, dtype=DT[c["cache"]]), None
    code, scale = _quantise(_normal(g, *shape, dtype=torch.float16), c["cache"])
    return code, scale


def prepare(case, seed):
    c = dict(case)
    c.pop("name", None)
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    s = {"case": c}
    if c["op"] == "rope":
        t, d = c["tokens"], c["dim"]
        s["q"] = _normal(g, t, c["heads"], d, dtype=DT[c["type"]])
        s["k"] = _normal(g, t, c["kv_heads"], d, dtype=DT[c["type"]])
        s["positions"] = torch.randint(0, c["reach"], (t,), generator=g, device=DEV, dtype=torch.int32)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s
    new, past = _lengths(c)
    s["cu"], total = _cum(new), sum(new)
    s["most_new"] = max(new)
    if c["op"] in ("kv", "paged"):
        table = -(-max(n + p for n, p in zip(new, past)) // c["page"])
        pages = c["seqs"] * table + 3
        order = torch.randperm(pages, generator=g, device=DEV)
        s["pages"] = order[:c["seqs"] * table].reshape(c["seqs"], table).to(torch.int32).contiguous()
        s["kv_len"] = torch.tensor([n + p for n, p in zip(new, past)], dtype=torch.int32).to(DEV)
        s["k_cache"], s["k_scale"] = _pool(g, c, pages)
        s["v_cache"], s["v_scale"] = _pool(g, c, pages)
    if c["op"] in ("kv", "packed"):
        # K and V as one product leaves them: a row holds both
        kv = _normal(g, total, 2 * c["kv_heads"], c["dim"], dtype=DT[c["type"]])
        s["k"], s["v"] = kv[:, :c["kv_heads"]], kv[:, c["kv_heads"]:]
    if c["op"] == "kv":
        s["k_out"] = torch.empty(total, c["kv_heads"], c["dim"], device=DEV, dtype=DT[c["type"]])
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        s["q"] = _normal(g, total, c["heads"], c["dim"], std=1.5, dtype=DT[c["type"]])
        s["out"] = torch.empty_like(s["q"])
    return s


# ---- one pass ----------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"rope": _own_rope, "kv": _own_kv, "paged": _own_paged, "packed": _own_packed}[op](s)
    return {"rope": _plain_rope, "kv": _plain_kv, "paged": _plain_paged, "packed": _plain_packed}[op](s)


# the framework's calls: the descriptors, which a program keeps beside its
# tensors, are made in the first pass on a state

def _elem(X, t):
    return {torch.float32: X.XP_ELEM_F32, torch.float16: X.XP_ELEM_F16, torch.bfloat16: X.XP_ELEM_BF16,
            torch.int8: X.XP_ELEM_I8, torch.float8_e4m3fn: X.XP_ELEM_E4M3}[t.dtype]


def _rows(X, t):
    return X.XpRows(t.data_ptr(), t.stride(0), t.shape[1], _elem(X, t))


def _cache(X, s):
    k, v = s["k_cache"], s["v_cache"]
    pages, kv_heads, page, dim = k.shape
    scales = (s["k_scale"].data_ptr(), s["v_scale"].data_ptr()) if s["k_scale"] is not None else (None, None)
    return X.XpPagedKv(k.data_ptr(), v.data_ptr(), *scales, _elem(X, k), pages, page, kv_heads, dim)


def _seqs(X, s, tokens):
    return X.XpPagedSeqs(s["kv_len"].numel(), tokens, s["cu"].data_ptr(), s["kv_len"].data_ptr(),
                         s["pages"].data_ptr(), s["pages"].shape[1])


def _own_rope(s):
    import xpose_amd as X
    c = s["case"]
    if "args" not in s:
        kind = {"none": X.XP_ROPE_PLAIN, "linear": X.XP_ROPE_LINEAR, "bands": X.XP_ROPE_BANDS,
                "parts": X.XP_ROPE_PARTS}[c["scaling"]]
        low, high = _RAMP.get(c["scaling"], (0.0, 0.0))
        spec = X.XpRope(c["rot"], X.XP_ROPE_HALF if c["layout"] == "half" else X.XP_ROPE_INTERLEAVED, c["theta"],
                        kind, _FACTOR, _LENGTH, low, high, _magnitude(c))
        s["args"] = (_rows(X, s["q_out"]), _rows(X, s["q"]), _rows(X, s["k_out"]), _rows(X, s["k"]),
                     s["positions"].data_ptr(), c["tokens"], c["dim"], spec, None)
    X.call("xp_rope_rows", *s["args"])
    return s["q_out"], s["k_out"]


def _own_kv(s):
    import xpose_amd as X
    if "args" not in s:
        where = (_cache(X, s), _seqs(X, s, s["k"].shape[0]))
        s["args"] = (*where, _rows(X, s["k"]), _rows(X, s["v"]), None)
        s["back"] = (*where, _rows(X, s["k_out"]), _rows(X, s["v_out"]), None)
    X.call("xp_paged_kv_write", *s["args"])
    X.call("xp_paged_kv_read", *s["back"])
    return s["k_out"], s["v_out"]


def _workspace(X, s):
    c = s["case"]
    n = X.attention_workspace(s["q"].shape[0], c["seqs"], c["heads"], c["kv_heads"], c["dim"])
    s["workspace"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    return s["workspace"].data_ptr(), n


def _own_paged(s):
    import xpose_amd as X
    c = s["case"]
    if "args" not in s:
        s["args"] = (_rows(X, s["out"]), _rows(X, s["q"]), _cache(X, s), _seqs(X, s, s["q"].shape[0]), c["window"],
                     c["dim"] ** -0.5, *_workspace(X, s), None)
    X.call("xp_attention_paged", *s["args"])
    return s["out"]


def _own_packed(s):
    import xpose_amd as X
    c = s["case"]
    if "args" not in s:
        s["args"] = (_rows(X, s["out"]), _rows(X, s["q"]), _rows(X, s["k"]), _rows(X, s["v"]), c["dim"],
                     c["seqs"], s["q"].shape[0], s["cu"].data_ptr(), c["window"], c["dim"] ** -0.5,
                     *_workspace(X, s), None)
    X.call("xp_attention_packed", *s["args"])
    return s["out"]


# ---- the plain forms ----------------------------------------------------------

_FACTOR, _LENGTH = 8.0, 8192.0
_RAMP = {"bands": (1.0, 4.0), "parts": (1.0, 32.0)}


def _magnitude(c):
    return 1.0 + 0.1 * math.log(_FACTOR) if c["scaling"] == "parts" else 1.0


def _frequencies(c):
    """Radians a position of each pair, in 64 bits."""
    i = torch.arange(c["rot"] // 2, device=DEV, dtype=F64)
    f = c["theta"] ** (-2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        return f / _FACTOR
    if c["scaling"] == "bands":       # whole turns over the trained length: many keep their frequency
        low, high = _RAMP["bands"]
        keep = ((_LENGTH * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * keep + f / _FACTOR * (1 - keep)
    if c["scaling"] == "parts":       # the same by the pair's index
        low, high = _RAMP["parts"]
        at = [c["rot"] * math.log(_LENGTH / (2 * math.pi * r)) / (2 * math.log(c["theta"])) for r in (high, low)]
        first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), c["rot"] - 1)
        keep = 1 - ((i - first) / max(last - first, 1e-3)).clamp(0, 1)
        return f * keep + f / _FACTOR * (1 - keep)
    return f


def _plain_rope(s):
    c = s["case"]
    angle = s["positions"].to(F64)[:, None] * _frequencies(c)
    cos, sin = ((f(angle) * _magnitude(c)).to(F32)[:, None] for f in (torch.cos, torch.sin))
    n, inter = c["rot"], c["layout"] == "interleaved"
    out = []
    for x in (s["q"], s["k"]):
        x = x.to(F32)
        a, b = (x[..., 0:n:2], x[..., 1:n:2]) if inter else (x[..., :n // 2], x[..., n // 2:n])
        y = (a * cos - b * sin, b * cos + a * sin)
        y = torch.stack(y, -1).flatten(-2) if inter else torch.cat(y, -1)
        out.append(torch.cat((y, x[..., n:]), -1).to(s["q"].dtype))
    return tuple(out)


def _quantise(x, cache):
    """(codes, scale of each row) of rows of finite values, the rounding in 64 bits."""
    x = x.to(F64)
    top = x.abs().amax(-1)
    if cache == "i8":
        scale = (top / 127).to(F32)
        code = torch.round(x / scale.to(F64).clamp(min=2.0 ** -126)[..., None]).to(torch.int8)
        return code, scale
    # the least power of two that brings the row below the type's largest value
    m, e = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), e - 9 + (m > 0.875).to(e.dtype)).to(F32)
    return (x / scale.to(F64)[..., None]).to(F32).to(torch.float8_e4m3fn), scale


def _slots(s):
    """The page and the slot in it of each packed token."""
    cu, page = s["cu"].long(), s["case"]["page"]
    t = torch.arange(s["k"].shape[0], device=DEV)
    seq = torch.bucketize(t, cu[1:], right=True)
    at = s["kv_len"].long()[seq] - (cu[seq + 1] - t)
    return s["pages"].long()[seq, at // page], at % page


def _plain_kv(s):
    cache, page, slot = s["case"]["cache"], *_slots(s)
    out = []
    for new, pool, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        if scale is None:
            pool[page, :, slot] = new.to(F32).to(pool.dtype)
            out.append(pool[page, :, slot].to(F32).to(new.dtype))
            continue
        code, row = _quantise(new, cache)
        pool.view(torch.uint8)[page, :, slot] = code.view(torch.uint8)
        scale[page, :, slot] = row
        code = pool.view(torch.uint8)[page, :, slot].view(pool.dtype)
        out.append((code.to(F32) * scale[page, :, slot][..., None]).to(new.dtype))
    return tuple(out)


def _gathered(pool, scale, pages):
    """[seq][kv head][position][dim] in 32 bits of the pages of each sequence."""
    n, h, page, d = pool.shape
    x = (pool.view(torch.uint8)[pages].view(pool.dtype) if scale is not None else pool[pages]).to(F32)
    if scale is not None:
        x = x * scale[pages][..., None]
    return x.transpose(1, 2).reshape(pages.shape[0], h, -1, d)


def _softmax(scores, seen):
    """Over the last axis, of the seen scores alone; a row that sees none is zeros."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _plain_paged(s):
    c, q, cu = s["case"], s["q"], s["cu"].long()
    n, hk, group = c["seqs"], c["kv_heads"], c["heads"] // c["kv_heads"]
    i = torch.arange(s["most_new"], device=DEV)
    new = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)                    # [seq][new]: padded to the longest
    k = _gathered(s["k_cache"], s["k_scale"], s["pages"].long())
    v = _gathered(s["v_cache"], s["v_scale"], s["pages"].long())
    qs = q.to(F32)[at].reshape(n, -1, hk, group, c["dim"]).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, c["dim"])
    scores = torch.matmul(qs, k.transpose(-1, -2).contiguous()).reshape(n, hk, group, i.numel(), -1) * c["dim"] ** -0.5
    place = (s["kv_len"].long() - new)[:, None] + i                       # of a query in its sequence
    j = torch.arange(scores.shape[-1], device=DEV)
    seen = (j <= place[..., None]) & (j < s["kv_len"].long()[:, None, None])
    if c["window"]:
        seen &= j > place[..., None] - c["window"]
    p = _softmax(scores, seen[:, None, None])
    out = torch.matmul(p.reshape(n, hk, -1, p.shape[-1]), v)
    out = out.reshape(n, hk, group, i.numel(), -1).permute(0, 3, 1, 2, 4).reshape(n, i.numel(), c["heads"], -1)
    t = torch.arange(q.shape[0], device=DEV)
    seq = torch.bucketize(t, cu[1:], right=True)
    return out[seq, t - cu[seq]].to(q.dtype)


def _plain_packed(s):
    c, q = s["case"], s["q"]
    t, hk, group = q.shape[0], c["kv_heads"], c["heads"] // c["kv_heads"]
    k, v = (x.to(F32).permute(1, 0, 2) for x in (s["k"], s["v"]))
    qs = q.to(F32).reshape(t, hk, group, -1).permute(1, 2, 0, 3).reshape(hk, group * t, -1)
    scores = torch.matmul(qs, k.transpose(1, 2).contiguous()).reshape(hk, group, t, t) * c["dim"] ** -0.5
    j = torch.arange(t, device=DEV)
    seq = torch.bucketize(j, s["cu"].long()[1:], right=True)
    seen = (seq[:, None] == seq) & (j <= j[:, None])
    if c["window"]:
        seen &= j > j[:, None] - c["window"]
    out = torch.matmul(_softmax(scores, seen).reshape(hk, group * t, t), v.contiguous())
    return out.reshape(hk, group, t, -1).permute(2, 0, 1, 3).reshape(t, c["heads"], -1).to(q.dtype)


# ---- what a pass cannot do without ----------------------------------------------

def _pairs(new, past, window):
    """(pairs of a query and a key that it sees, keys that any query sees) of one sequence."""
    seen = sum(min(past + i + 1, window or past + i + 1) for i in range(new))
    return seen, min(past + new, window - 1 + new if window else past + new)


def work(case):
    c = case
    if c["op"] == "rope":
        n = c["tokens"] * (c["heads"] + c["kv_heads"])
        return {"bytes": 2 * n * c["dim"] * SIZE[c["type"]] + 4 * c["tokens"], "flops": 3 * n * c["rot"]}
    new, past = _lengths(c)
    rows = sum(new) * c["kv_heads"] * 2
    if c["op"] == "kv":
        held = c["dim"] * SIZE[c["cache"]] + (4 if SIZE[c["cache"]] == 1 else 0)
        return {"bytes": 2 * rows * (c["dim"] * SIZE[c["type"]] + held), "flops": 3 * rows * c["dim"]}
    both = [_pairs(n, p, c["window"]) for n, p in zip(new, past)]
    flops = 4 * c["dim"] * c["heads"] * sum(b[0] for b in both)
    io = 2 * sum(new) * c["heads"] * c["dim"] * SIZE[c["type"]]
    kind = c.get("cache", c["type"])
    row = c["dim"] * SIZE[kind] + (4 if SIZE[kind] == 1 else 0)
    return {"bytes": io + 2 * sum(b[1] for b in both) * c["kv_heads"] * row, "flops": flops}


# ---- in 64 bits, from the definitions ---------------------------------------------

def _exact_rope(c, s):
    n = c["rot"]
    turns = []
    for i in range(n // 2):
        f = math.exp(-2.0 * i / n * math.log(c["theta"]))
        g = 1.0                                                # the share that keeps its frequency
        if c["scaling"] == "linear":
            g = 0.0
        elif c["scaling"] == "bands":
            low, high = _RAMP["bands"]
            g = min(max((_LENGTH * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
        elif c["scaling"] == "parts":
            low, high = _RAMP["parts"]
            index = [n / 2 * math.log(_LENGTH / (2 * math.pi * r)) / math.log(c["theta"]) for r in (high, low)]
            a, b = max(math.floor(index[0]), 0), min(math.ceil(index[1]), n - 1)
            g = 1.0 - min(max((i - a) / max(b - a, 1e-3), 0.0), 1.0)
        turns.append(f * (g + (1 - g) / _FACTOR))
    z = torch.polar(torch.full((len(turns),), _magnitude(c), dtype=F64, device=DEV).expand(c["tokens"], -1).contiguous(),
                    s["positions"].to(F64)[:, None] * torch.tensor(turns, dtype=F64, device=DEV))[:, None]
    out = []
    for x in (s["q"], s["k"]):
        y = x.to(F64).clone()
        if c["layout"] == "half":
            w = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * z
            y[..., :n // 2], y[..., n // 2:n] = w.real, w.imag
        else:
            w = torch.view_as_complex(y[..., :n].reshape(*y.shape[:2], n // 2, 2).contiguous()) * z
            y[..., :n] = torch.view_as_real(w).flatten(-2)
        out.append(y)
    return tuple(out)


def _exact_rows(x, cache):
    """The values that rows have after their stay in the cache."""
    x = x.to(F64)
    if cache == "f16":
        return x.to(torch.float16).to(F64)
    if cache == "bf16":
        return x.to(torch.bfloat16).to(F64)
    top = x.abs().max(-1, keepdim=True).values
    if cache == "i8":
        step = (top / 127).to(F32).to(F64)
        return torch.where(top > 0, torch.round(x / step) * step, torch.zeros_like(x))
    unit = (2.0 ** torch.ceil(torch.log2(top / 448) - 1e-12)).to(F32).to(F64)
    y = x / unit
    step = (2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)).to(F32).to(F64)
    return torch.round(y / step) * step * unit


def _exact_attention(c, q, k, v, first):
    """One sequence: q [new][heads][dim], k and v [position][kv head][dim], the queries' places from `first` on."""
    out = torch.empty(q.shape, dtype=F64, device=DEV)
    group = c["heads"] // c["kv_heads"]
    for h in range(c["heads"]):
        kh, vh = k[:, h // group].to(F64), v[:, h // group].to(F64)
        for a in range(0, q.shape[0], 2048):
            place = first + a + torch.arange(min(2048, q.shape[0] - a), device=DEV)[:, None]
            j = torch.arange(kh.shape[0], device=DEV)[None]
            hidden = (j > place) | (j <= place - c["window"]) if c["window"] else j > place
            w = (q[a:a + 2048, h].to(F64) @ kh.T) / math.sqrt(c["dim"])
            out[a:a + 2048, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ vh
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "rope":
        return _exact_rope(c, s)
    if c["op"] == "kv":
        return _exact_rows(s["k"], c["cache"]), _exact_rows(s["v"], c["cache"])
    new, past = _lengths(c)
    out, a = [], 0
    for b, (n, p) in enumerate(zip(new, past)):
        if c["op"] == "packed":
            k, v = s["k"][a:a + n], s["v"][a:a + n]
        else:
            at = s["pages"][b, :-(-(n + p) // c["page"])].long()
            k, v = ((x.view(torch.uint8)[at].view(x.dtype) if x.element_size() == 1 else x[at]).to(F64) * (1.0 if e is None else e[at][..., None].to(F64))
                    for x, e in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
            k, v = (x.transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])[:n + p] for x in (k, v))
        out.append(_exact_attention(c, s["q"][a:a + n], k, v, p))
        a += n
    return torch.cat(out)
