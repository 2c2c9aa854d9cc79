"""Measured workloads of the operators over part of a cache.

Four operators on a quantized KV cache: attention of ragged chunks of new tokens over a
paged cache (whole, or a sliding window and the first tokens), decode attention with a
sliding window and the first tokens, decode attention that adds up the weight every key
gets, and eviction of the keys with the least weight.  ``run`` is one call; with ``own``
false it computes the same in elementary torch operations in 32 bits, from the same
planes.  ``exact`` starts from the rows that the planes hold, in 64 bits, sequence by
sequence.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32  # values per q8_0 block
PAGE = 256  # tokens per page


# ---- the cases --------------------------------------------------------------------

def listed():
    gqa128 = {"q_heads": 32, "kv_heads": 8, "head_dim": 128}
    gqa256 = {"q_heads": 24, "kv_heads": 4, "head_dim": 256}
    return [
        # a serving step that mixes single tokens, drafted tokens and short turns
        {"name": "chunk_mixed_12", "kind": "chunk", **gqa256, "mode": "q8", "batch": 12, "new_low": 1, "new_high": 40,
         "low": 300, "high": 6000, "window": 0, "sinks": 0},
        # prompts' chunks in a layer with a sliding window and a few first tokens
        {"name": "chunk_window_4", "kind": "chunk", **gqa128, "mode": "q8", "batch": 4, "new_low": 300, "new_high": 1100,
         "low": 1500, "high": 8200, "window": 1024, "sinks": 4},
        # two sessions' 512-token chunks over 8k of context
        {"name": "chunk_512_8k", "kind": "chunk", **gqa256, "mode": "q8", "batch": 2, "new_low": 512, "new_high": 512,
         "low": 8704, "high": 8704, "window": 0, "sinks": 0},
        # whole prompts of several sessions at once, into an empty cache
        {"name": "chunk_prompts_3", "kind": "chunk", **gqa128, "mode": "q8", "batch": 3, "new_low": 700, "new_high": 3900,
         "low": 0, "high": 0, "window": 0, "sinks": 0},
        # one session's step in a windowed layer: launches and latency
        {"name": "window_one", "kind": "window", **gqa128, "mode": "q8", "q": "f16", "batch": 1, "tokens": 1,
         "low": 20001, "high": 20001, "window": 1024, "sinks": 4, "gate": False},
        # a serving batch in a windowed layer, contexts shorter and longer than the window
        {"name": "window_batch_24", "kind": "window", **gqa256, "mode": "q8", "q": "f16", "batch": 24, "tokens": 1,
         "low": 300, "high": 32768, "window": 4096, "sinks": 32, "gate": False},
        # verification of three drafted tokens, the fp16 cache, fp32 query, gated output
        {"name": "window_verify_8", "kind": "window", **gqa128, "mode": "f16", "q": "f32", "batch": 8, "tokens": 4,
         "low": 1900, "high": 12000, "window": 2048, "sinks": 16, "gate": True},
        # a long session's step that keeps the keys' weights
        {"name": "scored_one_32k", "kind": "scored", **gqa128, "mode": "q8", "q": "f16", "batch": 1, "tokens": 1,
         "low": 32768, "high": 32768, "gate": False},
        # a serving batch of chats that keeps them
        {"name": "scored_batch_20", "kind": "scored", **gqa256, "mode": "q8", "q": "f16", "batch": 20, "tokens": 1,
         "low": 200, "high": 6000, "gate": False},
        # the last tokens of prompts, whose weights the first eviction goes by
        {"name": "scored_last_4", "kind": "scored", **gqa128, "mode": "q8", "q": "f32", "batch": 4, "tokens": 4,
         "low": 1000, "high": 9001, "gate": True},
        # a long prompt cut down to its budget
        {"name": "evict_one_16k", "kind": "evict", **gqa128, "mode": "q8", "batch": 1, "low": 16384, "high": 16384,
         "budget": 4096, "sinks": 4, "recent": 256},
        # a batch of sessions cut down, some of them still below the budget
        {"name": "evict_batch_12", "kind": "evict", **gqa256, "mode": "q8", "batch": 12, "low": 1500, "high": 9000,
         "budget": 2048, "sinks": 16, "recent": 500},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hk, d = rng.choice([(32, 8, 128), (24, 4, 256)])
    kind = rng.choice(["chunk", "chunk", "window", "scored", "evict"])
    c = {"kind": kind, "q_heads": hq, "kv_heads": hk, "head_dim": d, "mode": rng.choice(["q8", "q8", "q8", "f16"])}
    if kind == "chunk":
        window = rng.choice([0, 0, _log(rng, 100, 4096)])
        high = _log(rng, 64, 8704)
        # no more (row, key) pairs than the two 512-token chunks over 8k have
        new = _log(rng, 1, min(high, 1100))
        batch = rng.randint(1, max(1, min(24, int(8.0e6 / (new * high)))))
        return {**c, "batch": batch, "new_low": max(1, new // rng.choice([1, 4, 16])), "new_high": new,
                "low": max(new, high // rng.choice([1, 2, 8])), "high": high, "window": window,
                "sinks": rng.choice([0, 4, rng.randint(1, 70)]) if window else 0}
    if kind == "evict":
        high = _log(rng, 200, 12000)
        budget = max(65, int(high * rng.uniform(0.1, 0.9)))
        recent = rng.randint(0, budget // 2)
        return {**c, "batch": rng.randint(1, min(32, max(1, 50000 // high))), "low": max(1, high // rng.choice([1, 2, 8])),
                "high": high, "budget": budget, "sinks": min(rng.choice([0, 4, rng.randint(1, 64)]), budget - recent),
                "recent": recent}
    tokens = rng.choice([1, 1, rng.randint(1, 16 // (hq // hk))])
    high = _log(rng, 64, 32768)
    window = _log(rng, 64, 4096)
    seen = min(high, window) if kind == "window" else high
    c.update({"q": rng.choice(["f16", "f32"]), "tokens": tokens, "low": max(tokens, high // rng.choice([1, 2, 8, 64])),
              "high": high, "gate": rng.random() < 0.4})
    if kind == "window":
        return {**c, "batch": rng.randint(1, max(1, min(32, 60000 // seen, 400000 // high))), "window": window,
                "sinks": rng.choice([0, 4, rng.randint(1, 200)])}
    return {**c, "batch": rng.randint(1, max(1, min(32, 32768 // seen)))}


# ---- inputs -----------------------------------------------------------------------

def _spread(n, lo, hi, step=0.6180339887):
    """n whole numbers, evenly over [lo, hi], in a mixed order."""
    return [lo + int((hi - lo + 1) * ((0.5 + i * step) % 1.0)) if hi > lo else lo for i in range(n)]


def _new(case):
    """New tokens of each sequence of a chunk case."""
    return _spread(case["batch"], case["new_low"], case["new_high"])


def _lengths(case):
    """Context lengths, the new tokens among them."""
    if case["kind"] != "chunk":
        return _spread(case["batch"], case["low"], case["high"], 0.7548776662)
    if case["high"] == 0:  # whole prompts
        return _new(case)
    return [max(n, L) for n, L in zip(_new(case), _spread(case["batch"], case["low"], case["high"], 0.7548776662))]


def _up(n, unit):
    return -(-n // unit) * unit


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 6151 + 29)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _inputs(case, seed):
    """Every random tensor of a case, from the seed alone: the rows of the pool's pages
    [pages, kv_heads, PAGE, head_dim], queries, gates and the weights so far."""
    g = _gen(seed)
    hq, hk, d, b = case["q_heads"], case["kv_heads"], case["head_dim"], case["batch"]
    lens = _lengths(case)
    rows = [_up(L, PAGE) // PAGE for L in lens]
    pages = sum(rows)
    width = max(rows)
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    start = torch.tensor([sum(rows[:i]) for i in range(b)], device=DEV)[:, None]
    slot = torch.arange(width, device=DEV)[None, :]
    here = slot < torch.tensor(rows, device=DEV)[:, None]
    x = {"table": torch.where(here, perm[torch.where(here, start + slot, 0)], -1).to(torch.int32).contiguous()}
    x["k"] = _randn(g, pages, hk, PAGE, d).to(torch.float16)
    x["v"] = _randn(g, pages, hk, PAGE, d).to(torch.float16)
    if case["kind"] == "evict":
        # sums of attention weights: a few keys have most of it, some have none
        u = torch.rand((b, hk, width * PAGE), generator=g, device=DEV)
        x["weights"] = torch.where(u < 0.05, 0.0, (-torch.log(u + 1e-7)) ** 3)
        return x
    # queries whose logits are a little sharper than of unit normal rows
    if case["kind"] == "chunk":
        x["q"] = (1.3 * _randn(g, sum(_new(case)), hq, d)).to(torch.bfloat16)
        return x
    q = 1.3 * _randn(g, b, case["tokens"], hq, d)
    x["q"] = q.to(torch.float16) if case["q"] == "f16" else q
    if case["gate"]:
        x["gate"] = _randn(g, b, case["tokens"], hq, d)
    if case["kind"] == "scored":
        x["weights"] = torch.rand((b, hk, width * PAGE), generator=g, device=DEV) ** 4
    return x


def _quantize(x):
    """(codes int8, scales fp16) of rows by the cache's rule: one scale per 32 values."""
    b = x.float().unflatten(-1, (x.shape[-1] // BLOCK, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / 127.0, torch.ones_like(top))
    code = torch.clamp(torch.round(b * (1.0 / scale)), -128, 127).to(torch.int8)
    return code.flatten(-2), scale.squeeze(-1).to(torch.float16)


def _tile_k(x):
    """Rows [pages, heads, PAGE, D] in the order of a K plane (16-token tiles, 8-dim runs)."""
    p, h, t, d = x.shape
    return x.view(p, h, t // 16, 16, d // 64, 2, 4, 8).permute(0, 1, 2, 4, 6, 3, 5, 7).contiguous().view(-1)


def _tile_v(x):
    """Rows [pages, heads, PAGE, D] in the order of a V plane (32 tokens of a dim together)."""
    p, h, t, d = x.shape
    return x.view(p, h, t // 32, 2, 4, 4, d).permute(0, 1, 2, 6, 4, 3, 5).contiguous().view(-1)


def _planes(x, mode):
    """The four planes of a cache that holds the rows."""
    if mode == "f16":
        return {"k_codes": _tile_k(x["k"]), "k_scales": None, "v_codes": _tile_v(x["v"]), "v_scales": None}
    (kc, ks), (vc, vs) = _quantize(x["k"]), _quantize(x["v"])
    return {"k_codes": _tile_k(kc), "k_scales": ks.view(torch.int16).reshape(-1),
            "v_codes": _tile_v(vc), "v_scales": vs.view(torch.int16).reshape(-1)}


def prepare(case, seed):
    x = _inputs(case, seed)
    hq, hk, d, b = case["q_heads"], case["kv_heads"], case["head_dim"], case["batch"]
    lens = _lengths(case)
    s = {"case": case, "lengths": torch.tensor(lens, dtype=torch.int32, device=DEV), "table": x["table"],
         "max_context": max(lens), "pages": x["k"].shape[0]}
    s["planes"] = _planes(x, case["mode"])
    for name in ("q", "gate", "weights"):
        if name in x:
            s[name] = x[name]
    if case["kind"] == "chunk":
        new = _new(case)
        s["offsets"] = torch.tensor([sum(new[:i]) for i in range(b + 1)], dtype=torch.int32, device=DEV)
        s["max_tokens"] = max(new)
        s["out"] = torch.empty_like(s["q"])
    elif case["kind"] == "evict":
        # the kept keys go to pages of their own: the old ones are shared with other sessions
        n = _up(case["budget"], PAGE) // PAGE
        for name, t in list(s["planes"].items()):
            if t is not None:
                s["planes"][name] = torch.cat([t, torch.zeros(b * n * (t.numel() // s["pages"]), dtype=t.dtype, device=DEV)])
        s["dst"] = (s["pages"] + torch.arange(b * n, dtype=torch.int32, device=DEV)).view(b, n).to(torch.int32)
        s["pages"] += b * n
        s["kept"] = torch.empty((b, hk, case["budget"]), dtype=torch.int32, device=DEV)
        s["new_lengths"] = torch.empty((b,), dtype=torch.int32, device=DEV)
        s["weights_out"] = torch.zeros((b, hk, n * PAGE), dtype=torch.float32, device=DEV)
    else:
        s["out"] = torch.empty((b, case["tokens"], hq, d), dtype=torch.float32, device=DEV)
    return s


# ---- the plain form ---------------------------------------------------------------

def _plane_views(s):
    """The planes as they are tiled: K codes [page, head, T, c, g, m, e, j], V codes [page,
    head, H, d, G, J, I], scales [page, head, token, block] (None for fp16 planes)."""
    p, c = s["planes"], s["case"]
    n, h, d = s["pages"], c["kv_heads"], c["head_dim"]
    k = p["k_codes"].view(n, h, PAGE // 16, d // 64, 4, 16, 2, 8)
    v = p["v_codes"].view(n, h, PAGE // 32, d, 4, 2, 4)
    if c["mode"] == "f16":
        return k, None, v, None
    return k, p["k_scales"].view(torch.float16).view(n, h, PAGE, d // BLOCK), v, \
        p["v_scales"].view(torch.float16).view(n, h, PAGE, d // BLOCK)


def _rows(s, pos):
    """Keys and values at positions pos [batch, n] of every sequence, in 32 bits:
    [batch, heads, n, d].  Positions past a sequence's pages give some page's rows."""
    k, ks, v, vs = _plane_views(s)
    page = s["table"].gather(1, torch.clamp(pos // PAGE, max=s["table"].shape[1] - 1)).clamp(min=0).long()
    at = pos % PAGE
    keys = k[page, :, at // 16, :, :, at % 16].permute(0, 2, 1, 3, 5, 4, 6).flatten(3).float()
    vals = v[page, :, at // 32, :, at % 16 // 4, at % 32 // 16, at % 4].permute(0, 2, 1, 3).float()
    if ks is not None:
        keys = keys * ks[page, :, at].permute(0, 2, 1, 3).float().repeat_interleave(BLOCK, -1)
        vals = vals * vs[page, :, at].permute(0, 2, 1, 3).float().repeat_interleave(BLOCK, -1)
    return keys.contiguous(), vals.contiguous()


def _softmax(logits, seen):
    """Softmax over the last axis of what is seen; a row that sees nothing gets zeros."""
    logits = torch.where(seen, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(logits - torch.where(top > -math.inf, top, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _seen(key, at, length, window, sinks):
    """Whether a token at position `at` sees key `key` of a context of `length` keys."""
    past = (key <= at) & (key < length)
    return past & ((key > at - window) | (key < sinks)) if window else past


def _attend(s, q, at, pos, window, sinks, twice):
    """Plain attention of q [batch, heads, n, d] (positions at [batch, n]) over the keys
    at positions pos [batch, m] (`twice`: positions that stand there a second time)."""
    c = s["case"]
    g = c["q_heads"] // c["kv_heads"]
    keys, vals = _rows(s, pos)
    b, h, m, d = keys.shape
    n = q.shape[2]
    seen = _seen(pos[:, None, :], at[:, :, None], s["lengths"][:, None, None], window, sinks) & ~twice[:, None, :]
    q = q.float().reshape(b, h, g * n, d)
    logits = torch.matmul(q, keys.transpose(-1, -2).contiguous()).view(b, h, g, n, m) / math.sqrt(d)
    p = _softmax(logits, seen[:, None, None])
    return torch.matmul(p.view(b, h, g * n, m), vals).view(b, h * g, n, d), p


def _plain_chunk(s):
    c = s["case"]
    most, b = s["max_tokens"], c["batch"]
    new = s["offsets"][1:] - s["offsets"][:-1]
    t = torch.arange(most, device=DEV)[None, :]
    row = s["offsets"][:-1, None] + t  # padded: [batch, most]
    at = s["lengths"][:, None] - new[:, None] + t
    q = s["q"][torch.clamp(row, max=s["q"].shape[0] - 1)].permute(0, 2, 1, 3).contiguous()
    pos = torch.arange(s["max_context"], device=DEV)[None, :].expand(b, -1)
    out, _ = _attend(s, q, at, pos, c["window"], c["sinks"], torch.zeros_like(pos, dtype=torch.bool))
    live = t < new[:, None]
    s["out"][row[live].long()] = out.permute(0, 2, 1, 3)[live].to(torch.bfloat16)
    return s["out"]


def _decode_at(s):
    t = s["case"]["tokens"]
    return s["lengths"][:, None] - t + torch.arange(t, device=DEV)[None, :]


def _gated(s, out):
    out = out.permute(0, 2, 1, 3)
    s["out"].copy_(out * (1.0 / (1.0 + torch.exp(-s["gate"]))) if s["case"]["gate"] else out)
    return s["out"]


def _plain_window(s):
    c = s["case"]
    # the window of the last tokens, and the first tokens in front of it
    span = min(c["window"] + c["tokens"] - 1, s["max_context"])
    tail = s["lengths"][:, None] - span + torch.arange(span, device=DEV)[None, :]
    head = torch.arange(min(c["sinks"], s["max_context"]), device=DEV)[None, :].expand(c["batch"], -1)
    pos = torch.cat([head, torch.clamp(tail, min=0)], 1)
    twice = torch.cat([torch.zeros_like(head, dtype=torch.bool), (tail < 0) | (tail < c["sinks"])], 1)
    out, _ = _attend(s, s["q"].permute(0, 2, 1, 3), _decode_at(s), pos.long(), c["window"], c["sinks"], twice)
    return _gated(s, out)


def _plain_scored(s):
    pos = torch.arange(s["max_context"], device=DEV)[None, :].expand(s["case"]["batch"], -1)
    out, p = _attend(s, s["q"].permute(0, 2, 1, 3), _decode_at(s), pos, 0, 0, torch.zeros_like(pos, dtype=torch.bool))
    s["weights"][:, :, :s["max_context"]] += p.sum((2, 3))
    return _gated(s, out), s["weights"]


def _plain_evict(s):
    c = s["case"]
    n = c["budget"]
    length = s["lengths"][:, None, None].long()
    weights = s["weights"]
    j = torch.arange(weights.shape[-1], device=DEV)[None, None, :]
    rank = torch.where((j < c["sinks"]) | (j >= length - c["recent"]), math.inf, weights)
    rank = torch.where(j < length, rank, -math.inf)
    if rank.shape[-1] < n:
        rank = torch.cat([rank, torch.full((*rank.shape[:-1], n - rank.shape[-1]), -math.inf, device=DEV)], -1)
    best = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :n]  # of equal weights the first ones
    keep = torch.sort(best, dim=-1)[0]
    live = torch.arange(n, device=DEV)[None, None, :] < length
    s["kept"].copy_(torch.where(live, keep, -1))
    s["new_lengths"].copy_(torch.clamp(s["lengths"], max=n))
    b, h, i = torch.nonzero(live.expand_as(keep), as_tuple=True)
    src = keep[b, h, i]
    s["weights_out"][b, h, i] = weights[b, h, src]
    sp, dp = s["table"][b, src // PAGE].long(), s["dst"][b, i // PAGE].long()
    src, dst = src % PAGE, i % PAGE
    k, ks, v, vs = _plane_views(s)
    k[dp, h, dst // 16, :, :, dst % 16] = k[sp, h, src // 16, :, :, src % 16]
    v[dp, h, dst // 32, :, dst % 16 // 4, dst % 32 // 16, dst % 4] = \
        v[sp, h, src // 32, :, src % 16 // 4, src % 32 // 16, src % 4]
    if ks is not None:
        ks[dp, h, dst] = ks[sp, h, src]
        vs[dp, h, dst] = vs[sp, h, src]
    return _evicted(s)


def _evicted(s):
    return s["kept"], s["new_lengths"], s["weights_out"], [t for t in s["planes"].values() if t is not None]


# ---- run --------------------------------------------------------------------------

def _held(s):
    """The cache object and workspace that a program keeps."""
    import miinfer_amd as m
    if "cache" not in s:
        c = s["case"]
        p = s["planes"]
        s["cache"] = m.KvCache.from_planes(c["kv_heads"], c["head_dim"], p["k_codes"], p["v_codes"], p["k_scales"],
                                           p["v_scales"], page_tokens=PAGE, block_table=s["table"])
        if c["kind"] == "chunk":
            need = m.chunk_workspace_bytes(s["cache"], c["q_heads"], c["batch"], s["q"].shape[0], s["max_tokens"],
                                           s["max_context"], c["window"], c["sinks"])
        elif c["kind"] == "window":
            need = m.window_workspace_bytes(s["cache"], c["q_heads"], c["batch"], c["tokens"], s["max_context"],
                                            c["window"], c["sinks"])
        elif c["kind"] == "scored":
            need = m.scored_workspace_bytes(s["cache"], c["q_heads"], c["batch"], c["tokens"], s["max_context"])
        else:
            need = 0  # eviction needs none
        s["ws"] = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    return m, s["cache"], s["ws"]


def _own(s):
    c = s["case"]
    m, cache, ws = _held(s)
    if c["kind"] == "chunk":
        m.chunk_attention(cache, s["q"], s["offsets"], s["lengths"], max_tokens=s["max_tokens"],
                          max_context=s["max_context"], window=c["window"], sinks=c["sinks"], out=s["out"], workspace=ws)
        return s["out"]
    if c["kind"] == "evict":
        m.evict(cache, s["weights"], s["lengths"], budget=c["budget"], sinks=c["sinks"], recent=c["recent"],
                max_context=s["max_context"], dst_table=s["dst"], kept=s["kept"], new_lengths=s["new_lengths"],
                weights_out=s["weights_out"])
        return _evicted(s)
    outs = {"gate": s["gate"], "gated_out": s["out"]} if c["gate"] else {"out": s["out"]}
    if c["kind"] == "window":
        m.window_attention(cache, s["q"], lengths=s["lengths"], max_context=s["max_context"], window=c["window"],
                           sinks=c["sinks"], workspace=ws, **outs)
        return s["out"]
    m.scored_attention(cache, s["q"], s["weights"], lengths=s["lengths"], max_context=s["max_context"], workspace=ws, **outs)
    return s["out"], s["weights"]


def run(s):
    if own:
        return _own(s)
    return {"chunk": _plain_chunk, "window": _plain_window, "scored": _plain_scored, "evict": _plain_evict}[s["case"]["kind"]](s)


# ---- what a pass cannot do without --------------------------------------------------

def _row_bytes(case):
    """Bytes of one position of the cache, all kv heads, K and V."""
    d = case["head_dim"]
    return 2 * case["kv_heads"] * (2 * d if case["mode"] == "f16" else d + d // 16)


def _pairs(case, n, length):
    """(pairs of a token and a key it sees, keys that any of them sees) of n tokens that
    end a context of `length`."""
    w, s = case.get("window", 0), case.get("sinks", 0)
    base = length - n
    if not w:
        return n * base + n * (n + 1) // 2, length
    near = sum(min(w, base + t + 1) for t in range(n))
    # first tokens in front of the window of each
    far = sum(min(s, max(0, base + t + 1 - w)) for t in range(n))
    first = max(0, base + 1 - w)
    return near + far, length - first + min(s, first)


def work(case):
    hq, hk, d, b = case["q_heads"], case["kv_heads"], case["head_dim"], case["batch"]
    lens = _lengths(case)
    if case["kind"] == "evict":
        moved = sum(min(L, case["budget"]) for L in lens)
        # weights read, kept rows moved with their weights, the list of them written
        return {"bytes": 4 * hk * sum(lens) + 2 * moved * _row_bytes(case) + 8 * hk * moved, "flops": 0}
    new = _new(case) if case["kind"] == "chunk" else [case["tokens"]] * b
    pairs, keys = map(sum, zip(*(_pairs(case, n, L) for n, L in zip(new, lens))))
    if case["kind"] == "chunk":
        row = hq * d * 4
    else:
        row = hq * d * ((2 if case["q"] == "f16" else 4) + 4 + (4 if case["gate"] else 0))
    more = 8 * hk * keys if case["kind"] == "scored" else 0  # weights read and written
    return {"bytes": keys * _row_bytes(case) + sum(new) * row + more, "flops": 4 * hq * d * pairs}


# ---- the same in 64 bits ------------------------------------------------------------

def _held_rows(rows, mode):
    """Rows as the cache holds them, in 64 bits."""
    if mode == "f16":
        return rows.double()
    b = rows.float().reshape(*rows.shape[:-1], -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / 127.0, torch.ones_like(top))
    code = torch.round(b * (1.0 / scale)).clamp(-128, 127)
    return (code.double() * scale.to(torch.float16).double()).reshape(rows.shape)


def _sequence(case, x, b, length):
    """Keys and values of sequence b, [heads, length, d]."""
    pages = x["table"][b, :_up(length, PAGE) // PAGE].long()
    take = lambda t: _held_rows(t[pages].transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])[:, :length], case["mode"])  # noqa: E731
    return take(x["k"]), take(x["v"])


def _exact_attention(case, q, k, v):
    """q [n, heads, d], the last n tokens of k, v [kv heads, length, d]: out [n, heads, d]
    and each kv head's weights [kv heads, length]."""
    n, hq, d = q.shape
    hk, length, _ = k.shape
    key = torch.arange(length, device=DEV)[None, :]
    at = (length - n + torch.arange(n, device=DEV))[:, None]
    hidden = key > at
    if case.get("window", 0):
        hidden |= (at - key >= case["window"]) & (key >= case["sinks"])
    out = torch.empty((n, hq, d), dtype=torch.float64, device=DEV)
    got = torch.zeros((hk, length), dtype=torch.float64, device=DEV)
    for h in range(hq):
        a = q[:, h].double() @ k[h * hk // hq].T.contiguous() / math.sqrt(d)
        p = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
        out[:, h] = p @ v[h * hk // hq]
        got[h * hk // hq] += p.sum(0)
    return out, got


def exact(case, seed):
    if case["kind"] == "evict":
        return None  # rows are moved, nothing is computed
    x = _inputs(case, seed)
    lens = _lengths(case)
    new = _new(case) if case["kind"] == "chunk" else [case["tokens"]] * case["batch"]
    outs, weights, at = [], x["weights"].double() if case["kind"] == "scored" else None, 0
    for b, (n, length) in enumerate(zip(new, lens)):
        q = x["q"][at:at + n] if case["kind"] == "chunk" else x["q"][b]
        k, v = _sequence(case, x, b, length)
        out, got = _exact_attention(case, q, k, v)
        outs.append(out)
        if weights is not None:
            weights[b, :, :length] += got
        at += n
    if case["kind"] == "chunk":
        return torch.cat(outs)
    out = torch.stack(outs)
    if case["gate"]:
        out = out * torch.sigmoid(x["gate"].double())
    return out if weights is None else (out, weights)
