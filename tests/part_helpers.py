"""64-bit oracle and caches for the operators over part of a cache."""
from __future__ import annotations

import math

import numpy as np
import torch


def paged(gpu, rng, hk, d, lengths, page=64, mode=None, spare=3, width=None):
    """A paged cache whose sequence b holds lengths[b] random rows on shuffled pages; table
    entries behind a sequence are -1."""
    import miinfer_amd as m
    from miinfer_amd import _lib
    rows = [-(-n // page) for n in lengths]
    perm = rng.permutation(sum(rows) + spare).astype(np.int32)
    table = np.full((len(lengths), width or max(max(rows), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(rows):
        table[b, :n] = perm[at:at + n]
        at += n
    cache = m.KvCache.paged_cache(hk, d, sum(rows) + spare, torch.from_numpy(table).to(gpu), page_tokens=page,
                                  quant_mode=_lib.KV_Q8_Q8 if mode is None else mode)
    fill(cache, gpu, rng, lengths)
    return cache


def fill(cache, gpu, rng, lengths):
    for b, n in enumerate(lengths):
        if n:
            k, v = (torch.from_numpy(rng.standard_normal((n, cache.kv_heads, cache.head_dim)).astype(np.float16)).to(gpu)
                    for _ in range(2))
            cache.append(k, v, seq=b)


def held(cache, seq, n):
    """(k, v) rows [heads, n, d] as the cache holds them, in 64 bits."""
    if n == 0:
        e = np.zeros((cache.kv_heads, 0, cache.head_dim))
        return e, e
    k, v = cache.export_dequant(seq, 0, n)
    return k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64)


def attend(q, k, v, length, scale, window=0, sinks=0):
    """q [t, heads, d], the last t tokens of a context of `length` keys k, v [kv heads,
    length, d]: (out [t, heads, d], weights [kv heads, length])."""
    t, hq, d = q.shape
    hk = k.shape[0]
    out = np.zeros((t, hq, d))
    got = np.zeros((hk, length))
    j = np.arange(length)
    for i in range(t):
        p = length - t + i
        seen = (j <= p) & ((window == 0) | (j > p - window) | (j < sinks))
        if p < 0 or not seen.any():
            continue
        for h in range(hq):
            g = h // (hq // hk)
            s = k[g][seen] @ q[i, h].astype(np.float64) * scale
            e = np.exp(s - s.max())
            e /= e.sum()
            out[i, h] = e @ v[g][seen]
            got[g][seen] += e
    return out, got


def logit_error(q, k, scale):
    """A bound on the error of a logit (natural units) computed with fp32 sums of exact
    products: the query in two fp16 parts is off by 2^-23 of its size and every one of
    at most d + d / 32 + 4 additions by 2^-24 of the largest partial sum, which |q| . |k|
    bounds; the MFMA's own order of additions is among them."""
    d = q.shape[-1]
    size = float(np.abs(q).max(axis=(0, 1)) @ np.abs(k).max(axis=(0, 1))) if k.size else 0.0
    # the bound over all keys is far above what happens: errors of d additions add up like
    # their square root, and the sum of absolute products like d * mean instead of maximum
    return scale * size * (math.sqrt(d) + 4) * 2.0 ** -24


def close_f32(got, want, q, k, v, scale, what=""):
    """Outputs of fp32 attention.  A probability is off by the logit's error (relative, twice:
    itself and the sum) and 2^-22 for exp2 and the two fp16 parts that it enters as; an
    output by that times the largest value."""
    got = np.asarray(got, np.float64)
    assert np.all(np.isfinite(got)), f"{what}: non-finite output"
    top = float(np.abs(v).max()) if v.size else 1.0
    tol = top * (2 * logit_error(q, k, scale) + 8 * 2.0 ** -22)
    err = float(np.abs(got - want).max()) if got.size else 0.0
    assert err <= tol, f"{what}: {err:.3e} > {tol:.3e}"


def close_weights(got, want, q, k, scale, terms, what=""):
    """Sums of `terms` probabilities of at most 1."""
    got = np.asarray(got, np.float64)
    tol = terms * (2 * logit_error(q, k, scale) + 8 * 2.0 ** -22)
    rel = np.abs(got - want) <= tol * np.maximum(np.abs(want), 2.0 ** -20)
    assert rel.all(), f"{what}: {np.abs(got - want).max():.3e}, tol {tol:.3e}"
