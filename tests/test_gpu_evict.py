"""Eviction against the same choice and moves on the host, byte for byte (GPU)."""
import math

import numpy as np
import pytest
import torch

from tests.part_helpers import attend, close_f32, fill, held, paged

pytestmark = pytest.mark.gpu

SHAPES = [(32, 8, 128), (24, 4, 256)]


def _dev(a, gpu):
    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


def _choose(w, n, budget, sinks, recent):
    """Positions that stay, ascending."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sinks, n - recent)
    rank = np.where(np.isnan(w[mid]), -np.inf, w[mid]).astype(np.float64)
    # a NaN is behind -inf too
    order = sorted(range(len(mid)), key=lambda i: (bool(np.isnan(w[mid[i]])), -rank[i], i))
    best = mid[sorted(order[:budget - sinks - recent])]
    return np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)])


def _rows(cache, seq, n):
    """Codes (and scales) of the first n rows, host, per plane."""
    return [None if t is None else t.cpu().numpy() for t in cache.export_canonical(seq, 0, n)]


def _weights(rng, shape):
    u = rng.random(shape)
    w = np.where(u < 0.2, 0.0, np.round(-np.log(u + 1e-6) * 4) / 4).astype(np.float32)  # many equal ones
    return w


def _check(cache, before, w, kept, lengths, new, budget, sinks, recent, out_w=None):
    kept = kept.cpu().numpy()
    for b, n in enumerate(lengths):
        left = min(n, budget)
        assert int(new[b]) == left
        if left == 0:
            assert (kept[b] == -1).all()
            continue
        after = _rows(cache, b, left)
        for h in range(cache.kv_heads):
            want = _choose(w[b, h], n, budget, sinks, recent)
            assert np.array_equal(kept[b, h, :left], want), (b, h)
            assert (kept[b, h, left:] == -1).all()
            for old, now in zip(before[b], after):
                if old is not None:
                    assert np.array_equal(old[h][want].view(np.uint8), now[h].view(np.uint8)), (b, h)
            if out_w is not None:
                assert np.array_equal(w[b, h][want].view(np.uint32), out_w[b, h, :left].cpu().numpy().view(np.uint32))


@pytest.mark.parametrize("hq,hk,d", SHAPES)
@pytest.mark.parametrize("mode", [3, 0, 1, 2])
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (33, 0, 0), (100, 4, 30), (256, 0, 256), (300, 7, 11),
                                                 (700, 64, 100)])
def test_evict(gpu, hq, hk, d, mode, inplace, budget, sinks, recent):
    import miinfer_amd as m
    rng = np.random.default_rng(budget + mode)
    lengths = [0, 1, 32, budget, budget + 1, 700, 1025]
    lengths = [min(n, 1088) for n in lengths]
    np_dst = -(-budget // 64)
    cache = paged(gpu, rng, hk, d, lengths, mode=mode, spare=len(lengths) * np_dst)
    before = [_rows(cache, b, n) if n else [None] * 4 for b, n in enumerate(lengths)]
    w = _weights(rng, (len(lengths), hk, 1100))
    lens = _dev(np.array(lengths, np.int32), gpu)
    dw = _dev(w, gpu)
    if inplace:
        kept, new = m.evict(cache, dw, lens, budget=budget, sinks=sinks, recent=recent, max_context=1088, new_lengths=lens,
                            weights_out=dw)
        assert new is lens
        _check(cache, before, w, kept, lengths, new, budget, sinks, recent, dw)
        for b, n in enumerate(lengths):  # what lay behind is no weight of the keys to come
            left = min(n, budget)
            assert not dw[b, :, left:n].any()
            assert np.array_equal(dw[b, :, n:].cpu().numpy(), w[b, :, n:])
        return
    used = set(cache.block_table.cpu().numpy().ravel().tolist())
    free = [p for p in range(cache.num_pages) if p not in used][:len(lengths) * np_dst]
    dst = _dev(np.array(free, np.int32).reshape(len(lengths), np_dst), gpu)
    out_w = torch.full((len(lengths), hk, max(budget, 1)), 7.0, device=gpu)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        if t is not None:  # every byte of the new pages known
            t.view(cache.num_pages, -1)[dst.flatten().long()] = 5
    kept, new = m.evict(cache, dw, lens, budget=budget, sinks=sinks, recent=recent, max_context=1088, dst_table=dst,
                        weights_out=out_w)
    old_table = cache.block_table
    for b, n in enumerate(lengths):  # the old pages are as they were
        if n:
            for x, y in zip(before[b], _rows(cache, b, n)):
                assert x is None or np.array_equal(x, y)
    assert np.array_equal(dw.cpu().numpy(), w)
    cache.set_block_table(dst)
    _check(cache, before, w, kept, lengths, new, budget, sinks, recent, out_w)
    for b, n in enumerate(lengths):  # rows and weights behind the kept ones are as they were
        left = min(n, budget)
        assert bool((out_w[b, :, left:] == 7).all())
        if left < np_dst * 64:
            for t in cache.export_canonical(b, left, np_dst * 64 - left):
                assert t is None or bool((t == 5).all()), b
    assert old_table is not cache.block_table


def test_evict_contiguous_and_repeated(gpu):
    """A contiguous cache cut down again and again, as a session that stays at its budget."""
    import miinfer_amd as m
    rng = np.random.default_rng(3)
    hk, d, cap = 8, 128, 4096
    cache = m.KvCache.contiguous(hk, d, cap)
    n = 4001
    fill(cache, gpu, rng, [n])
    w = _weights(rng, (1, hk, cap))
    w[:, :, n:] = 0
    dw = _dev(w, gpu)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    for budget in (3500, 1024, 1000, 999, 64):
        before = [_rows(cache, 0, n)]
        kept, _ = m.evict(cache, dw, lens, budget=budget, sinks=4, recent=50, new_lengths=lens, weights_out=dw)
        _check(cache, before, w, kept, [n], lens, budget, 4, 50, dw)
        w, n = dw.cpu().numpy(), budget
        assert not w[:, :, n:].any()


def test_evict_odd_weights(gpu):
    """NaN behind every number, infinities, both zeros equal, negative numbers, all equal."""
    import miinfer_amd as m
    rng = np.random.default_rng(4)
    hk, d, n = 4, 256, 500
    special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 2.5, 1e-42, -1e-42], np.float32)
    w = special[rng.integers(0, len(special), (2, hk, n))]
    w[1, 0] = 3.0
    w[1, 1] = np.nan
    w[1, 2] = -np.inf
    for budget in (40, 250, 300, 430):
        cache = paged(gpu, rng, hk, d, [n, n])
        before = [_rows(cache, b, n) for b in range(2)]
        kept, new = m.evict(cache, _dev(w, gpu), torch.tensor([n, n], dtype=torch.int32, device=gpu), budget=budget, sinks=2,
                            recent=5, max_context=n)
        _check(cache, before, w, kept, [n, n], new, budget, 2, 5)


def test_evict_long(gpu):
    """More keys than a select workgroup holds at once, nearly all equal weights among them."""
    import miinfer_amd as m
    rng = np.random.default_rng(5)
    hk, d, n = 2, 128, 70001
    cache = m.KvCache.contiguous(hk, d, 70016)
    fill(cache, gpu, rng, [n])
    w = np.zeros((1, hk, n), np.float32)
    w[0, 0, rng.integers(0, n, 900)] = 1.0
    w[0, 1] = rng.random(n)
    before = [_rows(cache, 0, n)]
    kept, new = m.evict(cache, _dev(w, gpu), torch.tensor([n], dtype=torch.int32, device=gpu), budget=30000, sinks=4, recent=1000,
                        max_context=n)
    _check(cache, before, w, kept, [n], new, 30000, 4, 1000)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("budget", [1024, 1025, 3070])
def test_evict_in_place_over_several_turns(gpu, d, mode, budget):
    """More rows than move at a time, in place, where kept keys stand close and far apart: every plane, sequences of
    which one stays as it is."""
    import miinfer_amd as m
    rng = np.random.default_rng(d + mode + budget)
    lengths = [5001, 900, budget + 1]
    cache = paged(gpu, rng, 2, d, lengths, mode=mode, page=128)
    w = rng.random((3, 2, 5100)).astype(np.float32)
    w[0, 0, :2500] += 1.0  # the front stays whole, then the rest moves far
    w[0, 1, 2500:] += 1.0
    before = [_rows(cache, b, n) for b, n in enumerate(lengths)]
    kept, new = m.evict(cache, _dev(w, gpu), _dev(np.array(lengths, np.int32), gpu), budget=budget, sinks=3, recent=20,
                        max_context=5100)
    _check(cache, before, w, kept, lengths, new, budget, 3, 20)


@pytest.mark.parametrize("n,budget,sinks,recent", [(16390, 9000, 4, 2), (16391, 9000, 4, 2), (40001, 21000, 0, 5000),
                                                   (40001, 39990, 7, 30000), (50000, 50, 25, 25), (33000, 32999, 0, 0)])
@pytest.mark.parametrize("own_rows", [True, False])
def test_evict_long_weights(gpu, n, budget, sinks, recent, own_rows):
    """Long contexts whose weights move too, over themselves or to rows of another stride; ties among them."""
    import miinfer_amd as m
    rng = np.random.default_rng(n + budget)
    hk, d, cap = 2, 128, 50048
    cache = m.KvCache.contiguous(hk, d, cap)
    fill(cache, gpu, rng, [n])
    w = np.zeros((1, hk, cap), np.float32)
    w[0, 0, :n] = rng.integers(0, 9, n)
    w[0, 1, :n] = rng.random(n)
    before = [_rows(cache, 0, n)]
    dw = _dev(w, gpu)
    out = dw if own_rows else torch.full((1, hk, budget + 3), 5.0, device=gpu)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    kept, new = m.evict(cache, dw, lens, budget=budget, sinks=sinks, recent=recent, weights_out=out)
    _check(cache, before, w, kept, [n], new, budget, sinks, recent)
    k = kept.cpu().numpy()
    for h in range(hk):
        got = out[0, h].cpu().numpy()
        assert np.array_equal(got[:budget], w[0, h, k[0, h]])
        assert np.all(got[budget:] == (0.0 if own_rows else 5.0))


def test_evict_graph(gpu):
    """A captured eviction to other pages, replayed with other weights and lengths."""
    import miinfer_amd as m
    rng = np.random.default_rng(6)
    hk, d, lengths, budget = 8, 128, [600, 333], 200
    cache = paged(gpu, rng, hk, d, lengths, spare=8)
    used = set(cache.block_table.cpu().numpy().ravel().tolist())
    dst = _dev(np.array([p for p in range(cache.num_pages) if p not in used][:8], np.int32).reshape(2, 4), gpu)
    dw = _dev(_weights(rng, (2, hk, 640)), gpu)
    lens = _dev(np.array(lengths, np.int32), gpu)
    kept = torch.empty((2, hk, budget), dtype=torch.int32, device=gpu)
    new = torch.empty(2, dtype=torch.int32, device=gpu)
    out_w = torch.zeros((2, hk, 256), device=gpu)
    args = dict(budget=budget, sinks=3, recent=20, max_context=640, dst_table=dst, kept=kept, new_lengths=new, weights_out=out_w)
    m.evict(cache, dw, lens, **args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.evict(cache, dw, lens, **args)
    table = cache.block_table
    before = [_rows(cache, b, n) for b, n in enumerate(lengths)]
    for turn in range(3):
        w = _weights(rng, (2, hk, 640))
        dw.copy_(_dev(w, gpu))
        now = [lengths[0] - 190 * turn, lengths[1] - 100 * turn]
        lens.copy_(_dev(np.array(now, np.int32), gpu))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        cache.set_block_table(dst)
        _check(cache, [[None if t is None else t[:, :x] for t in bf] for bf, x in zip(before, now)], w, kept, now, new, budget, 3,
               20, out_w)
        cache.set_block_table(table)


def test_pool_truncate_after_evict(gpu):
    """Pages that an eviction in place empties go back to the pool."""
    import miinfer_amd as m
    from miinfer_amd import reuse
    rng = np.random.default_rng(7)
    pool = reuse.PagePool(12)
    row = np.array([pool.alloc() for _ in range(10)], np.int32)
    cache = m.KvCache.paged_cache(8, 128, 12, _dev(row[None], gpu), page_tokens=64)
    fill(cache, gpu, rng, [600])
    w = _weights(rng, (1, 8, 640))
    before = [_rows(cache, 0, 600)]
    lens = torch.tensor([600], dtype=torch.int32, device=gpu)
    kept, new = m.evict(cache, _dev(w, gpu), lens, budget=130, recent=10)
    pool.truncate(row, 600, 130, 64)
    assert pool.free_pages == 2 + 7 and (row[3:] == -1).all()
    cache.set_block_table(_dev(row[None], gpu))
    _check(cache, before, w, kept, [600], new, 130, 0, 10)


@pytest.mark.parametrize("hq,hk,d", SHAPES)
def test_session_kept_at_its_budget(gpu, hq, hk, d):
    """The operators as a session uses them together: prompts' last tokens and every step add
    weights, sequences over the budget are cut, new rows are appended behind what stayed,
    and the next step sees exactly the rows that the choice kept."""
    import miinfer_amd as m
    rng = np.random.default_rng(d)
    scale = 1 / math.sqrt(d)
    budget, sinks, recent, cap, tokens = 96, 4, 16, 320, 16 // (hq // hk)
    n = [200, 60]
    cache = paged(gpu, rng, hk, d, n, width=cap // 64, spare=10)
    table = cache.block_table.cpu().numpy()
    free = iter(p for p in range(cache.num_pages) if p not in set(table.ravel().tolist()))
    for b in range(2):  # room for what is appended
        for i in range(3):
            if table[b, i] < 0:
                table[b, i] = next(free)
    cache.set_block_table(_dev(table, gpu))
    rows = [list(held(cache, b, n[b])) for b in range(2)]  # k, v per sequence [hk, n, d]
    w = [np.zeros((hk, x)) for x in n]
    dw = torch.zeros((2, hk, cap), device=gpu)
    lens = _dev(np.array(n, np.int32), gpu)
    q = (1.3 * rng.standard_normal((2, tokens, hq, d))).astype(np.float32)
    m.scored_attention(cache, _dev(q, gpu), dw, lengths=lens, max_context=cap)
    for step in range(6):
        if step:
            k_new, v_new = (rng.standard_normal((2, hk, d)).astype(np.float16) for _ in range(2))
            cache.append_batch(_dev(k_new, gpu), _dev(v_new, gpu), lens)
            lens += 1
            n = [x + 1 for x in n]
            q = (1.3 * rng.standard_normal((2, 1, hq, d))).astype(np.float32)
            out, _ = m.scored_attention(cache, _dev(q, gpu), dw, lengths=lens, max_context=cap)
            part, _ = m.window_attention(cache, _dev(q, gpu), lengths=lens, max_context=cap, window=40, sinks=sinks)
        for b in range(2):
            if step:
                k, v = held(cache, b, n[b])
                # what stayed, then the new row (as the cache rounds it)
                assert np.array_equal(k[:, :-1], rows[b][0]) and np.array_equal(v[:, :-1], rows[b][1])
                rows[b] = [k, v]
                w[b] = np.concatenate([w[b], np.zeros((hk, 1))], 1)
            want, got = attend(q[b], *rows[b], n[b], scale)
            w[b] = w[b] + got
            if step:
                close_f32(out[b].cpu().numpy(), want, q[b].astype(np.float64), *rows[b], scale, f"step {step}")
                want, _ = attend(q[b], *rows[b], n[b], scale, 40, sinks)
                close_f32(part[b].cpu().numpy(), want, q[b].astype(np.float64), *rows[b], scale, f"window, step {step}")
            # sums of up to `step + tokens` times the group's probabilities
            assert np.allclose(dw[b, :, :n[b]].cpu().numpy(), w[b], rtol=1e-4, atol=1e-6)
        host = dw.cpu().numpy()
        m.evict(cache, dw, lens, budget=budget, sinks=sinks, recent=recent, max_context=cap, new_lengths=lens, weights_out=dw)
        for b in range(2):
            keep = [_choose(host[b, h], n[b], budget, sinks, recent) for h in range(hk)]
            rows[b] = [np.stack([x[h][keep[h]] for h in range(hk)]) for x in rows[b]]
            w[b] = np.stack([w[b][h][keep[h]] for h in range(hk)])
            n[b] = min(n[b], budget)
        assert lens.tolist() == n
