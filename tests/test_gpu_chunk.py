"""Attention of a ragged batch of chunks over a paged cache against 64-bit attention over the
rows the cache holds (GPU).

Tolerance.  Query, key elements, probabilities and value elements are rounded to fp16 once
(2^-11 of their size each, at most).  With u = 2^-11: a logit is off by at most 2 u times
sum |q_d k_d| scale, taken as 2 u |q| |k| scale / sqrt(d) times 6 for errors that add up like
independent ones (six of their deviations); a probability by that, twice (its own and the
sum's), and u; a value by u.  Outputs are off by that times the largest |v|, and half a step
of the output's type."""
import math

import numpy as np
import pytest
import torch

from tests.part_helpers import attend, held, paged

pytestmark = pytest.mark.gpu

SHAPES = [(32, 8, 128), (24, 4, 256)]
STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _dev(a, gpu):
    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


def _check(cache, q, out, new, lengths, window=0, sinks=0, scale=None, what=""):
    d = cache.head_dim
    scale = 1 / math.sqrt(d) if scale is None else scale
    x = q.float().cpu().numpy().astype(np.float64)
    got = out.float().cpu().numpy().astype(np.float64)
    at, u = 0, 2.0 ** -11
    for b, (n, length) in enumerate(zip(new, lengths)):
        if n:
            k, v = held(cache, b, length)
            want, _ = attend(x[at:at + n], k, v, length, scale, window, sinks)
            top = float(np.abs(v).max()) if length else 0.0
            size = float(np.linalg.norm(x[at:at + n], axis=-1).max() * np.linalg.norm(k, axis=-1).max()) if length else 0.0
            logit = 2 * u * size * abs(scale) / math.sqrt(d) * 6
            tol = top * (2 * logit + 2 * u) + STEP[out.dtype] * np.abs(want) + 2.0 ** -24
            assert np.isfinite(got[at:at + n]).all(), f"{what} seq {b}"
            worst = (np.abs(got[at:at + n] - want) - tol).max()
            assert worst <= 0, f"{what} seq {b} new {n} length {length}: {worst:.3e} over the tolerance"
            # errors of many keys do not all point one way: the norm is off by far less
            rel = np.linalg.norm(got[at:at + n] - want) / max(np.linalg.norm(want), 1e-30)
            assert rel <= 4 * u + STEP[out.dtype], f"{what} seq {b}: relative {rel:.2e}"
        at += n


def _call(gpu, cache, q, new, lengths, **more):
    import miinfer_amd as m
    off = _dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), gpu)
    return m.chunk_attention(cache, q, off, _dev(np.array(lengths, np.int32), gpu), **more)


def _query(rng, gpu, shape, dtype):
    return torch.from_numpy(1.3 * rng.standard_normal(shape)).to(gpu).to(dtype)


@pytest.mark.parametrize("hq,hk,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 4), (100, 0), (64, 130), (5000, 7)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_chunk_ragged(gpu, hq, hk, d, window, sinks, dtype):
    """Empty chunks, single tokens, chunks of more and less than an item's rows, contexts around
    steps and pages, whole prompts."""
    rng = np.random.default_rng(window + sinks + d)
    new = [1, 0, 5, 33, 1, 70, 129, 2, 64, 11]
    lengths = [1, 77, 5, 64, 300, 70, 511, 2, 65, 1000]
    cache = paged(gpu, rng, hk, d, lengths)
    q = _query(rng, gpu, (sum(new), hq, d), dtype)
    out = _call(gpu, cache, q, new, lengths, max_tokens=129, max_context=1000, window=window, sinks=sinks)
    assert out.dtype == dtype
    _check(cache, q, out, new, lengths, window, sinks)


@pytest.mark.parametrize("hq,hk,d", SHAPES)
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_chunk_quant_modes(gpu, hq, hk, d, mode):
    rng = np.random.default_rng(mode)
    new, lengths = [90, 3, 200], [700, 400, 200]
    cache = paged(gpu, rng, hk, d, lengths, mode=mode, page=128)
    q = _query(rng, gpu, (sum(new), hq, d), torch.float16)
    for window, sinks in ((0, 0), (75, 40)):
        out = _call(gpu, cache, q, new, lengths, max_context=704, window=window, sinks=sinks)
        _check(cache, q, out, new, lengths, window, sinks, what=f"mode {mode} window {window}")


@pytest.mark.parametrize("hq,hk,d", [(1, 1, 128), (16, 1, 256), (34, 2, 128), (40, 1, 256)])
def test_chunk_groups(gpu, hq, hk, d):
    """Groups of one query head, sixteen, and numbers that do not divide an item's rows."""
    rng = np.random.default_rng(hq)
    new, lengths = [130, 17], [400, 301]
    cache = paged(gpu, rng, hk, d, lengths)
    q = _query(rng, gpu, (147, hq, d), torch.float16)
    for window, sinks in ((0, 0), (50, 3)):
        _check(cache, q, _call(gpu, cache, q, new, lengths, window=window, sinks=sinks), new, lengths, window, sinks)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("window,sinks,page", [(0, 0, 64), (70, 0, 128), (33, 4, 64), (64, 130, 192), (1, 0, 64)])
def test_chunk_many_rows(gpu, d, mode, window, sinks, page):
    """Many rows of every sequence: prompts, odd and even numbers of steps, an empty chunk, a single token."""
    rng = np.random.default_rng(d + mode + window)
    new, lengths = [130, 0, 200, 1, 160], [130, 40, 500, 333, 193]
    cache = paged(gpu, rng, 1, d, lengths, mode=mode, page=page)
    q = _query(rng, gpu, (sum(new), 16, d), torch.bfloat16)
    out = _call(gpu, cache, q, new, lengths, max_tokens=200, max_context=500, window=window, sinks=sinks)
    _check(cache, q, out, new, lengths, window, sinks)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("mode", [0, 3])
def test_chunk_many_rows_masked_keys_and_cuts(gpu, d, mode):
    """Many rows over a long context, whose items go over many workgroups; what no token sees may
    hold anything, and pages that no token sees may be missing."""
    rng = np.random.default_rng(d + mode)
    n, t = 3005, 100
    cache = paged(gpu, rng, 1, d, [n], mode=mode)
    q = _query(rng, gpu, (t, 16, d), torch.float16)
    for window, sinks in ((0, 0), (700, 5)):
        out = _call(gpu, cache, q, [t], [n], window=window, sinks=sinks, max_context=cache.capacity)
        _check(cache, q, out, [t], [n], window, sinks)
    page = cache.block_table[0].long()
    hidden = [j for j in range(3008) if not (n - t - window + 1 <= j < n or j < sinks)]
    for name, shape in (("k_scales", (cache.num_pages, 1, 64, d // 32)), ("v_scales", (cache.num_pages, 1, 64, d // 32)),
                        ("k_codes", (cache.num_pages, 1, 4, d // 64, 4, 16, 2, 8)),
                        ("v_codes", (cache.num_pages, 1, 2, d, 4, 2, 4))):
        x = getattr(cache, name)
        if x is None or x.dtype == torch.int8:
            continue
        x = x.view(torch.float16).view(shape)
        for i, j in enumerate(hidden):
            bad, s, p = float("nan") if i % 2 else float("inf"), j % 64, page[j // 64]
            if "scales" in name:
                x[p, :, s] = bad
            elif name == "k_codes":
                x[p, :, s // 16, :, :, s % 16] = bad
            else:
                x[p, :, s // 32, :, s % 16 // 4, s % 32 // 16, s % 4] = bad
    table = cache.block_table.clone()
    table[0, 1:(n - t - window) // 64] = -1
    cache.set_block_table(table)
    got = _call(gpu, cache, q, [t], [n], window=window, sinks=sinks, max_context=cache.capacity)
    assert torch.equal(got, out)


def test_chunk_long_items_are_cut(gpu):
    """Few rows over a long context: an item's keys go over many workgroups; and types of query
    and output that differ."""
    rng = np.random.default_rng(1)
    hq, hk, d, new, lengths = 32, 8, 128, [3, 40], [20000, 9001]
    cache = paged(gpu, rng, hk, d, lengths, page=256)
    q = _query(rng, gpu, (43, hq, d), torch.bfloat16)
    for out_type in (torch.float32, torch.float16):
        out = _call(gpu, cache, q, new, lengths, max_tokens=40, max_context=20000, out=torch.empty(q.shape, dtype=out_type, device=gpu))
        _check(cache, q, out, new, lengths)


def test_chunk_many_items(gpu):
    """More items and sequences than a workgroup's threads: the plan's sums go over several rounds."""
    rng = np.random.default_rng(2)
    hq, hk, d = 16, 2, 128
    new = [int(x) for x in rng.integers(0, 9, 700)]
    new[5], new[400] = 3000, 1500
    lengths = [n + int(x) for n, x in zip(new, rng.integers(0, 90, 700))]
    lengths[9] += 2000
    cache = paged(gpu, rng, hk, d, lengths, width=50)
    q = _query(rng, gpu, (sum(new), hq, d), torch.float16)
    out = _call(gpu, cache, q, new, lengths, max_tokens=3000, max_context=3200)
    pick = [i for i in range(700) if i not in (5, 400)]
    at = np.concatenate([[0], np.cumsum(new)])
    rows = torch.cat([torch.arange(at[i], at[i + 1]) for i in pick]).to(gpu)
    sub = cache.block_table[pick].contiguous()
    tables = cache.block_table
    cache.set_block_table(sub)
    _check(cache, q[rows], out[rows], [new[i] for i in pick], [lengths[i] for i in pick])
    cache.set_block_table(tables[[5, 400]].contiguous())
    # the long ones: their last tokens
    for b, i in enumerate((5, 400)):
        k, v = held(cache, b, lengths[i])
        want, _ = attend(q[at[i + 1] - 4:at[i + 1]].float().cpu().numpy(), k, v, lengths[i], 1 / math.sqrt(d))
        got = out[at[i + 1] - 4:at[i + 1]].float().cpu().numpy()
        assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(want)


def test_chunk_contiguous_scale_and_rows_left_alone(gpu):
    """One chunk over a contiguous cache; negative and zero scales; rows behind the last chunk and a
    context shorter than its tokens."""
    import miinfer_amd as m
    rng = np.random.default_rng(3)
    hq, hk, d, n, length = 32, 8, 128, 50, 333
    cache = m.KvCache.contiguous(hk, d, 384)
    cache.append(*(_dev(rng.standard_normal((length, hk, d)).astype(np.float16), gpu) for _ in range(2)))
    q = _query(rng, gpu, (60, hq, d), torch.float16)
    for scale in (None, -0.05, 0.0, 0.3):
        out = torch.full_like(q, 7.0)
        _call(gpu, cache, q, [n], [length], scale=scale, out=out)
        assert bool((out[n:] == 7).all())
        _check(cache, q[:n], out[:n], [n], [length], scale=scale, what=f"scale {scale}")
    # a length below the chunk: the tokens in front of position 0 see nothing
    out = _call(gpu, cache, q, [n], [20])
    assert not out[:n - 20].any()
    want = _call(gpu, cache, q[n - 20:n].contiguous(), [20], [20])
    assert torch.equal(out[n - 20:n], want)
    # an empty batch of chunks writes nothing
    out = torch.full_like(q, 7.0)
    _call(gpu, cache, q, [0], [length], out=out)
    assert bool((out == 7).all())


def test_chunk_masked_keys_may_hold_anything(gpu):
    """NaN and infinities behind the context and in front of every window leave the result alone."""
    rng = np.random.default_rng(4)
    hq, hk, d, new, n, window, sinks = 32, 8, 128, [9], 301, 100, 5
    for mode in (3, 0):
        cache = paged(gpu, rng, hk, d, [n], mode=mode, width=6)
        q = _query(rng, gpu, (9, hq, d), torch.float16)
        want = _call(gpu, cache, q, new, [n], max_context=384, window=window, sinks=sinks).clone()
        hidden = [j for j in range(320) if not (n - 9 - window + 1 <= j < n or j < sinks)]
        page = cache.block_table[0].long()
        for name, shape in (("k_scales", (cache.num_pages, hk, 64, d // 32)), ("v_scales", (cache.num_pages, hk, 64, d // 32)),
                            ("k_codes", (cache.num_pages, hk, 4, d // 64, 4, 16, 2, 8)),
                            ("v_codes", (cache.num_pages, hk, 2, d, 4, 2, 4))):
            t = getattr(cache, name)
            if t is None or t.dtype == torch.int8:
                continue
            t = t.view(torch.float16).view(shape)
            for i, j in enumerate(hidden):
                x, s, p = float("nan") if i % 2 else float("inf"), j % 64, page[j // 64]
                if "scales" in name:
                    t[p, :, s] = x
                elif name == "k_codes":
                    t[p, :, s // 16, :, :, s % 16] = x
                else:
                    t[p, :, s // 32, :, s % 16 // 4, s % 32 // 16, s % 4] = x
        table = cache.block_table.clone()
        table[0, 1:(n - 9 - window) // 64] = -1  # pages that no token sees
        cache.set_block_table(table)
        got = _call(gpu, cache, q, new, [n], max_context=384, window=window, sinks=sinks)
        assert torch.equal(got, want), f"mode {mode}"


def test_chunk_graphs_streams_and_equal_bits(gpu):
    """Two captured calls that share a workspace, replayed with other offsets and lengths, eager
    work between; another stream; the same bits every time."""
    import miinfer_amd as m
    rng = np.random.default_rng(5)
    hq, hk, d, cap, total = 24, 4, 256, 1024, 160
    full = [1000, 300, 640]
    cache = paged(gpu, rng, hk, d, full, width=cap // 64)
    q = [_query(rng, gpu, (total, hq, d), torch.bfloat16) for _ in range(2)]
    outs = [torch.zeros_like(x) for x in q]
    off = _dev(np.array([0, 100, 101, 160], np.int32), gpu)
    lens = _dev(np.array(full, np.int32), gpu)
    ws = torch.empty(m.chunk_workspace_bytes(cache, hq, 3, total, 120, cap, 200, 4), dtype=torch.uint8, device=gpu)

    def step(i, out, stream=None):
        return m.chunk_attention(cache, q[i], off, lens, max_tokens=120, max_context=cap, window=200, sinks=4, out=out,
                                 workspace=ws, stream=stream)

    step(0, outs[0])
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(i, outs[i])
        graphs.append(g)
    for turn, (o, n) in enumerate([([0, 100, 101, 160], full), ([0, 3, 60, 61], [500, 299, 64]), ([0, 0, 120, 120], [1, 200, 9]),
                                   ([0, 100, 101, 160], full)]):
        off.copy_(torch.tensor(o, dtype=torch.int32))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        for i in (0, 1):
            outs[i].fill_(3.0)
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            want = torch.full_like(outs[i], 3.0)
            step(i, want)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want), (turn, i)
            new = np.diff(o).tolist()
            _check(cache, q[i][:o[3]], want[:o[3]], new, n, 200, 4, what=f"turn {turn}")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = step(0, None, stream=s)
    s.synchronize()
    assert torch.equal(got[:160], outs[0][:160])


def test_chunk_many_rows_graph_and_two_streams(gpu):
    """A captured call over expanded keys, replayed with other offsets and lengths, some of them few rows;
    two calls at once on streams and workspaces of their own; out over q."""
    import miinfer_amd as m
    rng = np.random.default_rng(8)
    hq, hk, d, cap, total = 32, 2, 128, 1024, 300
    full = [1000, 300]
    cache = paged(gpu, rng, hk, d, full, width=cap // 64)
    q = _query(rng, gpu, (total, hq, d), torch.bfloat16)
    off = _dev(np.array([0, 150, 300], np.int32), gpu)
    lens = _dev(np.array(full, np.int32), gpu)

    def room():
        return torch.empty(m.chunk_workspace_bytes(cache, hq, 2, total, 200, cap, 300, 4), dtype=torch.uint8, device=gpu)

    def step(out, ws, x=q, stream=None):
        return m.chunk_attention(cache, x, off, lens, max_tokens=200, max_context=cap, window=300, sinks=4, out=out, workspace=ws,
                                 stream=stream)

    out, ws = torch.zeros_like(q), room()
    step(out, ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(out, ws)
    for o, n in (([0, 150, 300], full), ([0, 1, 9], [700, 8]), ([0, 0, 200], [5, 290]), ([0, 150, 300], full)):
        off.copy_(torch.tensor(o, dtype=torch.int32))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        want = step(torch.full_like(q, 3.0), room())
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        _check(cache, q[:o[2]], want[:o[2]], np.diff(o).tolist(), n, 300, 4)
        assert bool((want[o[2]:] == 3).all())
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces, outs = [room() for _ in streams], [torch.empty_like(q) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, w, o in zip(streams, spaces, outs):
            step(o, w, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], out) and torch.equal(outs[1], out)
    x = q.clone()
    assert torch.equal(step(x, ws, x=x), out)


def test_chunk_agrees_with_window_decode(gpu):
    """Chunks of one token are the decode form's rows."""
    import miinfer_amd as m
    rng = np.random.default_rng(6)
    hq, hk, d, lengths = 32, 8, 128, [1, 50, 700, 1030]
    cache = paged(gpu, rng, hk, d, lengths)
    q = _query(rng, gpu, (4, hq, d), torch.float16)
    lens = _dev(np.array(lengths, np.int32), gpu)
    off = torch.arange(5, dtype=torch.int32, device=gpu)
    a = m.chunk_attention(cache, q, off, lens, max_tokens=1, max_context=1030, window=300, sinks=8, out=torch.empty(q.shape, device=gpu))
    b, _ = m.window_attention(cache, q, lengths=lens, max_context=1030, window=300, sinks=8)
    assert float((a - b).norm()) <= 2.0 ** -9 * float(b.norm())
