"""Decode attention over a sliding window and the first tokens, and decode attention that
adds up every key's weight, against 64-bit attention over the rows the cache holds (GPU)."""
import math

import numpy as np
import pytest
import torch

from tests.part_helpers import attend, close_f32, close_weights, held, paged

pytestmark = pytest.mark.gpu

SHAPES = [(32, 8, 128), (24, 4, 256)]


def _dev(a, gpu):
    return torch.from_numpy(np.ascontiguousarray(a)).to(gpu)


def _query(rng, shape, f32):
    q = 1.3 * rng.standard_normal(shape)
    return q.astype(np.float32 if f32 else np.float16)


def _check(cache, q, out, lengths, window, sinks, gate=None, what=""):
    scale = 1 / math.sqrt(cache.head_dim)
    for b, n in enumerate(lengths):
        k, v = held(cache, b, n)
        want, _ = attend(q[b], k, v, n, scale, window, sinks)
        if gate is not None:
            want = want / (1 + np.exp(-gate[b].astype(np.float64)))
        close_f32(out[b], want, q[b].astype(np.float64), k, v, scale, f"{what} seq {b} length {n}")


@pytest.mark.parametrize("hq,hk,d", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (31, 0), (32, 4), (33, 33), (100, 31), (64, 200), (5000, 3)])
def test_window_masks(gpu, hq, hk, d, window, sinks):
    """Lengths around steps, pages and the window's own edges."""
    import miinfer_amd as m
    rng = np.random.default_rng(window * 7 + sinks + d)
    lengths = [0, 1, 2, 31, 32, 33, 63, 64, 65, 100, 129, 331, 700]
    cache = paged(gpu, rng, hk, d, lengths)
    q = _query(rng, (len(lengths), 1, hq, d), False)
    out, _ = m.window_attention(cache, _dev(q, gpu), lengths=_dev(np.array(lengths, np.int32), gpu), max_context=700,
                                window=window, sinks=sinks)
    _check(cache, q, out.cpu().numpy(), lengths, window, sinks)


@pytest.mark.parametrize("hq,hk,d", SHAPES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4])
@pytest.mark.parametrize("f32", [False, True])
def test_window_tokens(gpu, hq, hk, d, tokens, f32):
    """Several tokens: each its own mask; a context shorter than its tokens has rows that see
    nothing and get zeros."""
    import miinfer_amd as m
    if tokens * hq // hk > 16:
        pytest.skip("more columns than the kernel has")
    rng = np.random.default_rng(tokens + d)
    lengths = [1, tokens, 40, 64, 97, 300, 1025]
    cache = paged(gpu, rng, hk, d, lengths, page=128)
    q = _query(rng, (len(lengths), tokens, hq, d), f32)
    gate = rng.standard_normal(q.shape).astype(np.float32)
    lens = _dev(np.array(lengths, np.int32), gpu)
    for window, sinks in ((40, 5), (0, 0), (2, 0)):
        out, gated = m.window_attention(cache, _dev(q, gpu), lengths=lens, max_context=1100, window=window, sinks=sinks,
                                        gate=_dev(gate, gpu), out=torch.empty(q.shape, device=gpu))
        _check(cache, q, out.cpu().numpy(), lengths, window, sinks, what=f"window {window}")
        _check(cache, q, gated.cpu().numpy(), lengths, window, sinks, gate, f"gated, window {window}")


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("hq,hk,d", SHAPES)
def test_window_quant_modes(gpu, mode, hq, hk, d):
    import miinfer_amd as m
    rng = np.random.default_rng(mode)
    lengths = [77, 500, 260]
    cache = paged(gpu, rng, hk, d, lengths, mode=mode)
    for f32 in (False, True):
        q = _query(rng, (3, 2, hq, d), f32)
        out, _ = m.window_attention(cache, _dev(q, gpu), lengths=_dev(np.array(lengths, np.int32), gpu), max_context=512,
                                    window=130, sinks=9)
        _check(cache, q, out.cpu().numpy(), lengths, 130, 9)


@pytest.mark.parametrize("hq,hk,d", [(16, 1, 256), (16, 1, 128), (4, 4, 128), (10, 2, 256)])
def test_window_groups(gpu, hq, hk, d):
    """One query head per kv head, sixteen, and a number that is no power of two."""
    import miinfer_amd as m
    rng = np.random.default_rng(hq)
    lengths = [900, 33]
    cache = paged(gpu, rng, hk, d, lengths)
    q = _query(rng, (2, 1, hq, d), True)
    out, _ = m.window_attention(cache, _dev(q, gpu), lengths=_dev(np.array(lengths, np.int32), gpu), max_context=960,
                                window=300, sinks=70)
    _check(cache, q, out.cpu().numpy(), lengths, 300, 70)


def test_window_many_sequences(gpu):
    """More sequences than a wave has lanes, ragged: the plan's scan goes over two rounds."""
    import miinfer_amd as m
    rng = np.random.default_rng(5)
    lengths = [int(x) for x in rng.integers(0, 400, 150)]
    cache = paged(gpu, rng, 2, 128, lengths)
    q = _query(rng, (150, 1, 8, 128), False)
    lens = _dev(np.array(lengths, np.int32), gpu)
    for window, sinks in ((0, 0), (90, 3)):
        out, _ = m.window_attention(cache, _dev(q, gpu), lengths=lens, max_context=448, window=window, sinks=sinks)
        _check(cache, q, out.cpu().numpy(), lengths, window, sinks)


def test_window_long_context_contiguous_state(gpu):
    """A long contiguous cache, the length from a decode state, against the whole-context
    kernel where the window hides nothing."""
    import miinfer_amd as m
    rng = np.random.default_rng(6)
    hq, hk, d, n = 32, 8, 128, 20001
    cache = m.KvCache.contiguous(hk, d, 20032)
    k, v = (_dev(rng.standard_normal((n, hk, d)).astype(np.float16), gpu) for _ in range(2))
    cache.append(k, v)
    q = _query(rng, (1, hq, d), True)
    st = m.make_decode_state(n - 1, device=gpu)
    out, _ = m.window_attention(cache, _dev(q, gpu), decode_state=st, window=1024, sinks=4)
    _check(cache, q[:, None], out.cpu().numpy()[:, None], [n], 1024, 4)
    whole, _ = m.window_attention(cache, _dev(q, gpu), decode_state=st, window=0)
    ref, _ = m.decode_attention(cache, _dev(q, gpu), decode_state=st)
    # the older kernel rounds its probabilities to fp16 once: 2^-11 of sum p |v|
    assert float((whole - ref).abs().max()) <= 2.0 ** -11 * float(v.abs().max())


def test_window_masked_keys_may_hold_anything(gpu):
    """NaN and infinite scales at keys that no token sees (behind the context, in front of
    the window, in steps that are read for their other keys) leave the result alone."""
    import miinfer_amd as m
    rng = np.random.default_rng(7)
    hq, hk, d, n, window, sinks = 32, 8, 128, 301, 100, 5
    for mode in (3, 0):
        cache = paged(gpu, rng, hk, d, [n], mode=mode, width=6)
        q = _dev(_query(rng, (1, hq, d), False), gpu)
        lens = torch.tensor([n], dtype=torch.int32, device=gpu)
        args = dict(lengths=lens, max_context=384, window=window, sinks=sinks)
        want, _ = m.window_attention(cache, q, **args)
        want = want.clone()
        hidden = [j for j in range(320) if not (n - window <= j < n or j < sinks)]
        page = cache.block_table[0].long()
        for planes, shape in ((("k_scales", "v_scales"), (cache.num_pages, hk, 64, d // 32)),
                              (("k_codes",), (cache.num_pages, hk, 4, d // 64, 4, 16, 2, 8)),
                              (("v_codes",), (cache.num_pages, hk, 2, d, 4, 2, 4))):
            for name in planes:
                t = getattr(cache, name)
                if t is None or (t.dtype != torch.float16 and "codes" in name):
                    continue
                t = t.view(torch.float16).view(shape)
                for i, j in enumerate(hidden):
                    x = float("nan") if i % 2 else float("inf")
                    s = j % 64
                    if "scales" in name:
                        t[page[j // 64], :, s] = x
                    elif name == "k_codes":
                        t[page[j // 64], :, s // 16, :, :, s % 16] = x
                    else:
                        t[page[j // 64], :, s // 32, :, s % 16 // 4, s % 32 // 16, s % 4] = x
        got, _ = m.window_attention(cache, q, **args)
        assert torch.equal(got, want), f"mode {mode}"


def test_window_unseen_pages_need_no_entry(gpu):
    """Pages in front of the window may be given back: their entries are -1."""
    import miinfer_amd as m
    rng = np.random.default_rng(8)
    cache = paged(gpu, rng, 8, 128, [1000])
    q = _dev(_query(rng, (1, 32, 128), False), gpu)
    args = dict(lengths=torch.tensor([1000], dtype=torch.int32, device=gpu), max_context=1000, window=150, sinks=10)
    want = m.window_attention(cache, q, **args)[0].clone()
    table = cache.block_table.clone()
    table[0, 1:(1000 - 150) // 64] = -1
    cache.set_block_table(table)
    assert torch.equal(m.window_attention(cache, q, **args)[0], want)


@pytest.mark.parametrize("scored", [False, True])
def test_part_graphs_share_a_workspace(gpu, scored):
    """Two captured steps that share one workspace, replayed in turn with eager work and
    new lengths between them."""
    import miinfer_amd as m
    rng = np.random.default_rng(9)
    hq, hk, d, cap = 32, 8, 128, 1024
    lens0 = [900, 40, 513]
    cache = paged(gpu, rng, hk, d, lens0, width=cap // 64)
    lens = _dev(np.array(lens0, np.int32), gpu)
    q = [_dev(_query(rng, (3, 1, hq, d), False), gpu) for _ in range(2)]
    outs = [torch.zeros((3, 1, hq, d), device=gpu) for _ in range(2)]
    weights = torch.zeros((3, hk, cap), device=gpu)
    need = m.scored_workspace_bytes(cache, hq, 3, 1, cap) if scored else m.window_workspace_bytes(cache, hq, 3, 1, cap, 200, 4)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)

    def step(i, out, w):
        if scored:
            m.scored_attention(cache, q[i], w, lengths=lens, max_context=cap, out=out, workspace=ws)
        else:
            m.window_attention(cache, q[i], lengths=lens, max_context=cap, window=200, sinks=4, out=out, workspace=ws)

    step(0, outs[0], weights)
    weights.zero_()
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(i, outs[i], weights)
        graphs.append(g)
    want_w = torch.zeros_like(weights)
    for turn in range(4):
        lens.copy_(torch.tensor([900 - 250 * turn, 40 - turn, 513 - 64 * turn], dtype=torch.int32))
        for i in (0, 1):
            outs[i].zero_()
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            want = torch.zeros_like(outs[i])
            step(i, want, want_w)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want), (turn, i)
        if scored:
            assert torch.equal(weights, want_w)


def test_gated_output_is_made_when_all_else_is_given(gpu):
    import miinfer_amd as m
    rng = np.random.default_rng(21)
    cache = paged(gpu, rng, 8, 128, [100])
    q = _dev(_query(rng, (1, 32, 128), False), gpu)
    gate = torch.randn(q.shape, device=gpu)
    lens = _dev(np.array([100], np.int32), gpu)
    w = torch.zeros((1, 8, 128), device=gpu)
    out, both = m.window_attention(cache, q, window=0, lengths=lens, max_context=128, gate=gate)
    assert out is None
    ws = torch.empty(m.scored_workspace_bytes(cache, 32, 1, 1, 128), dtype=torch.uint8, device=gpu)
    for call in (lambda **o: m.window_attention(cache, q, window=0, **o), lambda **o: m.scored_attention(cache, q, w, **o)):
        out, gated = call(lengths=lens, max_context=128, gate=gate, out=torch.empty(q.shape, device=gpu), workspace=ws)
        assert torch.equal(gated, both)
        assert float((out * torch.sigmoid(gate) - gated).abs().max()) <= 1e-5


def test_part_other_stream(gpu):
    import miinfer_amd as m
    rng = np.random.default_rng(10)
    cache = paged(gpu, rng, 4, 256, [700, 90])
    q = _dev(_query(rng, (2, 24, 256), False), gpu)
    lens = _dev(np.array([700, 90], np.int32), gpu)
    want = m.window_attention(cache, q, lengths=lens, max_context=704, window=300)[0].clone()
    w = torch.zeros((2, 4, 704), device=gpu)
    m.scored_attention(cache, q, w, lengths=lens, max_context=704)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    w2 = torch.zeros_like(w)
    s.wait_stream(torch.cuda.current_stream())
    got, _ = m.window_attention(cache, q, lengths=lens, max_context=704, window=300, stream=s)
    m.scored_attention(cache, q, w2, lengths=lens, max_context=704, stream=s)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(w2, w)


@pytest.mark.parametrize("hq,hk,d", SHAPES)
@pytest.mark.parametrize("tokens,f32,mode", [(1, False, 3), (2, True, 3), (1, True, 0), (2, False, 1), (1, False, 2)])
def test_scored_weights(gpu, hq, hk, d, tokens, f32, mode):
    """Weights grow from what they were; entries at or behind a sequence's length stay."""
    import miinfer_amd as m
    rng = np.random.default_rng(tokens + d + mode)
    lengths = [0, 1, 2, 33, 64, 257, 1200]
    cache = paged(gpu, rng, hk, d, lengths, mode=mode, width=24)
    q = _query(rng, (len(lengths), tokens, hq, d), f32)
    lens = _dev(np.array(lengths, np.int32), gpu)
    w0 = rng.random((len(lengths), hk, 1300)).astype(np.float32)
    w = _dev(w0, gpu)
    z = torch.zeros_like(w)
    out, _ = m.scored_attention(cache, _dev(q, gpu), w, lengths=lens, max_context=1216)
    m.scored_attention(cache, _dev(q, gpu), z, lengths=lens, max_context=1216)
    assert torch.equal(_dev(w0, gpu) + z, w)  # one addition to what was there
    scale = 1 / math.sqrt(d)
    for b, n in enumerate(lengths):
        k, v = held(cache, b, n)
        want, weight = attend(q[b], k, v, n, scale)
        x = q[b].astype(np.float64)
        close_f32(out[b].cpu().numpy(), want, x, k, v, scale, f"length {n}")
        close_weights(z[b, :, :n].cpu().numpy(), weight, x, k, scale, tokens * hq // hk, f"length {n}")
        assert not z[b, :, n:].any()
        # every token that sees a key gives its heads' weight away once
        total = hq // hk * min(tokens, n)
        assert abs(float(z[b].double().sum()) - hk * total) <= 1e-4 * max(1, hk * total)


def test_scored_equal_bits(gpu):
    """No order of additions depends on timing."""
    import miinfer_amd as m
    rng = np.random.default_rng(12)
    cache = paged(gpu, rng, 8, 128, [9000, 3000], page=256)
    q = _dev(_query(rng, (2, 32, 128), False), gpu)
    lens = _dev(np.array([9000, 3000], np.int32), gpu)
    got = []
    for _ in range(8):
        w = torch.zeros((2, 8, 9000), device=gpu)
        out, _ = m.scored_attention(cache, q, w, lengths=lens, max_context=9000)
        got.append((out, w))
    for out, w in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(w, got[0][1])
