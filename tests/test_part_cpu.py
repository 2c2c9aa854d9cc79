"""Refusals of the operators over part of a cache, and their host bookkeeping: nothing is
launched, so no GPU is needed."""
import ctypes

import numpy as np
import pytest

from tests.test_abi_cpu import _lib, _view

P = ctypes.c_void_p(0x10000)
F = ctypes.c_float(0.1)


def _paged(**over):
    args = {"layout": 1, "page_tokens": 256, "num_pages": 64, "block_table": 0x4000, "table_stride": 16}
    args.update(over)
    return _view(**args)


def _window(lib, v, **over):
    a = dict(q=P, dtype=0, heads=32, scale=F, batch=2, tokens=1, lengths=P, state=None, most=4096, window=128, sinks=4, out=P,
             gate=None, gated=None, ws=P, bytes=1 << 40)
    a.update(over)
    return lib.miikv_decode_attn_window(None if v is None else ctypes.byref(v), a["q"], a["dtype"], a["heads"], a["scale"],
                                        a["batch"], a["tokens"], a["lengths"], a["state"], a["most"], a["window"],
                                        a["sinks"], a["out"], a["gate"], a["gated"], a["ws"], a["bytes"], None)


BAD = [
    ({"q": None}, 1), ({"dtype": 2}, 1), ({"heads": 30}, 1), ({"heads": 0}, 1), ({"scale": ctypes.c_float(float("nan"))}, 1),
    ({"batch": 0}, 1), ({"batch": 70000}, 1), ({"tokens": 0}, 1), ({"tokens": 5}, 2), ({"tokens": 0xffffffff}, 2),
    ({"lengths": None}, 1), ({"lengths": None, "state": P}, 1), ({"most": 0}, 1), ({"most": 4097}, 1),
    ({"out": None}, 1), ({"gate": P}, 1), ({"gated": P}, 1),
    ({"ws": None}, 3), ({"bytes": 16}, 3),
    ({"q": ctypes.c_void_p(0x10002)}, 1), ({"out": ctypes.c_void_p(0x10004)}, 1), ({"ws": ctypes.c_void_p(0x10008)}, 1),
    ({"gate": ctypes.c_void_p(0x10004), "gated": P}, 1),
]


@pytest.mark.parametrize("over,status", BAD)
def test_window_refuses(over, status):
    L = _lib()
    assert _window(L.lib(), _paged(), **over) == status


@pytest.mark.parametrize("over,status", [({"head_dim": 64}, 2), ({"quant_mode": 9}, 1), ({"block_table": None}, 1),
                                         ({"k_codes": 0x1008}, 1), ({"v_scales": 0x2004}, 1), ({"page_tokens": 100}, 1)])
def test_window_refuses_views(over, status):
    L = _lib()
    assert _window(L.lib(), _paged(**over)) == status
    assert _window(L.lib(), None) == 1
    # a contiguous cache holds one sequence
    assert _window(L.lib(), _view(), batch=2) == 1


@pytest.mark.parametrize("over,status", BAD)
def test_scored_refuses(over, status):
    L = _lib()
    lib = L.lib()
    a = dict(q=P, dtype=0, heads=32, scale=F, batch=2, tokens=1, lengths=P, state=None, most=4096, w=P, stride=4096, out=P,
             gate=None, gated=None, ws=P, bytes=1 << 40)

    def go(**more):
        x = {**a, **more}
        return lib.miikv_decode_attn_scored(ctypes.byref(_paged()), x["q"], x["dtype"], x["heads"], x["scale"], x["batch"],
                                            x["tokens"], x["lengths"], x["state"], x["most"], x["w"], x["stride"], x["out"],
                                            x["gate"], x["gated"], x["ws"], x["bytes"], None)
    assert go(**over) == status
    assert go(w=None) == 1 and go(stride=4095) == 1


def test_workspace_sizes():
    L = _lib()
    lib = L.lib()
    v = _paged()
    r = ctypes.byref(v)
    one = lib.miikv_window_workspace_bytes(r, 32, 1, 1, 4096, 1024, 4)
    assert 0 < one <= lib.miikv_window_workspace_bytes(r, 32, 1, 1, 4096, 0, 0)
    # a window that hides nothing takes what the whole context takes, however large it is
    assert lib.miikv_window_workspace_bytes(r, 32, 1, 1, 4096, 0xffffffff, 0xffffffff) == \
        lib.miikv_window_workspace_bytes(r, 32, 1, 1, 4096, 0, 0)
    # scores of every column and key besides
    assert lib.miikv_scored_workspace_bytes(r, 32, 2, 2, 4001) >= 2 * 8 * 8 * 4001 * 4
    for bad in ((30, 1, 1, 4096), (32, 0, 1, 4096), (32, 1, 5, 4096), (32, 1, 1, 0), (32, 1, 1, 4097)):
        assert lib.miikv_window_workspace_bytes(r, *bad, 64, 0) == 0
        assert lib.miikv_scored_workspace_bytes(r, *bad) == 0
    # the size asked for is the one that is checked
    need = lib.miikv_window_workspace_bytes(r, 32, 2, 1, 4096, 128, 4)
    assert _window(lib, v, bytes=need - 1) == L.MIIKV_EWORKSPACE


def _evict(lib, v, **over):
    a = dict(w=P, stride=4096, batch=2, lengths=P, most=4096, sinks=4, recent=16, budget=256, dst=None, dst_stride=0, kept=P,
             new=P, out=None, out_stride=0)
    a.update(over)
    return lib.miikv_evict(None if v is None else ctypes.byref(v), a["w"], a["stride"], a["batch"], a["lengths"], a["most"],
                           a["sinks"], a["recent"], a["budget"], a["dst"], a["dst_stride"], a["kept"], a["new"], a["out"],
                           a["out_stride"], None)


@pytest.mark.parametrize("over", [
    {"w": None}, {"stride": 4095}, {"batch": 0}, {"batch": 70000}, {"lengths": None}, {"most": 0}, {"most": 4097}, {"budget": 0},
    {"budget": 19}, {"sinks": 0xffffffff, "recent": 1}, {"kept": None}, {"new": None},
    {"dst": P, "dst_stride": 0}, {"dst": P, "dst_stride": 3, "budget": 769}, {"out": ctypes.c_void_p(0x20000), "out_stride": 255},
    {"out": P, "out_stride": 4000},
    # weights over each other, not in place: behind the start, in the last row, in front and reaching in
    {"out": ctypes.c_void_p(P.value + 4), "out_stride": 4096},
    {"out": ctypes.c_void_p(P.value + 4 * (15 * 4096 + 4095)), "out_stride": 256},
    {"out": ctypes.c_void_p(P.value - 4 * (15 * 256 + 255)), "out_stride": 256},
])
def test_evict_refuses(over):
    L = _lib()
    assert _evict(L.lib(), _paged(), **over) == L.MIIKV_EINVAL
    assert _evict(L.lib(), None) == L.MIIKV_EINVAL
    # a contiguous cache holds one sequence and has no pages to move to
    assert _evict(L.lib(), _view(), batch=2) == L.MIIKV_EINVAL
    assert _evict(L.lib(), _view(), batch=1, dst=P, dst_stride=16) == L.MIIKV_EINVAL


def test_pool_truncate():
    from miinfer_amd import MiikvError, reuse
    pool = reuse.PagePool(8)
    row = np.array([pool.alloc() for _ in range(5)] + [-1], np.int32)
    child, copies = pool.fork(row, 4 * 64, 64)
    pool.truncate(row, 5 * 64 - 3, 2 * 64 + 1, 64)
    assert (row >= 0).tolist() == [True, True, True, False, False, False]
    assert pool.free_pages == 4  # the fourth page is still the fork's
    assert pool.refcount(int(child[3])) == 1
    pool.truncate(row, 3 * 64, 3 * 64, 64)  # nothing to drop
    for length, new in ((64, 65), (5 * 64, 64)):  # longer than it was; pages that the row does not hold
        before = row.copy()
        with pytest.raises(MiikvError):
            pool.truncate(row, length, new, 64)
        assert (row == before).all()
    pool.truncate(row, 3 * 64, 0, 64)
    assert (row == -1).all() and not copies


def test_python_refusals():
    """The wrappers refuse what the library cannot see: types, shapes, devices."""
    import torch

    import miinfer_amd as m
    planes = [torch.zeros(2 * 8 * 64 * 128, dtype=torch.int8) for _ in range(2)]
    scales = [torch.zeros(2 * 8 * 64 * 4, dtype=torch.int16) for _ in range(2)]
    table = torch.zeros((1, 2), dtype=torch.int32)
    cache = m.KvCache.from_planes(8, 128, *planes, *scales, page_tokens=64, block_table=table)
    assert cache.num_pages == 2 and cache.capacity == 128 and not cache.k_f16
    half = [t.to(torch.float16) for t in planes]
    assert m.KvCache.from_planes(8, 128, *half, page_tokens=128).quant_mode == 0
    for bad in (dict(page_tokens=100), dict(page_tokens=64), dict(page_tokens=256, block_table=table)):
        with pytest.raises(ValueError):
            m.KvCache.from_planes(8, 128, *planes, *scales, **bad)
    with pytest.raises(ValueError):
        m.KvCache.from_planes(8, 128, *planes, page_tokens=64, block_table=table)
    with pytest.raises(ValueError):
        m.KvCache.from_planes(8, 128, *half, *scales, page_tokens=64, block_table=table)
    q = torch.zeros((1, 32, 128), dtype=torch.float16)
    lens = torch.ones(1, dtype=torch.int32)
    w = torch.zeros((1, 8, 128))
    with pytest.raises(ValueError, match="GPU"):
        m.window_attention(cache, q, window=8, lengths=lens)
    for bad in (dict(window=-1), dict(window=8, sinks=-1), dict(window=8, max_context=0), dict(window=8, gate=q),
                dict(window=8, out=torch.zeros((1, 32, 64)))):
        with pytest.raises(ValueError):
            m.window_attention(cache, q, lengths=lens, **bad)
    with pytest.raises(ValueError):
        m.window_attention(cache, q.expand(2, 32, 128), window=8, lengths=torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        m.window_attention(cache, q.double(), window=8, lengths=lens)
    with pytest.raises(ValueError):
        m.window_attention(cache, q, window=8, lengths=lens.long())
    for weights in (w.half(), w[:, :4], w[:, :, :100], torch.zeros((1, 8, 256))[:, :, ::2]):
        with pytest.raises(ValueError):
            m.scored_attention(cache, q, weights, lengths=lens)
    with pytest.raises(ValueError):
        m.evict(cache, w, lens, budget=10, sinks=6, recent=5)
    for bad in (dict(budget=0), dict(budget=16, kept=torch.zeros((1, 8, 15), dtype=torch.int32)), dict(budget=16, sinks=-1),
                dict(budget=100, dst_table=torch.zeros((1, 1), dtype=torch.int32)), dict(budget=16, weights_out=w[:, :, :8]),
                dict(budget=16, new_lengths=torch.zeros(1))):
        with pytest.raises(ValueError):
            m.evict(cache, w, lens, **bad)


def _chunk(lib, v, **over):
    a = dict(q=P, qt=2, heads=32, scale=F, batch=3, total=100, off=P, lengths=P, most_tokens=64, most=4096, window=128, sinks=4,
             out=P, ot=2, ws=P, bytes=1 << 40)
    a.update(over)
    return lib.miikv_chunk_attn(None if v is None else ctypes.byref(v), a["q"], a["qt"], a["heads"], a["scale"], a["batch"],
                                a["total"], a["off"], a["lengths"], a["most_tokens"], a["most"], a["window"], a["sinks"],
                                a["out"], a["ot"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("over,status", [
    ({"q": None}, 1), ({"out": None}, 1), ({"off": None}, 1), ({"lengths": None}, 1), ({"qt": 3}, 1), ({"ot": 3}, 1),
    ({"heads": 30}, 1), ({"heads": 0}, 1), ({"scale": ctypes.c_float(float("inf"))}, 1), ({"batch": 0}, 1), ({"total": 0}, 1),
    ({"most_tokens": 0}, 1), ({"most_tokens": 101}, 1), ({"total": 9000, "most_tokens": 5000}, 1), ({"most": 0}, 1),
    ({"most": 4097}, 1), ({"ws": None}, 3), ({"bytes": 256}, 3), ({"q": ctypes.c_void_p(0x10008)}, 1),
    ({"out": ctypes.c_void_p(0x10004)}, 1), ({"ws": ctypes.c_void_p(0x10008)}, 1),
    ({"batch": 70000}, 2), ({"batch": 60000}, 2), ({"total": 0x7fffffff}, 2),
])
def test_chunk_refuses(over, status):
    L = _lib()
    assert _chunk(L.lib(), _paged(), **over) == status
    assert _chunk(L.lib(), None) == L.MIIKV_EINVAL
    assert _chunk(L.lib(), _view(), batch=2) == L.MIIKV_EINVAL  # a contiguous cache holds one sequence


def test_chunk_workspace_sizes():
    L = _lib()
    lib = L.lib()
    v = _paged()
    r = ctypes.byref(v)
    need = lib.miikv_chunk_workspace_bytes(r, 32, 3, 100, 64, 4096, 128, 4)
    assert need > 0 and _chunk(lib, v, bytes=need - 1) == L.MIIKV_EWORKSPACE
    assert lib.miikv_chunk_workspace_bytes(r, 32, 3, 100, 64, 4096, 0xffffffff, 0xffffffff) == \
        lib.miikv_chunk_workspace_bytes(r, 32, 3, 100, 64, 4096, 0, 0)
    for bad in ((30, 3, 100, 64, 4096), (32, 0, 100, 64, 4096), (32, 3, 0, 1, 4096), (32, 3, 100, 101, 4096), (32, 3, 100, 64, 4097)):
        assert lib.miikv_chunk_workspace_bytes(r, *bad, 0, 0) == 0


def test_chunk_python_refusals():
    import torch

    import miinfer_amd as m
    planes = [torch.zeros(2 * 8 * 64 * 128, dtype=torch.float16) for _ in range(2)]
    cache = m.KvCache.from_planes(8, 128, *planes, page_tokens=64, block_table=torch.zeros((1, 2), dtype=torch.int32))
    q = torch.zeros((4, 32, 128), dtype=torch.bfloat16)
    off, lens = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([9], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        m.chunk_attention(cache, q, off, lens)
    for args, kw in (((q.double(), off, lens), {}), ((q[:, :, ::2], off, lens), {}), ((q, off[:1], lens), {}),
                     ((q, off.long(), lens), {}), ((q, off, lens), {"out": q.int()}), ((q, off, lens), {"out": q[:3]}),
                     ((q, off, lens), {"window": -1}), ((q, off, lens), {"max_tokens": 0}),
                     ((q, torch.tensor([0, 1, 4], dtype=torch.int32), torch.ones(2, dtype=torch.int32)), {})):
        with pytest.raises(ValueError):
            m.chunk_attention(cache, *args, **kw)
