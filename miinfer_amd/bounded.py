"""Attention over part of a cache, and caches that are made smaller.

``chunk_attention`` is attention of a ragged batch of chunks of new tokens, over the whole
cache or a sliding window and the first tokens that stay visible, ``window_attention`` its
form for single tokens, ``scored_attention`` decode attention that adds up the weight every key
gets, ``evict`` keeps the keys with the largest weights and moves their rows together.
Every call goes through libmiikv; there is no fallback path.  The reference has no
counterpart: its attention layers keep and see the whole context.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _lib
from ._lib import call, lib
from .kv import KvCache, _on_stream, _ptr

_INDEX = (torch.int32, torch.uint32)


def _on_device(dev: torch.device):
    """The cache's device current for the launch, where it is not already."""
    if dev.type != "cuda":
        raise ValueError("the cache must live on a GPU")
    if dev.index is None or dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _queue(dev: torch.device, stream) -> ctypes.c_void_p:
    # (the device is named: current_stream() would look for it first, about 0.5 us of a call)
    return ctypes.c_void_p((torch.cuda.current_stream(dev) if stream is None else stream).cuda_stream)


def _check(cache: KvCache, stream, **tensors) -> None:
    """Every tensor on the cache's device, contiguous; the stream on it too."""
    dev = cache.k_codes.device
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != dev:
            raise ValueError(f"{name} must live on the cache's device")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if stream is not None and stream.device != dev:
        raise ValueError("stream must be one of the cache's device")


def _u32_arg(name: str, x: int, least: int = 0) -> int:
    if not least <= x <= 0x7FFFFFFF:
        raise ValueError(f"{name} out of range")
    return x


def _part_shape(cache: KvCache, q: torch.Tensor):
    if q.dim() not in (3, 4) or q.shape[-1] != cache.head_dim or q.dtype not in (torch.float16, torch.float32):
        raise ValueError("q must be fp16/fp32 [batch, q_heads, head_dim] or [batch, tokens, q_heads, head_dim]")
    return q.shape[0], q.shape[1] if q.dim() == 4 else 1, q.shape[-2]


def _check_batch(cache: KvCache, batch: int) -> None:
    if cache.paged and batch > cache.block_table.shape[0]:
        raise ValueError("batch exceeds the block-table rows")


def _check_part(cache, q, lengths, decode_state, gate, out, gated_out, stream, **more):
    batch, tokens, q_heads = _part_shape(cache, q)
    _check(cache, stream, q=q, lengths=lengths, decode_state=decode_state, gate=gate, out=out, gated_out=gated_out, **more)
    _check_batch(cache, batch)
    if lengths is not None and (lengths.numel() < batch or lengths.dtype not in _INDEX):
        raise ValueError("lengths must be int32 with one entry per sequence")
    if decode_state is not None and decode_state.numel() * decode_state.element_size() < 64:
        raise ValueError("decode_state must be a 64-byte device buffer")
    for t in (gate, out, gated_out):
        if t is not None and (t.shape != q.shape or t.dtype != torch.float32):
            raise ValueError("gate/out/gated_out must be fp32, of q's shape")
    return batch, tokens, q_heads


def _outputs(q, gate, out, gated_out):
    if out is None and gate is None:
        out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    if gate is not None and gated_out is None:
        gated_out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    return out, gated_out


def _workspace(need: int, q: torch.Tensor) -> torch.Tensor:
    if need == 0:
        raise ValueError("the sizes are not ones that this call serves")
    return torch.empty(need, dtype=torch.uint8, device=q.device)


_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def chunk_workspace_bytes(cache: KvCache, q_heads: int, batch: int, total_tokens: int, max_tokens: int, max_context: int,
                          window: int = 0, sinks: int = 0) -> int:
    return int(lib().miikv_chunk_workspace_bytes(cache.view, q_heads, batch, total_tokens, max_tokens, max_context, window, sinks))


def chunk_attention(cache: KvCache, q: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor,
                    scale: float | None = None, *, max_tokens: int | None = None, max_context: int | None = None,
                    window: int = 0, sinks: int = 0, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal attention of a ragged batch of chunks of new tokens, whose rows the cache holds:
    prompts' chunks, chat turns, drafted tokens and single steps in one call.

    q: [total_tokens, q_heads, head_dim], fp16, bf16 or fp32; sequence b's tokens are rows
    offsets[b] .. offsets[b + 1] - 1 (device int32 [batch + 1]) and end its context of
    lengths[b] keys (device int32 [batch]).  With `window` the token at position p sees the
    keys j <= p with j > p - window or j < sinks.  max_tokens and max_context bound a chunk and
    a context (by default total_tokens and the cache's capacity; nearer bounds make smaller
    workspaces).  Returns `out` ([total_tokens, q_heads, head_dim], fp16, bf16 or fp32; by
    default of q's type); rows that belong to no chunk stay as they were."""
    if q.dim() != 3 or q.shape[-1] != cache.head_dim or q.dtype not in _DTYPES:
        raise ValueError("q must be fp16/bf16/fp32 [total_tokens, q_heads, head_dim]")
    total, q_heads = q.shape[0], q.shape[1]
    batch = lengths.numel()
    if lengths.dtype not in _INDEX or offsets.dtype not in _INDEX or offsets.numel() != batch + 1:
        raise ValueError("offsets and lengths must be int32 [batch + 1] and [batch]")
    if out is not None and (out.shape != q.shape or out.dtype not in _DTYPES):
        raise ValueError("out must be fp16/bf16/fp32, of q's shape")
    _check(cache, stream, q=q, offsets=offsets, lengths=lengths, out=out, workspace=workspace)
    _check_batch(cache, batch)
    if max_context is None:
        max_context = cache.capacity
    if max_tokens is None:
        max_tokens = min(total, max_context)
    _u32_arg("max_tokens", max_tokens, 1)
    _u32_arg("max_context", max_context, 1)
    _u32_arg("window", window)
    _u32_arg("sinks", sinks)
    dev = cache.k_codes.device
    with _on_device(dev):
        if workspace is None or out is None:
            with _on_stream(stream):
                if workspace is None:
                    workspace = _workspace(chunk_workspace_bytes(cache, q_heads, batch, total, max_tokens, max_context, window,
                                                                 sinks), q)
                if out is None:
                    out = torch.empty_like(q)
        call("miikv_chunk_attn", cache.view, q.data_ptr(), _DTYPES[q.dtype], q_heads,
             1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale), batch, total, offsets.data_ptr(),
             lengths.data_ptr(), max_tokens, max_context, window, sinks, out.data_ptr(), _DTYPES[out.dtype],
             workspace.data_ptr(), workspace.numel() * workspace.element_size(), _queue(dev, stream))
    return out


def window_workspace_bytes(cache: KvCache, q_heads: int, batch: int, tokens: int, max_context: int, window: int,
                           sinks: int = 0) -> int:
    return int(lib().miikv_window_workspace_bytes(cache.view, q_heads, batch, tokens, max_context, window, sinks))


def window_attention(cache: KvCache, q: torch.Tensor, scale: float | None = None, *, window: int, sinks: int = 0,
                     lengths: torch.Tensor | None = None, decode_state: torch.Tensor | None = None,
                     max_context: int | None = None, gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     gated_out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None):
    """Decode attention with a sliding window: the token at position p sees the keys j <= p
    with j > p - window (window 0: all of them) or j < sinks.

    q: [batch, q_heads, head_dim], or [batch, tokens, q_heads, head_dim] for the last `tokens`
    tokens of every sequence (their rows already appended), fp16 or fp32.  Context lengths,
    the new tokens included, come from `lengths` (device [batch]) or `decode_state`
    (position + 1).  `workspace`: a uint8 tensor of window_workspace_bytes() (allocated when
    not given); calls that may overlap need their own.  Returns (out, gated_out), fp32 of q's
    shape."""
    batch, tokens, q_heads = _check_part(cache, q, lengths, decode_state, gate, out, gated_out, stream, workspace=workspace)
    if max_context is None:
        max_context = cache.capacity
    _u32_arg("window", window)
    _u32_arg("sinks", sinks)
    _u32_arg("max_context", max_context, 1)
    dev = cache.k_codes.device
    with _on_device(dev):
        if workspace is None or out is None or (gate is not None and gated_out is None):
            with _on_stream(stream):
                if workspace is None:
                    workspace = _workspace(window_workspace_bytes(cache, q_heads, batch, tokens, max_context, window, sinks), q)
                out, gated_out = _outputs(q, gate, out, gated_out)
        call("miikv_decode_attn_window", cache.view, q.data_ptr(), 0 if q.dtype == torch.float16 else 1, q_heads,
             1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale), batch, tokens, _ptr(lengths),
             _ptr(decode_state), max_context, window, sinks, _ptr(out), _ptr(gate), _ptr(gated_out),
             workspace.data_ptr(), workspace.numel() * workspace.element_size(), _queue(dev, stream))
    return out, gated_out


def scored_workspace_bytes(cache: KvCache, q_heads: int, batch: int, tokens: int, max_context: int) -> int:
    return int(lib().miikv_scored_workspace_bytes(cache.view, q_heads, batch, tokens, max_context))


def scored_attention(cache: KvCache, q: torch.Tensor, key_weights: torch.Tensor, scale: float | None = None, *,
                     lengths: torch.Tensor | None = None, decode_state: torch.Tensor | None = None,
                     max_context: int | None = None, gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     gated_out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None):
    """Decode attention over the whole context that adds every key's probabilities, summed
    over the call's tokens and the query heads of a kv head, to `key_weights` (fp32 [batch,
    kv_heads, n], n >= max_context; zeros for keys not seen yet).  The last tokens of a
    prompt (q with a token axis) give the weights a first eviction goes by.  Other arguments
    as window_attention.  Returns (out, gated_out)."""
    batch, tokens, q_heads = _check_part(cache, q, lengths, decode_state, gate, out, gated_out, stream, workspace=workspace,
                                         key_weights=key_weights)
    if max_context is None:
        max_context = cache.capacity
    _u32_arg("max_context", max_context, 1)
    _check_weights("key_weights", key_weights, batch, cache.kv_heads, max_context)
    dev = cache.k_codes.device
    with _on_device(dev):
        if workspace is None or out is None or (gate is not None and gated_out is None):
            with _on_stream(stream):
                if workspace is None:
                    workspace = _workspace(scored_workspace_bytes(cache, q_heads, batch, tokens, max_context), q)
                out, gated_out = _outputs(q, gate, out, gated_out)
        call("miikv_decode_attn_scored", cache.view, q.data_ptr(), 0 if q.dtype == torch.float16 else 1, q_heads,
             1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale), batch, tokens, _ptr(lengths),
             _ptr(decode_state), max_context, key_weights.data_ptr(), key_weights.shape[2], _ptr(out), _ptr(gate),
             _ptr(gated_out), workspace.data_ptr(), workspace.numel() * workspace.element_size(), _queue(dev, stream))
    return out, gated_out


def _check_weights(name, w, batch, kv_heads, least):
    if w.dtype != torch.float32 or w.dim() != 3 or w.shape[0] < batch or w.shape[1] != kv_heads or w.shape[2] < least:
        raise ValueError(f"{name} must be fp32 [batch, kv_heads, >= {least}]")


def evict(cache: KvCache, key_weights: torch.Tensor, lengths: torch.Tensor, *, budget: int, sinks: int = 0, recent: int = 0,
          max_context: int | None = None, dst_table: torch.Tensor | None = None, kept: torch.Tensor | None = None,
          new_lengths: torch.Tensor | None = None, weights_out: torch.Tensor | None = None, stream=None):
    """Cut every sequence longer than `budget` down to it: per kv head the first `sinks` keys
    stay, the last `recent`, and of those between the ones with the largest `key_weights`
    ([batch, kv_heads, n], n >= max_context; of equal ones the first).  Their rows move, in order, to
    positions 0, 1, ...: within the sequence's own pages, which nothing else may share then
    (``PagePool.truncate`` gives the free ones back), or to the pages of `dst_table` (int32
    [batch, pages], pages that the batch does not use; ``cache.set_block_table`` with it
    afterwards).  `weights_out` (None: not kept) receives the kept keys' weights and may be
    `key_weights`; `new_lengths` may be `lengths`.

    A kept key keeps the rotation of its old position, so rows appended later have to come
    rotated by theirs.  Returns (kept, new_lengths): the positions that stayed, int32 [batch,
    kv_heads, budget], -1 past the new length, and min(length, budget)."""
    dev = cache.k_codes.device
    batch = key_weights.shape[0] if key_weights.dim() == 3 else 0
    if lengths.dtype not in _INDEX or lengths.dim() != 1 or lengths.shape[0] != batch:
        raise ValueError("lengths must be int32 [batch], with key_weights [batch, kv_heads, n]")
    if max_context is None:
        max_context = min(cache.capacity, key_weights.shape[2])
    _u32_arg("max_context", max_context, 1)
    _u32_arg("budget", budget, 1)
    _u32_arg("sinks", sinks)
    _u32_arg("recent", recent)
    if sinks + recent > budget:
        raise ValueError("sinks + recent exceed the budget")
    _check_weights("key_weights", key_weights, batch, cache.kv_heads, max_context)
    _check_batch(cache, batch)
    _check(cache, stream, key_weights=key_weights, lengths=lengths, dst_table=dst_table, kept=kept, new_lengths=new_lengths,
           weights_out=weights_out)
    most = min(budget, max_context)
    if weights_out is not None:
        _check_weights("weights_out", weights_out, batch, cache.kv_heads, most)
        if weights_out.shape[0] != batch:
            raise ValueError("weights_out must have a row per sequence")
    if kept is not None and (kept.dtype != torch.int32 or tuple(kept.shape) != (batch, cache.kv_heads, budget)):
        raise ValueError("kept must be int32 [batch, kv_heads, budget]")
    if new_lengths is not None and (new_lengths.dtype not in _INDEX or tuple(new_lengths.shape) != (batch,)):
        raise ValueError("new_lengths must be int32 [batch]")
    if dst_table is not None and (not cache.paged or dst_table.dtype != torch.int32 or dst_table.dim() != 2 or
                                  dst_table.shape[0] < batch or dst_table.shape[1] * cache.page_tokens < most):
        raise ValueError("dst_table must be int32 [batch, pages for the budget], of a paged cache")
    with _on_device(dev):
        if kept is None or new_lengths is None:
            with _on_stream(stream):
                if kept is None:
                    kept = torch.empty((batch, cache.kv_heads, budget), dtype=torch.int32, device=dev)
                if new_lengths is None:
                    new_lengths = torch.empty((batch,), dtype=torch.int32, device=dev)
        call("miikv_evict", cache.view, key_weights.data_ptr(), key_weights.shape[2], batch, lengths.data_ptr(), max_context,
             sinks, recent, budget, _ptr(dst_table), 0 if dst_table is None else dst_table.shape[1], kept.data_ptr(),
             new_lengths.data_ptr(), _ptr(weights_out), 0 if weights_out is None else weights_out.shape[2], _queue(dev, stream))
    return kept, new_lengths
