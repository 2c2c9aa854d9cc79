"""miinfer_amd — MI355X-native quantized KV-cache path (q8_0 append, split-K GQA
decode attention, suffix attention, attention over part of a cache and eviction,
prefix-state reuse) behind the C ABI in include/miikv.h.  This package is the host-side mirror of the reference's
KV-cache / attention call surface; all compute runs in libmiikv.so (HIP,
gfx950) and fails loudly when that library is missing.
"""
from ._lib import MiikvError, lib  # noqa: F401
from .bounded import (  # noqa: F401
    chunk_attention,
    chunk_workspace_bytes,
    evict,
    scored_attention,
    scored_workspace_bytes,
    window_attention,
    window_workspace_bytes,
)
from .kv import (  # noqa: F401
    DecodeWorkspace,
    advance_decode_state,
    KvCache,
    clone_state,
    copy_segments,
    decode_attention,
    make_decode_state,
    make_prefill_state,
    suffix_attention,
    suffix_workspace_bytes,
)

__all__ = [
    "MiikvError", "lib", "advance_decode_state", "KvCache", "DecodeWorkspace", "decode_attention", "clone_state",
    "copy_segments", "make_decode_state", "make_prefill_state", "suffix_attention", "suffix_workspace_bytes",
    "chunk_attention", "chunk_workspace_bytes", "evict", "scored_attention", "scored_workspace_bytes", "window_attention",
    "window_workspace_bytes",
]
