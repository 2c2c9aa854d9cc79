// What the operators over part of a cache share: which keys a token sees, and the checks
// of their arguments.
#pragma once

#include "miikv_common.hpp"

#include <cmath>

namespace miikv {

int validate_view(const miikv_view* v);
uint64_t view_seq_capacity(const miikv_view* v);

constexpr float kLog2eF = 1.4426950408889634f;

// The 32-key steps of a context of L keys that hold a key which one of its last `tokens`
// tokens sees: steps [0, head) and [first, end).  A token at position p sees keys j <= p
// with j > p - window (window == 0: all of them) or j < sinks.
struct Visible {
    uint32_t head, first, end;
    uint32_t lo;  // the first key inside the window of the earliest of the tokens
    __host__ __device__ __forceinline__ uint32_t steps() const { return head + (end - first); }
    // The i-th of them.
    __host__ __device__ __forceinline__ uint32_t step(uint32_t i) const { return i < head ? i : first + (i - head); }
};
__host__ __device__ __forceinline__ Visible visible_steps(uint32_t L, uint32_t tokens, uint32_t window, uint32_t sinks) {
    Visible v;
    const uint32_t at = L > tokens ? L - tokens : 0u;  // the earliest token's position
    v.lo = window != 0 && at + 1 > window ? at + 1 - window : 0u;
    v.end = (L + kChunk - 1) / kChunk;
    v.first = v.lo / kChunk;
    const uint32_t s = sinks / kChunk + (sinks % kChunk != 0 ? 1u : 0u);
    v.head = s < v.first ? s : v.first;
    return v;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ uint32_t sum_to_lane(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, true);  // row_bcast:15, to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, true);  // row_bcast:31, to rows 2 and 3
    return x;
}

// The most steps that a context of at most max_context keys can have.
inline uint32_t most_visible_steps(uint32_t max_context, uint32_t tokens, uint32_t window, uint32_t sinks) {
    const uint64_t all = (static_cast<uint64_t>(max_context) + kChunk - 1) / kChunk;
    if (window == 0) return static_cast<uint32_t>(all);
    // the window of `tokens` tokens touches one step more than it fills
    const uint64_t near = (static_cast<uint64_t>(window) + tokens - 1 + kChunk - 1) / kChunk + 1;
    const uint64_t head = (static_cast<uint64_t>(sinks) + kChunk - 1) / kChunk;
    const uint64_t n = near + head;
    return static_cast<uint32_t>(n < all ? n : all);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace miikv
