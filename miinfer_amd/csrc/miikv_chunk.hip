// Attention of a ragged batch of chunks of new tokens over a paged cache, causal, with an
// optional sliding window and the first tokens (gfx950, wave64, MFMA).
//
// Token t of sequence b's n_b new ones stands at p = L_b - n_b + t and sees the keys j <= p
// with j > p - window (window == 0: all) or j < sinks:
//   s_j = scale * q . k_j,  o = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m}.
//
// Work.  The rows of a (sequence, kv head) are its (token, query head of the group) pairs;
// kRows of them are an item, whose tokens together see a run of 32-key steps (and the steps
// of the first tokens).  Items differ in length (short chunks, causality, windows), so the
// items of all kv heads are laid on one axis, some units per item and per step, and the
// axis is cut into equal parts, one per workgroup of the one resident round: every CU has the
// same work whatever the lengths are.  An item that lies in one part is written straight
// to the output; the parts of one that is cut leave records, which the second launch merges.
//
// A workgroup's eight waves own 32 rows each and share the key tiles in LDS.  Per step
//   S^T[key][row] = K (32 keys x D) Q^T,  O^T[dim][row] += V^T (dims x 32 keys) P^T
// with v_mfma_f32_32x32x16_f16: S's result layout (a lane holds 16 keys of one row) is the B
// operand of the second product as it stands.  Steps come into a ring in LDS as the cache holds
// them, by copies that pass no registers (at D = 256 O^T and the query take 192 of the 256);
// the next step's codes are turned into fp16 rows (code * scale, rounded once) in the other tile
// buffer before this step's tile is multiplied.
//
// With many rows per sequence expand_kernel makes the fp16 tiles first, and the ring holds those.
//
// Bound: the matrix unit where rows are many (two 512-token chunks over 8704 keys, head_dim 256: this kernel
// 196 us, 1.08 PFLOP/s, 61% of its cycles in MFMAs; prompts at head_dim 128: 152 us, 0.85 PFLOP/s, with half the
// MFMAs for the same exponentials); where they are few, the conversions and what an item costs before its
// first step and after its last (12 sequences of 3 to 39 tokens: 41 us).
//
// Precision: query, code * scale and probabilities are fp16, the matrix unit's operands, sums and
// statistics fp32; the records' normalised outputs are fp16, half the bytes that the merge reads. Outputs are
// 4e-4 of their norm off in all.
#include "miikv_part.hpp"

#include <algorithm>
#include <type_traits>

namespace miikv {
namespace {

constexpr uint32_t kChunkWaves = 8;
constexpr uint32_t kChunkThreads = 64 * kChunkWaves;
constexpr uint32_t kRows = 32 * kChunkWaves;  // rows of an item
// Units of the axis: of a step, of one whose codes are converted by waves without rows, and an item's fixed
// cost (12 chunks of 40 and of 20 tokens over 9000 more keys, head_dim 256: 122 and 80 us more; prompts
// with 4 and 8 steps as an item's cost: 180 and 165 us).
constexpr uint32_t kStepCost = 3, kHelpedCost = 2;
constexpr uint32_t kItemCost = 8 * kStepCost;
constexpr uint32_t kMinUnits = 12 * kStepCost;  // per workgroup, at least
constexpr uint32_t kMaxParts = 256;           // one workgroup per CU
// Keys are expanded to fp16 tiles first from this many items per (sequence, kv head) on, of a call's
// average: an expansion costs about the read and the write of the tiles, and saves its items' conversions.
// (Four sequences of 8192 keys, us without and with: head_dim 128, 4 items 170 and 173, 8 items 316 and
// 292; head_dim 256, 4 items 173 and 181, 8 items 284 and 275; fp16 planes 168 and 183, 312 and 300,
// 199 and 189, 311 and 283.)
constexpr uint32_t kTileItems = 6;
constexpr uint64_t kMaxTileBytes = 1ull << 30;
constexpr uint32_t kStageBytes = 4096;        // of a wave, for rows on their way to and from memory
constexpr float kSlack = 8.0f;                // the maximum may grow by this (log2) before sums are rescaled

struct ChunkItem {
    uint32_t b;      // sequence
    uint32_t rows0;  // its first row
    uint32_t start;  // units of one kv head before it
    uint32_t steps;
    uint32_t rows;   // of it
    uint32_t tok0;   // row0's token, in q
    uint32_t head0;  // and query head of the group
    uint32_t last;   // axis places from its first turn to its last one
};

struct ChunkArgs {
    Geo g;
    const void* q;
    uint32_t q_dtype;
    uint32_t q_heads;
    uint32_t group;  // query heads per kv head
    float scale_log2;  // above 0: a negative scale negates the query
    uint32_t negate;
    uint32_t batch;
    uint32_t total_tokens;
    uint32_t max_tokens;
    uint32_t max_context;
    uint32_t window;
    uint32_t sinks;
    const uint32_t* offsets;
    const uint32_t* lengths;
    void* out;
    uint32_t out_dtype;
    uint32_t most_items;  // of one kv head
    uint32_t parts;
    uint32_t page_steps;  // steps per page, and for small ones 2^32 / page_steps, rounded up
    uint32_t page_magic;
    // workspace
    uint32_t* head;      // [0] items of one kv head, [1] units of one kv head, [2] units per part
    ChunkItem* items;    // [most_items]
    uint32_t most_steps; // tiles of a (sequence, kv head)
    const half8* tiles;  // [batch][kv_heads][most_steps]
    _Float16* rec_o;     // [2 * parts][kRows][D]: outputs over the part's keys
    float2* rec_ml;      // [2 * parts][kRows]: maximum (log2 units) and sum
};

// Sequence b's chunk: its first row in q, its tokens and its context, all within the bounds
// that the host knows (so that wrong device data reads and writes no further).
struct Chunk {
    uint32_t q0, tokens, length;
};
__device__ __forceinline__ Chunk chunk_of(const ChunkArgs& a, uint32_t b) {
    Chunk c;
    c.q0 = min(a.offsets[b], a.total_tokens);
    const uint32_t end = min(a.offsets[b + 1], a.total_tokens);
    c.tokens = end > c.q0 ? min(end - c.q0, a.max_tokens) : 0u;
    c.length = min(a.lengths[b], a.max_context);
    return c;
}

// chunk_of a wave-uniform b, in scalar registers.
__device__ __forceinline__ Chunk chunk_of_uniform(const ChunkArgs& a, uint32_t b) {
    Chunk c;
    c.q0 = min(scalar_load(a.offsets + b), a.total_tokens);
    const uint32_t end = min(scalar_load(a.offsets + b + 1), a.total_tokens);
    c.tokens = end > c.q0 ? min(end - c.q0, a.max_tokens) : 0u;
    c.length = min(scalar_load(a.lengths + b), a.max_context);
    return c;
}
// Workgroup barrier after this wave's LDS reads have returned and its writes are done;
// copies to LDS stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ const char* uniform_ptr(const char* p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const char*>(static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 | uniform(static_cast<uint32_t>(x)));
}

// What the rows rows0 .. of a chunk see together: the context of the last of them, their
// tokens and the steps.
struct Span {
    uint32_t rows;   // of the item
    uint32_t past;   // keys up to the last token's own
    uint32_t tokens;
    Visible vis;
};
__device__ __forceinline__ Span span_of(const ChunkArgs& a, const Chunk& c, uint32_t rows0) {
    Span s;
    s.rows = min(kRows, c.tokens * a.group - rows0);
    const uint32_t t0 = rows0 / a.group, t1 = (rows0 + s.rows - 1) / a.group;
    s.past = c.length + t1 + 1 > c.tokens ? c.length + t1 + 1 - c.tokens : 0u;
    s.tokens = t1 - t0 + 1;
    s.vis = visible_steps(s.past, s.tokens, a.window, a.sinks);
    return s;
}

// Inclusive sums over the workgroup's threads; `total` is the last one's.
__device__ __forceinline__ uint32_t scan_threads(uint32_t x, uint32_t* s_wave, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t incl = sum_to_lane(x);
    __syncthreads();
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    total = 0;
    uint32_t before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kChunkWaves; ++w) {
        if (w < wave) before += s_wave[w];
        total += s_wave[w];
    }
    return before + incl;
}

__device__ __forceinline__ float16v mfma_32x32x16(half8 a, half8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
// 16 bytes per lane from `base` + `off` to LDS at `lds` + 16 * lane (`base` and `lds` wave-uniform;
// counted by the caller, as copy_to_lds).
__device__ __forceinline__ void copy_to_lds_from(const char* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(uniform_ptr(base))
                 : "memory", "m0");
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// `use`(zero of the type that `dtype` names): one branch per loop, not per element.
template <typename F>
__device__ __forceinline__ void with_type(uint32_t dtype, F use) {
    if (dtype == MIIKV_DTYPE_BF16) use(__bf16{});
    else if (dtype == MIIKV_DTYPE_F16) use(_Float16{});
    else use(float{});
}
// Four values to element `at` of an array of T, rounded to nearest even.
template <typename T>
__device__ __forceinline__ void store4(void* out, size_t at, float4 x) {
    typedef T vec __attribute__((ext_vector_type(4)));
    *reinterpret_cast<vec*>(static_cast<T*>(out) + at) =
        vec{static_cast<T>(x.x), static_cast<T>(x.y), static_cast<T>(x.z), static_cast<T>(x.w)};
}
// Eight query values, rounded to fp16.
template <typename T>
__device__ __forceinline__ half8 load_query(const void* q, size_t at) {
    typedef T vec __attribute__((ext_vector_type(8)));
    const vec x = *reinterpret_cast<const vec*>(static_cast<const T*>(q) + at);
    if constexpr (std::is_same<T, _Float16>::value) {
        return x;
    } else {
        half8 r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = static_cast<_Float16>(static_cast<float>(x[i]));
        return r;
    }
}

// Block scales of a tile: 128 * 511.75 = 65504 is the largest that leaves every code finite.
// (Larger ones stand for blocks within 0.8% of fp16's maximum.)
__device__ __forceinline__ half2v tile_scales(half2v s) {
    return __builtin_elementwise_min(s, half2v{static_cast<_Float16>(511.75f), static_cast<_Float16>(511.75f)});
}

// LDS of chunk_kernel: two fp16 tiles of a step, K units [D / 8][32 keys] and V units [4][D + 4]
// of 8 values (V's rows of units are 64 bytes longer than they need be: neighbouring threads
// write units of two rows), and a ring of steps as the cache holds them: K codes, V codes, K
// scales, V scales.
template <uint32_t D, bool KF16, bool VF16>
struct ChunkLds {
    static constexpr uint32_t k_units = D / 8 * kChunk;
    static constexpr uint32_t v_row = D + 4;
    static constexpr uint32_t units = k_units + 4 * v_row;
    static constexpr uint32_t k_bytes = kChunk * D * (KF16 ? 2 : 1), v_bytes = kChunk * D * (VF16 ? 2 : 1);
    static constexpr uint32_t scale_bytes = kChunk * (D / 32) * 2;
    static constexpr uint32_t raw = k_bytes + v_bytes + 2 * scale_bytes;
    // Steps of the ring, as far as 160 KB go; how many steps ahead of the one being multiplied
    // must have landed (V's scales are put in order a step before its codes are converted); and
    // the copies that each wave issues per step (with scales of one plane only, four waves issue
    // one less, so those modes wait for all copies).
    static constexpr uint32_t bufs = D == 128 || !(KF16 || VF16) ? 4 : (KF16 && VF16 ? 2 : 3);
    static constexpr uint32_t landed = VF16 ? 1 : 2;
    static constexpr uint32_t ops = (k_bytes + v_bytes) / 1024 / kChunkWaves + (KF16 && VF16 ? 0 : 1);
    // Whether the waves of a SIMD take turns at the matrix and the vector unit: where the ring holds
    // four steps.
    static constexpr bool turns = !KF16 && !VF16;
    static constexpr uint32_t vsc_bytes = 2 * 2 * D;  // V's scales of two steps in the order of its units
    static constexpr uint32_t bytes = 2 * units * 16 + bufs * raw + vsc_bytes;
};

// With tiles that expand_kernel has made: a ring of them, K units [D / 8][32 keys] and V units
// [4][D] of 8 values.
template <uint32_t D>
struct TileLds {
    static constexpr uint32_t k_units = D / 8 * kChunk;
    static constexpr uint32_t v_row = D;
    static constexpr uint32_t units = k_units + 4 * v_row;
    static constexpr uint32_t wide = D == 128 ? 2 : 1;  // steps of a turn
    static constexpr uint32_t places = 4;               // turns of the ring
    static constexpr uint32_t step_ops = units * 16 / 1024 / kChunkWaves, ops = wide * step_ops;
    static constexpr uint32_t bytes = places * wide * units * 16;
    static_assert(wide * units * 16 >= kChunkWaves * kStageBytes, "a place holds the waves' stages");
};

// Tile of a step (counted among the steps that any token of the chunk sees, `all`) of (b, h).
__device__ __forceinline__ const half8* tile_at(const ChunkArgs& a, uint32_t b, uint32_t h, const Visible& all, uint32_t step, uint32_t units) {
    const uint32_t i = step < all.head ? step : all.head + (step - all.first);
    return a.tiles + ((static_cast<size_t>(b) * a.g.kv_heads + h) * a.most_steps + i) * units;
}

// One step of (sequence z, kv head y) as an fp16 tile: code * scale, rounded once.  Keys that no
// token of the chunk sees may hold anything: their values become 0.
// Bound: HBM (the codes once, the tiles once: two sequences of 8704 keys, head_dim 256, 109 MB in 23 us).
template <uint32_t D, bool KF16, bool VF16>
__global__ void __launch_bounds__(256) expand_kernel(ChunkArgs a) {
    constexpr uint32_t NB = D / 32, KE = KF16 ? 2 : 1, VE = VF16 ? 2 : 1, kRuns = 2 * D;  // 16 codes each, of K and of V
    using Lds = TileLds<D>;
    const uint32_t b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const Geo& geo = a.g;
    const Chunk c = chunk_of_uniform(a, b);
    if (c.tokens == 0) return;
    const Visible all = visible_steps(c.length, c.tokens, a.window, a.sinks);
    if (blockIdx.x >= all.steps()) return;
    const uint32_t tok0 = all.step(blockIdx.x) * kChunk;
    uint32_t page = 0, tp = tok0;
    if (geo.layout == MIIKV_LAYOUT_PAGED) {
        const uint32_t e = tok0 / geo.page_tokens;
        tp = tok0 - e * geo.page_tokens;
        page = min(static_cast<uint32_t>(scalar_load(geo.table + static_cast<size_t>(b) * geo.table_stride + e)), geo.num_pages - 1);
    }
    const size_t row = (static_cast<size_t>(page) * geo.kv_heads + h) * geo.page_tokens + tp;
    half8* tile = const_cast<half8*>(tile_at(a, b, h, all, tok0 / kChunk, Lds::units));
    const uint4* kc = reinterpret_cast<const uint4*>(geo.k_codes + row * (D * KE));
    const uint4* vc = reinterpret_cast<const uint4*>(geo.v_codes + row * (D * VE));
    uint4 kw[kRuns / 256][KE], vw[kRuns / 256][VE];
    half2v ks[kRuns / 256];
#pragma unroll
    for (uint32_t j = 0; j < kRuns / 256; ++j) {
        const uint32_t idx = j * 256 + tid;
#pragma unroll
        for (uint32_t e = 0; e < KE; ++e) kw[j][e] = kc[idx * KE + e];
#pragma unroll
        for (uint32_t e = 0; e < VE; ++e) vw[j][e] = vc[idx * VE + e];
        if constexpr (!KF16)
            ks[j] = *reinterpret_cast<const half2v*>(geo.k_scales + (row + 16 * (idx / D) + idx % 16) * NB + 2 * (idx / 64 % (D / 64)));
    }
    auto unseen = [&](uint32_t t) { return (t >= c.length) | ((t < all.lo) & (t >= a.sinks)); };
    __shared__ __align__(16) _Float16 s_vsc[D];  // V's scales in the order of its units
    if (!VF16 && tid < D / 2) {
        const uint32_t key = tid / (NB / 2), blk = tid % (NB / 2) * 2;
        half2v w = tile_scales(*reinterpret_cast<const half2v*>(geo.v_scales + row * NB + 2 * tid));
        if (unseen(tok0 + key)) w = half2v{static_cast<_Float16>(0.0f), static_cast<_Float16>(0.0f)};
        _Float16* to = s_vsc + blk * 32 + (key / 4 % 4) * 8 + key / 16 * 4 + key % 4;
        to[0] = w[0];
        to[32] = w[1];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kRuns / 256; ++j) {
        const uint32_t idx = j * 256 + tid;
        {  // key 16 T + m, dims 64 c + 8 g and 64 c + 32 + 8 g
            half8* to = tile + (8 * (idx / 64 % (D / 64)) + idx / 16 % 4) * kChunk + 16 * (idx / D) + idx % 16;
            if constexpr (KF16) {
                to[0] = __builtin_bit_cast(half8, kw[j][0]);
                to[4 * kChunk] = __builtin_bit_cast(half8, kw[j][KE - 1]);
            } else {
                const half2v f = tile_scales(ks[j]);
                to[0] = codes8_to_half8(kw[j][0].x, kw[j][0].y) * f[0];
                to[4 * kChunk] = codes8_to_half8(kw[j][0].z, kw[j][0].w) * f[1];
            }
        }
        {  // dim d, keys of units 2x and 2x + 1
            const uint32_t d = idx / 2, x = idx % 2;
            half8* to = tile + Lds::k_units + 2 * x * Lds::v_row + d;
            half8 v[2];
            if constexpr (VF16) {
                v[0] = __builtin_bit_cast(half8, vw[j][0]);
                v[1] = __builtin_bit_cast(half8, vw[j][VE - 1]);
#pragma unroll
                for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
                    for (uint32_t y = 0; y < 8; ++y)
                        v[u][y] = unseen(tok0 + 16 * (y / 4) + 4 * (2 * x + u) + y % 4) ? static_cast<_Float16>(0.0f) : v[u][y];
            } else {
                const half8* f = reinterpret_cast<const half8*>(s_vsc + d / 32 * 32 + 16 * x);
                v[0] = codes8_to_half8(vw[j][0].x, vw[j][0].y) * f[0];
                v[1] = codes8_to_half8(vw[j][0].z, vw[j][0].w) * f[1];
            }
            to[0] = v[0];
            to[Lds::v_row] = v[1];
        }
    }
}

// TILES: steps come as tiles that expand_kernel has made (KF16 and VF16 are of no account), else
// as the cache holds them.
template <uint32_t D, bool KF16, bool VF16, bool TILES>
__global__ void __launch_bounds__(kChunkThreads) __attribute__((amdgpu_waves_per_eu(2))) chunk_kernel(ChunkArgs a) {
    constexpr uint32_t NB = D / 32;
    constexpr uint32_t NQ = D / 16;  // K-axis chunks of the first product
    constexpr uint32_t KE = KF16 ? 2 : 1, VE = VF16 ? 2 : 1;
    constexpr uint32_t kAhead = D == 128 ? 8 : 4;  // fragments read ahead of their MFMAs
    using Raw = ChunkLds<D, KF16, VF16>;
    using Lds = typename std::conditional<TILES, TileLds<D>, Raw>::type;
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr uint32_t W = TILES ? TileLds<D>::wide : 1;         // steps of a turn
    constexpr uint32_t kPlaces = TILES ? TileLds<D>::places : 2;  // turns whose tiles are held
    half8* const s_tile = reinterpret_cast<half8*>(lds);  // [kPlaces][W]
    uint8_t* const s_raw = lds + 2 * Raw::units * 16;
    _Float16* const s_vsc = reinterpret_cast<_Float16*>(s_raw + Raw::bufs * Raw::raw);  // [2][NB][4][8]
    uint32_t* const s_first = reinterpret_cast<uint32_t*>(lds + Lds::bytes);  // [batch + 1]: items before sequence b
    uint32_t* const s_start = s_first + a.batch + 1;                          // [most_items + 1]: units before item i
    __shared__ uint32_t s_wave[kChunkWaves];

    const uint32_t tid = threadIdx.x, lane = tid & 63, n = lane & 31, hh = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Geo& geo = a.g;

    // ---- the plan, by every workgroup for itself
    auto turn_cost = [](uint32_t rows) { return W * (!TILES && Raw::turns && rows <= kRows / 2 ? kHelpedCost : kStepCost); };
    uint32_t base = 0, total;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kChunkThreads) {
        const uint32_t b = b0 + tid;
        const uint32_t mine = b < a.batch ? (chunk_of(a, b).tokens * a.group + kRows - 1) / kRows : 0u;
        const uint32_t incl = scan_threads(mine, s_wave, total);
        if (b < a.batch) s_first[b] = base + incl - mine;
        base += total;
    }
    const uint32_t items = uniform(min(base, a.most_items));
    if (tid == 0) s_first[a.batch] = base;
    __syncthreads();
    uint32_t units = 0;
    for (uint32_t i0 = 0; i0 < items; i0 += kChunkThreads) {
        const uint32_t i = i0 + tid;
        uint32_t mine = 0;
        ChunkItem it{};
        if (i < items) {
            uint32_t lo = 0, hi = a.batch;  // the last sequence whose items start at or before i
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (s_first[mid] <= i) lo = mid;
                else hi = mid;
            }
            it.b = lo;
            it.rows0 = (i - s_first[lo]) * kRows;
            const Chunk c = chunk_of(a, lo);
            const Span span = span_of(a, c, it.rows0);
            it.steps = span.vis.steps();
            it.rows = span.rows;
            it.tok0 = c.q0 + it.rows0 / a.group;
            it.head0 = it.rows0 % a.group;
            const uint32_t turns = (it.steps + W - 1) / W, cost = turn_cost(span.rows);
            it.last = turns == 0 ? 0u : (turns - 1) * cost;
            mine = kItemCost + turns * cost;
        }
        const uint32_t incl = scan_threads(mine, s_wave, total);
        if (i < items) {
            it.start = units + incl - mine;
            s_start[i] = it.start;
            if (blockIdx.x == 0) a.items[i] = it;
        }
        units += total;
    }
    units = uniform(units);
    const uint32_t axis = units * geo.kv_heads;  // the host has seen that it fits 32 bits
    const uint32_t quota = uniform(max(axis / a.parts + (axis % a.parts != 0 ? 1u : 0u), kMinUnits));
    if (tid == 0) {
        s_start[items] = units;
        if (blockIdx.x == 0) {
            a.head[0] = items;
            a.head[1] = units;
            a.head[2] = quota;
        }
    }
    __syncthreads();
    // Parts that follow each other on the axis read the same keys: they go to one XCD (workgroup
    // w runs on XCD w % 8).
    const uint32_t per = (a.parts + 7) / 8;
    const uint32_t part = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (part >= a.parts) return;
    if (static_cast<uint64_t>(part) * quota >= axis) return;
    const uint32_t begin = part * quota, end = axis - begin < quota ? axis : begin + quota;
    uint32_t at = begin;
    uint32_t h = uniform(at / units);
    uint32_t i = 0, b = 0;  // the item that holds `at`, and its sequence
    for (uint32_t hi = items; hi - i > 1;) {
        const uint32_t mid = (i + hi) / 2;
        if (uniform(s_start[mid]) <= at - h * units) i = mid;
        else hi = mid;
    }
    for (uint32_t hi = a.batch; hi - b > 1;) {
        const uint32_t mid = (b + hi) / 2;
        if (uniform(s_first[mid]) <= i) b = mid;
        else hi = mid;
    }
    uint32_t place = 1;  // of the ring, that no wave reads at an item's end
    for (; at < end; ++i) {
        if (i == items) {  // the next kv head's first
            ++h;
            i = 0;
            b = 0;
        }
        while (uniform(s_first[b + 1]) <= i) ++b;
        const uint32_t start = h * units + uniform(s_start[i]), stop = h * units + uniform(s_start[i + 1]);
        const Chunk c = chunk_of_uniform(a, b);
        const uint32_t rows0 = (i - uniform(s_first[b])) * kRows;
        Span span = span_of(a, c, rows0);
        // (the divisions by the group leave these in vector registers)
        span.rows = uniform(span.rows);
        span.past = uniform(span.past);
        span.vis = {uniform(span.vis.head), uniform(span.vis.first), uniform(span.vis.end), uniform(span.vis.lo)};
        const uint32_t steps = span.vis.steps();
        const uint32_t first = start + kItemCost;  // the axis place of its first turn
        // the turns that start within the part
        const bool full = W * kStepCost == turn_cost(span.rows);
        auto turns_to = [&](uint32_t x) { return full ? (x + W * kStepCost - 1) / (W * kStepCost) : (x + W * kHelpedCost - 1) / (W * kHelpedCost); };
        const uint32_t s0 = uniform(at > first ? turns_to(at - first) * W : 0u);
        const uint32_t s1 = uniform(end > first ? min(turns_to(end - first) * W, steps) : 0u);
        at = stop;
        if (s0 >= s1 && !(steps == 0 && start >= begin)) continue;  // only some of its fixed cost is here

        // ---- this wave's rows
        const uint32_t r = wave * 32 + n;  // of the item
        const uint32_t row = rows0 + min(r, span.rows - 1);
        const uint32_t tok = row / a.group, head = h * a.group + (row - tok * a.group);
        const uint32_t past = c.length + tok + 1 > c.tokens ? c.length + tok + 1 - c.tokens : 0u;
        const uint32_t low = a.window != 0 && past > a.window ? past - a.window : 0u;
        const uint32_t row_index = (c.q0 + tok) * a.q_heads + head;  // of q and out; the host has seen that it fits 31 bits
        const bool wave_live = wave * 32 < span.rows;
        // of the wave's first and last row
        const uint32_t past_a = __builtin_amdgcn_readfirstlane(past), low_a = __builtin_amdgcn_readfirstlane(low);
        const uint32_t past_z = __builtin_amdgcn_readlane(past, 31), low_z = __builtin_amdgcn_readlane(low, 31);

        // The thread's number, at D = 256 made anew at each use: what is derived from it is then not
        // kept in registers through the loop (which has none left there).
        auto here = [&]() __attribute__((always_inline)) {
            uint32_t t = tid;
            if constexpr (D == 256) asm volatile("" : "+v"(t));
            return t;
        };
        // Steps go into the ring one after another, by copies that pass no registers: the waves share
        // the KiB of codes, and each copies an eighth of the scales.  A wave keeps the addresses of
        // its pieces and steps them on; at a page's end (and where the steps of the first tokens end) they
        // are made anew, from 64 entries of the block table held by the lanes.
        constexpr uint32_t kPieces = TILES ? 1 : (Raw::k_bytes + Raw::v_bytes + 1024 * kChunkWaves - 1) / 1024 / kChunkWaves;
        constexpr uint32_t kScalePiece = 2 * Raw::scale_bytes / kChunkWaves;  // of K's, then of V's
        const bool scale_of_k = wave < kChunkWaves / 2;
        const char* src[kPieces];
        const char* src_scale = nullptr;
        uint32_t next = s0, run_left = 0;
        uint32_t tab = 0, tab0 = 0x80000000u;  // (none yet)
        const Visible all = visible_steps(c.length, c.tokens, a.window, a.sinks);  // what any token of the chunk sees
        auto locate = [&]() __attribute__((always_inline)) {
            const uint32_t st = uniform(span.vis.step(next));
            if constexpr (TILES) {
                run_left = next < span.vis.head ? span.vis.head - next : 0x7fffffffu;
                src[0] = uniform_ptr(reinterpret_cast<const char*>(tile_at(a, b, h, all, st, Lds::units)) + wave * 1024);
                return;
            }
            uint32_t page = 0, slot = st;
            run_left = 0x7fffffffu;
            if (geo.layout == MIIKV_LAYOUT_PAGED) {
                const uint32_t e = a.page_magic != 0 ? __umulhi(st, a.page_magic) : uniform(st / a.page_steps);
                if (e - tab0 >= 64u) {
                    tab0 = e;
                    // (waited for here, in asm: the compiler would wait for every copy at each use)
                    const int32_t* from = geo.table + static_cast<size_t>(b) * geo.table_stride + min(e + lane, geo.table_stride - 1);
                    asm volatile("global_load_dword %0, %1, off\n\ts_waitcnt vmcnt(0)" : "=&v"(tab) : "v"(from) : "memory");
                    tab = min(tab, geo.num_pages - 1);
                }
                page = __builtin_amdgcn_readlane(tab, e - tab0);
                slot = st - e * a.page_steps;
                run_left = a.page_steps - slot;
            }
            if (next < span.vis.head) run_left = min(run_left, span.vis.head - next);
            const size_t kv = (static_cast<size_t>(page) * geo.kv_heads + h) * geo.page_tokens + slot * kChunk;
#pragma unroll
            for (uint32_t x = 0; x < kPieces; ++x) {
                const uint32_t at = (wave + x * kChunkWaves) * 1024;
                src[x] = uniform_ptr(at < Raw::k_bytes ? reinterpret_cast<const char*>(geo.k_codes) + kv * (D * KE) + at
                                                       : reinterpret_cast<const char*>(geo.v_codes) + kv * (D * VE) + (at - Raw::k_bytes));
            }
            src_scale = uniform_ptr(scale_of_k ? reinterpret_cast<const char*>(geo.k_scales + kv * NB) + wave * kScalePiece
                                               : reinterpret_cast<const char*>(geo.v_scales + kv * NB) + (wave * kScalePiece - Raw::scale_bytes));
        };
        auto fetch = [&]() __attribute__((always_inline)) {
            if (run_left == 0) locate();
            if constexpr (TILES) {  // of one step
                // (behind the last step of an odd number, that one again: its probabilities are 0)
                const uint32_t to = lds_offset(s_tile) + (next - s0) % (kPlaces * W) * Lds::units * 16 + wave * 1024;
#pragma unroll
                for (uint32_t x = 0; x < TileLds<D>::step_ops; ++x)
                    copy_to_lds_from(src[0] + x * kChunkWaves * 1024, lane * 16, to + x * kChunkWaves * 1024);
                if (next + 1 < s1) {
                    src[0] += Lds::units * 16;
                    --run_left;
                }
                ++next;
                return;
            }
            const uint32_t to = lds_offset(s_raw) + next % Raw::bufs * Raw::raw;
#pragma unroll
            for (uint32_t x = 0; x < kPieces; ++x) {
                const uint32_t at = (wave + x * kChunkWaves) * 1024;
                if (at < Raw::k_bytes + Raw::v_bytes)  // (12 KiB in the mixed modes at D = 128)
                    copy_to_lds_from(src[x], lane * 16, to + at);
                src[x] += at < Raw::k_bytes ? kChunk * D * KE : kChunk * D * VE;
            }
            if constexpr (!(KF16 && VF16)) {
                if (!(scale_of_k ? KF16 : VF16) && lane < kScalePiece / 16)
                    copy_to_lds_from(src_scale, lane * 16, to + Raw::k_bytes + Raw::v_bytes + wave * kScalePiece);
                src_scale += Raw::scale_bytes;
            }
            ++next;
            --run_left;
        };
        // The item's first `count` steps (whole turns of tiles).
        constexpr uint32_t kFirst = TILES ? W : Raw::turns ? 2 : Raw::landed + 1;
        auto fetch_to = [&](uint32_t count) __attribute__((always_inline)) {
            const uint32_t to = s0 + min(count, (s1 - s0 + W - 1) / W * W);
            while (next < to) fetch();
        };
        // Keys of the step that no row of the item sees may hold anything: their values are zeroed.
        auto unseen = [&](uint32_t t) __attribute__((always_inline)) {
            return (t >= span.past) | ((t < span.vis.lo) & (t >= a.sinks));
        };
        // Whether the step at tok0 holds such keys.
        auto edge = [&](uint32_t tok0) __attribute__((always_inline)) {
            return (tok0 + kChunk > span.past) | ((tok0 < span.vis.lo) & (tok0 + kChunk > a.sinks));
        };
        // V's scales in the order of V's units: each of the first D / 2 threads puts those of two keys, one
        // behind the other in a unit, together.
        auto order_scales = [&](uint32_t i) __attribute__((always_inline)) {
            if (VF16 || wave >= D / 128) return;
            const uint32_t t = here(), blk = t / 16, x = t % 16 * 2;  // element x of the block's 32: G = x / 8, J = x / 4 % 2
            const uint32_t key = x / 4 % 2 * 16 + x / 8 * 4 + x % 4;
            const _Float16* from = reinterpret_cast<const _Float16*>(s_raw + i % Raw::bufs * Raw::raw + Raw::k_bytes + Raw::v_bytes + Raw::scale_bytes) +
                                   key * NB + blk;
            half2v w = {from[0], from[NB]};
            const uint32_t tok0 = uniform(span.vis.step(i) * kChunk);
            if (edge(tok0)) {
                w[0] = unseen(tok0 + key) ? static_cast<_Float16>(0.0f) : w[0];
                w[1] = unseen(tok0 + key + 1) ? static_cast<_Float16>(0.0f) : w[1];
            }
            *reinterpret_cast<half2v*>(s_vsc + (i & 1) * D + 2 * t) = tile_scales(w);
        };
        // A step's codes to fp16: each thread 16 codes of K and / or of V (D = 128: the first four
        // waves K's, the others V's).
        constexpr bool kBoth = D == 256;
        auto convert_k_run = [&](uint32_t i, uint32_t idx) __attribute__((always_inline)) {
            const uint8_t* raw = s_raw + i % Raw::bufs * Raw::raw;
            half8* tile = s_tile + (i & 1) * Raw::units;
            {
                // key 16 T + m, dims 64 c + 8 g and 64 c + 32 + 8 g
                const uint32_t T = idx / D, c = idx / 64 % (D / 64), g = idx / 16 % 4, m = idx % 16;
                half8* to = tile + (8 * c + g) * kChunk + 16 * T + m;
                const uint4* from = reinterpret_cast<const uint4*>(raw) + idx * KE;
                if constexpr (KF16) {
                    to[0] = __builtin_bit_cast(half8, from[0]);
                    to[4 * kChunk] = __builtin_bit_cast(half8, from[1]);
                } else {
                    const uint4 w = from[0];
                    const half2v f = tile_scales(*reinterpret_cast<const half2v*>(raw + Raw::k_bytes + Raw::v_bytes + ((16 * T + m) * NB + 2 * c) * 2));
                    to[0] = codes8_to_half8(w.x, w.y) * f[0];
                    to[4 * kChunk] = codes8_to_half8(w.z, w.w) * f[1];
                }
            }
        };
        auto convert_v_run = [&](uint32_t i, uint32_t idx) __attribute__((always_inline)) {
            const uint8_t* raw = s_raw + i % Raw::bufs * Raw::raw;
            half8* tile = s_tile + (i & 1) * Raw::units;
            {
                // dim d, keys of units 2x and 2x + 1
                const uint32_t d = idx / 2, x = idx % 2;
                half8* to = tile + Raw::k_units + 2 * x * Raw::v_row + d;
                const uint4* from = reinterpret_cast<const uint4*>(raw + Raw::k_bytes) + idx * VE;
                if constexpr (VF16) {
                    half8 v[2] = {__builtin_bit_cast(half8, from[0]), __builtin_bit_cast(half8, from[VF16 ? 1 : 0])};
                    const uint32_t tok0 = uniform(span.vis.step(i) * kChunk);
                    if (edge(tok0)) {
#pragma unroll
                        for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
                            for (uint32_t y = 0; y < 8; ++y)
                                v[u][y] = unseen(tok0 + 16 * (y / 4) + 4 * (2 * x + u) + y % 4) ? static_cast<_Float16>(0.0f) : v[u][y];
                    }
                    to[0] = v[0];
                    to[Raw::v_row] = v[1];
                } else {
                    const uint4 w = from[0];
                    const half8* f = reinterpret_cast<const half8*>(s_vsc + (i & 1) * D + d / 32 * 32 + 16 * x);
                    to[0] = codes8_to_half8(w.x, w.y) * f[0];
                    to[Raw::v_row] = codes8_to_half8(w.z, w.w) * f[1];
                }
            }
        };

        float m_run = -INFINITY, l_run = 0.0f;
        float16v O[NB];

        auto convert_k = [&](uint32_t i) __attribute__((always_inline)) {
            if (kBoth || wave < 4) convert_k_run(i, here());
        };
        auto convert_v = [&](uint32_t i) __attribute__((always_inline)) {
            if (kBoth || wave >= 4) convert_v_run(i, kBoth ? here() : here() & 255u);
        };

        // Whether this wave's rows see anything of a step (wave-uniform).
        auto seen = [&](uint32_t s) __attribute__((always_inline)) {
            const uint32_t tok0 = uniform(span.vis.step(s) * kChunk);
            return wave_live & (tok0 < past_z) & ((a.window == 0) | (tok0 + kChunk > low_a) | (tok0 < a.sinks));
        };
        half8 qf[NQ];
        float16v S[W];
        half8 P[2 * W];
        // O^T += V^T P^T of turn j - 1 (VALUES), then S^T = K Q^T of turn j (SCORES): one run of MFMAs
        // whose fragments are read kAhead ahead.
        auto multiply = [&](auto with_values, auto with_scores, uint32_t j) __attribute__((always_inline)) {
            constexpr uint32_t NV = decltype(with_values)::value ? 2 * NB * W : 0, N = NV + (decltype(with_scores)::value ? NQ * W : 0);
            // value fragment c of a step: dims 32 (c / 2) .., keys of units 2 (c % 2) + hh; key fragment: dims 16 c + 8 hh ..
            const half8* v = s_tile + (j - 1) % kPlaces * W * Lds::units + Lds::k_units + hh * Lds::v_row + n;
            const half8* k = s_tile + j % kPlaces * W * Lds::units + hh * kChunk + n;
            auto at = [&](uint32_t c) __attribute__((always_inline)) {
                return c < NV ? v[c / (2 * NB) * Lds::units + c % (2 * NB) / 2 * kChunk + c % 2 * 2 * Lds::v_row]
                              : k[(c - NV) / NQ * Lds::units + (c - NV) % NQ * 2 * kChunk];
            };
            half8 f[kAhead];
#pragma unroll
            for (uint32_t c = 0; c < kAhead; ++c) f[c] = at(c);
            if constexpr (decltype(with_scores)::value)
#pragma unroll
                for (uint32_t u = 0; u < W; ++u)
#pragma unroll
                    for (uint32_t x = 0; x < 16; ++x) S[u][x] = 0.0f;
            __builtin_amdgcn_sched_barrier(0);  // the scheduler would move reads to their use, or all of them up here
#pragma unroll
            for (uint32_t c = 0; c < N; ++c) {
                if (c < NV) O[c % (2 * NB) / 2] = mfma_32x32x16(f[c % kAhead], P[c / (2 * NB) * 2 + c % 2], O[c % (2 * NB) / 2]);
                else S[(c - NV) / NQ] = mfma_32x32x16(f[c % kAhead], qf[(c - NV) % NQ], S[(c - NV) / NQ]);
                if (c + kAhead < N) f[c % kAhead] = at(c + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const std::true_type yes{};
        const std::false_type no{};
        // Of the turn whose first step is s.
        auto softmax = [&](uint32_t s) __attribute__((always_inline)) {
            float top = -INFINITY;
#pragma unroll
            for (uint32_t u = 0; u < W; ++u) {
                const uint32_t tok0 = uniform(span.vis.step(s + u) * kChunk);
                const bool there = W == 1 || s + u < s1;
                const bool whole = there & (tok0 + kChunk <= past_a) & ((a.window == 0) | (tok0 + kChunk <= a.sinks) | (tok0 >= low_z));
                if (!whole) {
#pragma unroll
                    for (uint32_t x = 0; x < 16; ++x) {
                        const uint32_t t = tok0 + 8 * (x / 4) + 4 * hh + x % 4;
                        S[u][x] = !there | (t >= past) | ((t < low) & (t >= a.sinks)) ? -INFINITY : S[u][x];
                    }
                }
                // (fmaxf would first quieten each of its inputs)
                top = max3(top, max3(max3(S[u][0], S[u][1], S[u][2]), max3(S[u][3], S[u][4], S[u][5]), max3(S[u][6], S[u][7], S[u][8])),
                           max3(max3(S[u][9], S[u][10], S[u][11]), max3(S[u][12], S[u][13], S[u][14]), S[u][15]));
            }
            top = swap32_reduce(top, MaxOp{}) * a.scale_log2;
            if (__any(top > m_run + kSlack)) {
                const float to = fmaxf(m_run, top);
                const float f = m_run == -INFINITY ? 0.0f : exp2_fast(m_run - to);
                m_run = to;
                l_run *= f;
#pragma unroll
                for (uint32_t mt = 0; mt < NB; ++mt) O[mt] *= f;
            }
            const float use = m_run == -INFINITY ? 0.0f : m_run;
            // and the sum of the probabilities as the second product takes them
            const half2v one = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
            float sum[2 * W] = {};
#pragma unroll
            for (uint32_t u = 0; u < W; ++u) {
#pragma unroll
                for (uint32_t x = 0; x < 16; ++x)
                    P[2 * u + x / 4 % 2][x % 4 + x / 8 * 4] = static_cast<_Float16>(exp2_fast(fmaf(S[u][x], a.scale_log2, -use)));
#pragma unroll
                for (uint32_t x = 0; x < 8; x += 2)
#pragma unroll
                    for (uint32_t y = 2 * u; y < 2 * u + 2; ++y) sum[y] = __builtin_amdgcn_fdot2(half2v{P[y][x], P[y][x + 1]}, one, sum[y], false);
            }
#pragma unroll
            for (uint32_t y = 0; y < 2 * W; y += 2) l_run += sum[y] + sum[y + 1];
        };
        if (s0 < s1) {
            lds_barrier();  // the previous item's tiles and ring have been read
            // no more than the first pass reads: the query is waited for behind these
            fetch_to(kFirst);
        }
        // The query comes row by row, each wave's through LDS of its own where no tile is yet.  (Fragments
        // read straight from memory touch a line in each of 32 rows at a time.)
        if (s0 < s1)
            with_type(a.q_dtype, [&](auto t) __attribute__((always_inline)) {
                const uint32_t me = here() % 64, mn = me % 32, mh = me / 32;
                half8* const stage = s_tile + (TILES ? (kPlaces - 1) * W * Lds::units : 0) + wave * (kStageBytes / 16);
#pragma unroll
                for (uint32_t d0 = 0; d0 < D; d0 += 128) {
                    half8 x[4][2];
#pragma unroll
                    for (uint32_t p = 0; p < 4; ++p) {
                        const size_t at = static_cast<size_t>(__shfl(static_cast<int>(row_index), 8 * p + me / 8, 64)) * D + d0 + 8 * (me % 8);
                        x[p][0] = load_query<decltype(t)>(a.q, at);
                        x[p][1] = load_query<decltype(t)>(a.q, at + 64);
                    }
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
#pragma unroll
                        for (uint32_t p = 0; p < 4; ++p) stage[(8 * p + me / 8) * 8 + (me % 8 ^ me / 8)] = x[p][e];
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) qf[d0 / 16 + 4 * e + k] = stage[mn * 8 + ((2 * k + mh) ^ (mn % 8))];
                    }
                }
            });
        if (a.negate)
#pragma unroll
            for (uint32_t k = 0; k < NQ; ++k) qf[k] = -qf[k];
        // The query has arrived: otherwise its loads are waited for in every step, and with them
        // the copies, which the compiler does not count.
#pragma unroll
        for (uint32_t k = 0; k < NQ; ++k) asm volatile("" : "+v"(qf[k]));

#pragma unroll
        for (uint32_t mt = 0; mt < NB; ++mt)
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) O[mt][x] = 0.0f;

        if (s0 < s1) {
            wait_vmem();
            if constexpr (TILES) {
                lds_barrier();
                fetch_to(kPlaces * W);
            } else {
                fetch_to(Raw::bufs);
                lds_barrier();
                order_scales(s0);
                if (!Raw::turns && s0 + 1 < s1) order_scales(s0 + 1);
                lds_barrier();
                convert_k(s0);
                if (!Raw::turns || wave >= 4) convert_v(s0);
            }
        }
        if constexpr (TILES) {
            // The two waves of a SIMD take turns of W steps: while waves 0..3 multiply (values of turn j - 1,
            // scores of turn j), waves 4..7 do the softmax of turn j - 1, and the other way round.
            // The first half multiplies in interval 2j and computes in 2j + 1, the second half one
            // interval later.  Turn j is read from 2j to 2j + 3 and must have landed before 2j; its
            // place is fetched into anew from 2j + 4 on, in the intervals of turn j + 2.
            const bool second = wave >= 4;
            const uint32_t turns = (s1 - s0 + W - 1) / W;
            auto turns_of = [&](auto live) __attribute__((always_inline)) {
                constexpr bool kLive = decltype(live)::value;
                if (second) lds_barrier();
                if constexpr (kLive) multiply(no, yes, 0);
                // (The last pass multiplies scores that nothing uses: leaving the loop in front of them would
                // hold the accumulators twice.)
                for (uint32_t j = 0; j < turns; ++j) {
                    if (second) {  // turn j + 1 has landed
                        if (j + kPlaces - 3 < turns) wait_vmem_le<(kPlaces - 4) * TileLds<D>::ops>();
                        else wait_vmem();
                    }
                    lds_barrier();
                    if (j >= 2 && j + kPlaces - 2 < turns)  // turn j + 2
#pragma unroll
                        for (uint32_t u = 0; u < W; ++u) fetch();
                    if constexpr (kLive) softmax(s0 + j * W);
                    if (!second) {
                        if (j + kPlaces - 2 < turns) wait_vmem_le<(kPlaces - 3) * TileLds<D>::ops>();
                        else wait_vmem();
                    }
                    // (the exponentials would move behind the barrier, into the turn that multiplies)
                    __builtin_amdgcn_sched_barrier(0);
                    lds_barrier();
                    if constexpr (kLive) {
                        __builtin_amdgcn_s_setprio(1);
                        multiply(yes, yes, j + 1);
                        __builtin_amdgcn_s_setprio(0);
                    }
                }
                if (!second) lds_barrier();
            };
            if (s0 < s1) {
                if (wave_live) turns_of(yes);
                else turns_of(no);
                place = (turns + 1) % kPlaces;
            }
        } else if constexpr (Raw::turns) {
            // The two waves of a SIMD take turns: while waves 0..3 multiply (values of step s - 1, scores
            // of step s), waves 4..7 do what is left to the vector unit (softmax of step s - 1, codes to
            // fp16), and the other way round.  With t = s - s0, in interval 2t the first half multiplies,
            // in 2t + 1 it computes; the second half is one interval later.  A tile's K is
            // whole before interval 2t: its codes are converted by the first half in 2t - 1, by the
            // second in 2t - 2; its V before 2t + 2: in 2t + 1 and 2t.  Each overwrites what was
            // last read an interval before or earlier: K of step s - 2 in 2t - 3, V of step s - 2 in
            // 2t - 1.  The ring's place of step s is free from 2t + 2.
            // A wave without rows only copies and converts.  (What a wave's rows do not see of the item's
            // steps is multiplied and masked: with a branch around it the accumulators would be held
            // twice.)
            // Where the rows fill no wave of the second half, it converts all codes, K of step s + 1 in
            // interval 2t and V of step s in 2t + 1.
            const bool second = wave >= 4;
            const bool helped = span.rows <= kRows / 2;
            auto steps_of = [&](auto live) __attribute__((always_inline)) {
                constexpr bool kLive = decltype(live)::value;
                if (second) {
                    if (s0 + 1 < s1) convert_k(s0 + 1);
                    lds_barrier();
                }
                lds_barrier();
                if constexpr (kLive) multiply(no, yes, s0);
                // (The last pass multiplies scores that nothing uses, of whatever the tile holds: leaving
                // the loop in front of them would hold the accumulators twice.)
                for (uint32_t s = s0; s < s1; ++s) {
                    if (second) wait_vmem();  // step s + 2 has landed
                    lds_barrier();
                    if (s != s0 && s + 3 < s1) fetch();  // step s + 3
                    if (!second && s + 1 < s1) order_scales(s + 1);
                    if constexpr (kLive) softmax(s);
                    if (second) {
                        if (s + 2 < s1) convert_k(s + 2);
                        if (s + 1 < s1) convert_v(s + 1);
                    } else {
                        if (!helped) {
                            if (s + 1 < s1) convert_k(s + 1);
                            convert_v(s);
                        }
                        if (s + 3 < s1) wait_vmem_le<Raw::ops>();  // step s + 2 has landed
                        else wait_vmem();
                    }
                    lds_barrier();
                    if constexpr (kLive) {
                        __builtin_amdgcn_s_setprio(1);
                        multiply(yes, yes, s + 1);
                        __builtin_amdgcn_s_setprio(0);
                    }
                }
                if (!second) lds_barrier();
            };
            auto help = [&]() __attribute__((always_inline)) {
                constexpr uint32_t kRuns = kBoth ? 2 : 1;
                lds_barrier();
                for (uint32_t s = s0; s < s1; ++s) {
                    if (s >= s0 + 2 && s + 2 < s1) fetch();  // step s + 2
                    if (s + 1 < s1)
#pragma unroll
                        for (uint32_t x = 0; x < kRuns; ++x) convert_k_run(s + 1, (here() & 255u) + 256 * x);
                    lds_barrier();
#pragma unroll
                    for (uint32_t x = 0; x < kRuns; ++x) convert_v_run(s, (here() & 255u) + 256 * x);
                    wait_vmem();  // step s + 2 has landed
                    lds_barrier();
                }
                lds_barrier();
            };
            if (s0 < s1) {
                if (helped & second) help();
                else if (wave_live) steps_of(yes);
                else steps_of(no);
            }
        } else {
            for (uint32_t s = s0; s < s1; ++s) {
                // The step that is `landed` ahead is whole in the ring, of every wave's copies.
                if (s != s0) {
                    if (KF16 == VF16 && s + Raw::bufs - 1 < s1) wait_vmem_le<(Raw::bufs - 1 - Raw::landed) * Raw::ops>();
                    else wait_vmem();
                }
                lds_barrier();
                if (s + Raw::bufs < s1) fetch();  // where step s was, which is a tile now
                if (s + 2 < s1) order_scales(s + 2);
                if (s + 1 < s1) {
                    convert_k(s + 1);
                    convert_v(s + 1);
                }
                if (!seen(s)) continue;
                multiply(no, yes, s);
                softmax(s);
                multiply(yes, no, s + 1);
            }
        }
        l_run = swap32_reduce(l_run, AddOp{});
        const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;  // a token that sees no key: zeros
        // Out row by row, through LDS that no wave reads any more: of a ring of tiles the place behind the
        // scores that nothing uses, else the ring of codes.
        uint8_t* const stage = (TILES ? lds + place * W * Lds::units * 16 : s_raw) + wave * kStageBytes;
        auto put = [&](auto t, void* to, bool whole) __attribute__((always_inline)) {
            const uint32_t me = here() % 64, mn = me % 32, mh = me / 32;
            using T = decltype(t);
            typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
            typedef T vec4 __attribute__((ext_vector_type(4)));
            constexpr uint32_t kDims = 128 / sizeof(T);  // 128 bytes of each row at a time
            const size_t rec = static_cast<size_t>(2 * part + (first < begin ? 0u : 1u)) * kRows + wave * 32;
#pragma unroll
            for (uint32_t d0 = 0; d0 < D; d0 += kDims) {
#pragma unroll
                for (uint32_t d = 0; d < kDims; d += 8) {  // this lane's 4 of 8
                    const uint32_t mt = (d0 + d) / 32, x = (d0 + d) % 32 / 2, byte = (d + 4 * mh) * sizeof(T);
                    *reinterpret_cast<vec4*>(stage + mn * 128 + ((byte / 16 ^ mn % 8) * 16) + byte % 16) =
                        vec4{static_cast<T>(O[mt][x] * inv), static_cast<T>(O[mt][x + 1] * inv), static_cast<T>(O[mt][x + 2] * inv), static_cast<T>(O[mt][x + 3] * inv)};
                }
#pragma unroll
                for (uint32_t p = 0; p < 4; ++p) {
                    const uint32_t y = 8 * p + me / 8;
                    const vec v = *reinterpret_cast<const vec*>(stage + y * 128 + (me % 8 ^ me / 8) * 16);
                    const size_t at = whole ? static_cast<size_t>(__shfl(static_cast<int>(row_index), y, 64)) : rec + y;
                    if (wave * 32 + y < span.rows)
                        *reinterpret_cast<vec*>(static_cast<T*>(to) + at * D + d0 + me % 8 * (16 / sizeof(T))) = v;
                }
            }
        };
        if (!wave_live) continue;
        if (s1 - s0 == steps) {
            with_type(a.out_dtype, [&](auto t) __attribute__((always_inline)) { put(t, a.out, true); });
        } else {
            put(_Float16{}, a.rec_o, false);
            const uint32_t me = here() % 64, y = wave * 32 + me % 32;
            if ((me < 32) & (y < span.rows))
                a.rec_ml[static_cast<size_t>(2 * part + (first < begin ? 0u : 1u)) * kRows + y] = make_float2(m_run, l_run);
        }
    }
}

// Merge of the items that were cut (8 to 11 us: two dependent reads, then up to 512 records of 64 or 128 KiB):
// workgroup (item, kv head, merge_rows<D> rows), D / 16 threads per row.
template <uint32_t D>
constexpr uint32_t merge_rows = 256 * 16 / D;
template <uint32_t D>
__global__ void __launch_bounds__(256) chunk_merge_kernel(ChunkArgs a) {
    constexpr uint32_t kThreads = D / 16, kMergeRows = merge_rows<D>;
    const uint32_t i = blockIdx.x / (kRows / kMergeRows), h = blockIdx.y;
    const uint32_t r = blockIdx.x % (kRows / kMergeRows) * kMergeRows + threadIdx.x / kThreads, part = threadIdx.x % kThreads;
    const ChunkItem it = a.items[i];  // (of nothing behind the last one: read with `head`, not after it)
    const uint32_t items = a.head[0], units = a.head[1], quota = a.head[2];
    if (i >= items || it.steps == 0 || r >= it.rows) return;
    const uint32_t first = h * units + it.start + kItemCost;
    const uint32_t w0 = uniform(first / quota), w1 = uniform((first + it.last) / quota);
    if (w0 == w1) return;  // written whole
    const uint32_t tok = it.tok0 + (it.head0 + r) / a.group, head = h * a.group + (it.head0 + r) % a.group;
    constexpr uint32_t kPer = 2;  // groups of 8 values per thread
    constexpr uint32_t kDepth = 4;     // records read at a time
    float acc[kPer][8] = {};
    float m = -INFINITY, sum = 0.0f;
    for (uint32_t w = w0; w <= w1; w += kDepth) {
        float2 ml[kDepth];
        half8 o[kDepth][kPer];
#pragma unroll
        for (uint32_t j = 0; j < kDepth; ++j) {
            ml[j] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (uint32_t k = 0; k < kPer; ++k) o[j][k] = half8{};
            if (w + j <= w1) {
                const size_t rec = static_cast<size_t>(2 * (w + j) + (first < (w + j) * quota ? 0u : 1u)) * kRows + r;
                ml[j] = a.rec_ml[rec];
#pragma unroll
                for (uint32_t k = 0; k < kPer; ++k) o[j][k] = *reinterpret_cast<const half8*>(a.rec_o + rec * D + D / 2 * k + 8 * part);
            }
        }
        float to = m;
#pragma unroll
        for (uint32_t j = 0; j < kDepth; ++j) to = fmaxf(to, ml[j].x);
        const float keep = m == -INFINITY ? 0.0f : exp2_fast(m - to);
        m = to;
        sum *= keep;
        float f[kDepth];
#pragma unroll
        for (uint32_t j = 0; j < kDepth; ++j) {
            f[j] = ml[j].x == -INFINITY ? 0.0f : ml[j].y * exp2_fast(ml[j].x - m);
            sum += f[j];
        }
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
#pragma unroll
            for (uint32_t x = 0; x < 8; ++x) {
                acc[k][x] *= keep;
#pragma unroll
                for (uint32_t j = 0; j < kDepth; ++j) acc[k][x] = fmaf(static_cast<float>(o[j][k][x]), f[j], acc[k][x]);
            }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    const size_t at = (static_cast<size_t>(tok) * a.q_heads + head) * D + 8 * part;
    with_type(a.out_dtype, [&](auto t) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t k = 0; k < kPer; ++k)
#pragma unroll
            for (uint32_t x = 0; x < 8; x += 4)
                store4<decltype(t)>(a.out, at + D / 2 * k + x, make_float4(acc[k][x] * inv, acc[k][x + 1] * inv, acc[k][x + 2] * inv, acc[k][x + 3] * inv));
    });
}

uint64_t up256(uint64_t x) { return (x + 255) / 256 * 256; }

uint32_t chunk_lds_bytes(uint32_t D, bool kf, bool vf) {
    if (D == 128)
        return kf ? (vf ? ChunkLds<128, true, true>::bytes : ChunkLds<128, true, false>::bytes)
                  : (vf ? ChunkLds<128, false, true>::bytes : ChunkLds<128, false, false>::bytes);
    return kf ? (vf ? ChunkLds<256, true, true>::bytes : ChunkLds<256, true, false>::bytes)
              : (vf ? ChunkLds<256, false, true>::bytes : ChunkLds<256, false, false>::bytes);
}

struct ChunkPlan {
    uint64_t items;  // of one kv head, at most
    uint32_t parts;
    size_t lds;
    uint32_t steps;  // of a (sequence, kv head), at most
    bool tiles;      // expand first
    uint64_t item_bytes, o_bytes, ml_bytes, tile_bytes;
    uint64_t bytes() const { return 256 + item_bytes + o_bytes + ml_bytes + tile_bytes; }
};

// Sizes and the plan's bounds; a status.
int chunk_plan(const miikv_view* v, uint32_t q_heads, uint32_t batch, uint32_t total_tokens, uint32_t max_tokens,
               uint32_t max_context, uint32_t window, uint32_t sinks, ChunkPlan& p) {
    const int st = validate_view(v);
    if (st != MIIKV_OK) return st;
    if (batch == 0 || total_tokens == 0 || max_tokens == 0 || q_heads == 0 || q_heads % v->kv_heads != 0) return MIIKV_EINVAL;
    if (max_context == 0 || max_context > view_seq_capacity(v) || max_context > 0x7fffffffu) return MIIKV_EINVAL;
    if (max_tokens > total_tokens || max_tokens > max_context) return MIIKV_EINVAL;
    if (v->layout == MIIKV_LAYOUT_CONTIGUOUS && batch != 1) return MIIKV_EINVAL;
    const uint64_t rows = static_cast<uint64_t>(total_tokens) * (q_heads / v->kv_heads);
    if (rows > 0x7fffffffu || static_cast<uint64_t>(total_tokens) * q_heads > 0x7fffffffu || batch > 65535u || v->kv_heads > 65535u) return MIIKV_EUNSUPPORTED;
    // every sequence's last item may be a part of one
    p.items = std::min<uint64_t>(rows / kRows + batch, rows);
    p.steps = most_visible_steps(max_context, max_tokens, window, sinks);
    const uint64_t most = kItemCost + (p.steps + 1ull) * kStepCost;  // (whole turns)
    const uint64_t axis = p.items * most * v->kv_heads;
    if (axis / v->kv_heads / most != p.items || axis > 0xf0000000u) return MIIKV_EUNSUPPORTED;  // 32-bit places on the axis
    p.parts = static_cast<uint32_t>(std::min<uint64_t>(kMaxParts, (axis + kMinUnits - 1) / kMinUnits));
    const uint32_t D = v->head_dim;
    const uint64_t tile_bytes = static_cast<uint64_t>(batch) * v->kv_heads * p.steps * (128u * D);
    p.tiles = rows >= static_cast<uint64_t>(kTileItems) * kRows * batch && tile_bytes <= kMaxTileBytes && batch <= 65535u;
    p.tile_bytes = p.tiles ? tile_bytes : 0u;
    p.lds = p.tiles ? (D == 128 ? TileLds<128>::bytes : TileLds<256>::bytes) : chunk_lds_bytes(D, mode_k_f16(v->quant_mode), mode_v_f16(v->quant_mode));
    p.lds += (static_cast<size_t>(batch) + 1 + p.items + 1) * sizeof(uint32_t);
    if (p.lds > 159 * 1024) return MIIKV_EUNSUPPORTED;
    p.item_bytes = up256(p.items * sizeof(ChunkItem));
    p.o_bytes = up256(2ull * p.parts * kRows * D * sizeof(uint16_t));
    p.ml_bytes = up256(2ull * p.parts * kRows * 2 * sizeof(float));
    return MIIKV_OK;
}

template <uint32_t D>
int launch_chunk(const ChunkArgs& a, const ChunkPlan& p, bool kf, bool vf, hipStream_t s) {
    const dim3 grid((p.parts + 7) / 8 * 8);
    const auto go = [&](auto k, auto v) {
        constexpr bool KF = decltype(k)::value, VF = decltype(v)::value;
        if (p.tiles) {
            hipLaunchKernelGGL((expand_kernel<D, KF, VF>), dim3(p.steps, a.g.kv_heads, a.batch), dim3(256), 0, s, a);
            hipLaunchKernelGGL((chunk_kernel<D, false, false, true>), grid, dim3(kChunkThreads), p.lds, s, a);
        } else {
            hipLaunchKernelGGL((chunk_kernel<D, KF, VF, false>), grid, dim3(kChunkThreads), p.lds, s, a);
        }
    };
    const auto with_v = [&](auto k) { vf ? go(k, std::true_type{}) : go(k, std::false_type{}); };
    kf ? with_v(std::true_type{}) : with_v(std::false_type{});
    hipLaunchKernelGGL((chunk_merge_kernel<D>), dim3(static_cast<uint32_t>(p.items) * (kRows / merge_rows<D>), a.g.kv_heads), dim3(256), 0, s, a);
    return hip_status(hipGetLastError());
}

}  // namespace
}  // namespace miikv

using namespace miikv;

extern "C" uint64_t miikv_chunk_workspace_bytes(const miikv_view* view, uint32_t q_heads, uint32_t batch,
                                                uint32_t total_tokens, uint32_t max_tokens, uint32_t max_context,
                                                uint32_t window, uint32_t sinks) {
    ChunkPlan p{};
    if (window >= max_context) window = 0;
    if (chunk_plan(view, q_heads, batch, total_tokens, max_tokens, max_context, window, std::min(sinks, max_context), p) != MIIKV_OK)
        return 0;
    return p.bytes();
}

extern "C" miikv_status miikv_chunk_attn(const miikv_view* view, const void* q, uint32_t q_dtype, uint32_t q_heads,
                                         float scale, uint32_t batch, uint32_t total_tokens, const uint32_t* d_offsets,
                                         const uint32_t* d_lengths, uint32_t max_tokens, uint32_t max_context,
                                         uint32_t window, uint32_t sinks, void* out, uint32_t out_dtype, void* workspace,
                                         uint64_t workspace_bytes, void* stream) {
    ChunkPlan p{};
    if (window >= max_context) window = 0;  // hides nothing
    sinks = std::min(sinks, max_context);
    const int st = chunk_plan(view, q_heads, batch, total_tokens, max_tokens, max_context, window, sinks, p);
    if (st != MIIKV_OK) return st;
    if (q == nullptr || out == nullptr || d_offsets == nullptr || d_lengths == nullptr || !std::isfinite(scale) ||
        q_dtype > MIIKV_DTYPE_BF16 || out_dtype > MIIKV_DTYPE_BF16)
        return MIIKV_EINVAL;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || !aligned16(view->k_codes) || !aligned16(view->v_codes) ||
        !aligned16(view->k_scales) || !aligned16(view->v_scales))
        return MIIKV_EINVAL;
    if (workspace == nullptr || workspace_bytes < p.bytes()) return MIIKV_EWORKSPACE;
    ChunkArgs a{};
    a.g = make_geo(*view);
    a.q = q;
    a.q_dtype = q_dtype;
    a.q_heads = q_heads;
    a.group = q_heads / view->kv_heads;
    a.scale_log2 = std::max(std::fabs(scale) * kLog2eF, 1e-30f);  // (0 times a hidden key's -inf would be NaN)
    a.negate = scale < 0.0f ? 1u : 0u;
    a.batch = batch;
    a.total_tokens = total_tokens;
    a.max_tokens = max_tokens;
    a.max_context = max_context;
    a.window = window;
    a.sinks = sinks;
    a.offsets = d_offsets;
    a.lengths = d_lengths;
    a.out = out;
    a.out_dtype = out_dtype;
    a.most_items = static_cast<uint32_t>(p.items);
    a.parts = p.parts;
    a.page_steps = view->page_tokens / kChunk;
    // mulhi(x, ceil(2^32 / d)) == x / d where x * d < 2^32
    const uint64_t steps = (static_cast<uint64_t>(max_context) + kChunk - 1) / kChunk;
    a.page_magic = steps * a.page_steps < 0xffffffffu ? static_cast<uint32_t>((0x100000000ull + a.page_steps - 1) / a.page_steps) : 0u;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.head = reinterpret_cast<uint32_t*>(ws);
    a.items = reinterpret_cast<ChunkItem*>(ws + 256);
    a.rec_o = reinterpret_cast<_Float16*>(ws + 256 + p.item_bytes);
    a.rec_ml = reinterpret_cast<float2*>(ws + 256 + p.item_bytes + p.o_bytes);
    a.most_steps = p.steps;
    a.tiles = reinterpret_cast<const half8*>(ws + 256 + p.item_bytes + p.o_bytes + p.ml_bytes);
    const bool kf = mode_k_f16(view->quant_mode), vf = mode_v_f16(view->quant_mode);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return view->head_dim == 128 ? launch_chunk<128>(a, p, kf, vf, s) : launch_chunk<256>(a, p, kf, vf, s);
}
