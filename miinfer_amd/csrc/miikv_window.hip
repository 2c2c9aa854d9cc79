// Decode attention over part of a cache (a sliding window and the first tokens), and over
// the whole of it with the weight that every key gets (gfx950, wave64, MFMA).
//
// For the last T tokens of a sequence (T * G <= 16, G query heads per kv head) and the
// keys j that token t sees:
//   s_tj = scale * q_t . k_j,  o_t = sum_j e^{s_tj - m_t} v_j / l_t,  m_t = max_j s_tj,
//   l_t = sum_j e^{s_tj - m_t};  weights: w_j += sum over t and the G heads of
//   e^{s_tj - m_t} / l_t.
// One pass over the keys keeps (m, l, o) per column (token, head); the T * G columns of a
// kv head share every byte that is read.
//
// Bound: the stream of the visible keys' codes (HBM) where it is long (24 sequences, window 4096, head_dim 256:
// 191 MB in 40 us, 5 of them before the first data), the chain of dependent reads and the second launch where it
// is short (one sequence, window 1024: 6 + 4 us).
//
// The results are fp32 and hold fp32's precision: the codes enter the MFMAs as exact fp16
// integers, K's block scales are applied to fp32 sums, an fp32 query as hi + lo fp16 parts,
// and the probabilities (times V's block scale) as hi + lo fp16 parts too, 22 bits in all.
// P enters 2^shift above its value, so that both parts of a probability of 2^-20 stay clear
// of fp16's denormals: p <= 1 is multiplied by V's block scale, so shift is what the largest
// scale so far leaves below 2^15 (values of 0.02: outputs 4.5e-7 off; with a shift of 6 they
// were 3.4e-6 to 4.9e-6 off).
//
// Work: the visible 32-key steps of all sequences are cut into runs, one workgroup (of four
// waves) each, as many as the chip holds.  Their length is chosen on the device from the
// lengths, so that the runs of a ragged batch fill the chip whatever the lengths are.  A workgroup writes one record (o, m, l)
// per run; the second launch merges the records and, for weights, turns the kept scores
// into probabilities with the merged m and l.
#include "miikv_part.hpp"

#include <algorithm>
#include <type_traits>

namespace miikv {
namespace {

constexpr uint32_t kWaves = 4;            // waves per workgroup
constexpr int kMinShift = -1;             // 2^-1 * 65504 < 2^15
constexpr int kMaxShift = 24;
constexpr uint32_t kTargetWgs = 512;      // two workgroups per CU
constexpr uint32_t kWeightKeys = 256;     // keys per workgroup of the weights pass

struct PartArgs {
    Geo g;
    const void* q;
    uint32_t q_heads;
    uint32_t heads;   // query heads per kv head
    uint32_t tokens;  // tokens per sequence
    uint32_t cols;    // heads * tokens <= 16
    float scale_log2;
    const uint32_t* len_ptr;  // context length of sequence b: len_ptr[b * len_stride] + len_add
    uint32_t len_stride;
    uint32_t len_add;
    uint32_t max_context;
    uint32_t window;
    uint32_t sinks;
    uint32_t batch;
    uint32_t* runs;  // [batch][kv_heads][2]: first record and records of a pair that has any
    float* part;     // a record per run: o [cols][D], r [cols], l [cols], padded to 4, where
                     // o = sum of 2^(s - r) v and l = sum of 2^(s - r)
    float* logits;   // SCORED: scores in log2 units [batch][kv_heads][cols][logit_keys]
    uint32_t logit_keys;
    float* weights;  // SCORED: [batch][kv_heads][weight_stride]
    uint64_t weight_stride;
    uint32_t combine_wgs;  // workgroups of the second launch that merge records
    float* out;
    const float* gate;
    float* gated_out;
};

__host__ __device__ __forceinline__ uint32_t part_record(uint32_t cols, uint32_t D) { return cols * D + (2 * cols + 3) / 4 * 4; }

__device__ __forceinline__ uint32_t part_length(const PartArgs& a, uint32_t b) {
    const uint32_t L = a.len_ptr[static_cast<size_t>(b) * a.len_stride] + a.len_add;
    return min(L, a.max_context);
}
__device__ __forceinline__ uint32_t part_steps(const PartArgs& a, uint32_t b) {
    return visible_steps(part_length(a, b), a.tokens, a.window, a.sinks).steps();
}

// Run of one workgroup.
struct Run {
    uint32_t b, h;
    uint32_t split;  // number of the run among (b, h)'s
    uint32_t runs;   // of (b, h)
    bool live;
};

__device__ __forceinline__ uint32_t lane_of(uint32_t x, uint32_t lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), static_cast<int>(lane)));
}

// The run of workgroup w (all lanes take part, the result is wave-uniform).  In the order
// (sequence, kv head, split), sequence b has kv_heads * runs_of(its steps) runs.
__device__ __forceinline__ Run find_run(const PartArgs& a, uint32_t w) {
    const uint32_t lane = threadIdx.x & 63, heads = a.g.kv_heads;
    Run r{};
    unsigned long long sum = 0;
    uint32_t mine = 0;  // steps of sequence `lane`
    if (a.batch <= 64) {
        mine = lane < a.batch ? part_steps(a, lane) : 0u;
        sum = lane_of(sum_to_lane(mine), 63);  // (64 contexts of at most 2^26 steps, not all of them that long)
    } else {
        for (uint32_t b = lane; b < a.batch; b += 64) sum += part_steps(a, b);
#pragma unroll
        for (uint32_t off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
    }
    sum *= heads;
    // The longest run, in sixteenths of a step: as short as leaves no more runs than slots, a step per wave at
    // least.  (Multiples of four steps left a quarter of the slots empty or a few runs for a second round: 4
    // sequences of 4 tokens 26.7 and 25.0 us.  Shorter runs for the workgroups that the CUs get second, which end
    // later, were slower: 24.3 and 25.8 us for one sequence of 32768 keys.)
    const unsigned long long share = (sum * 16 + kTargetWgs - 1) / kTargetWgs;
    const uint32_t even = share < 0x3fffffffull ? static_cast<uint32_t>(share) : 0x3fffffffu;
    uint32_t most = max(even, 16 * kWaves), n = 0, total = 0;
    auto runs_of = [&](uint32_t steps) { return (16 * steps + most - 1) / most; };
    if (a.batch <= 64) {
        for (uint32_t x = 0;; ++x) {
            n = runs_of(mine) * heads;
            total = lane_of(sum_to_lane(n), 63);
            if (total <= kTargetWgs || x == 16) break;
            most = max(even + even / 16 * (x + 1) + 1, 16 * kWaves);
        }
    } else {
        for (uint32_t b = lane; b < a.batch; b += 64) total += runs_of(part_steps(a, b)) * heads;
        total = lane_of(sum_to_lane(total), 63);
    }
    if (w >= total) return r;
    uint32_t base = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        if (a.batch > 64) n = b0 + lane < a.batch ? runs_of(part_steps(a, b0 + lane)) * heads : 0u;
        const uint32_t upto = base + sum_to_lane(n);
        const unsigned long long behind = __ballot(w < upto);
        if (behind != 0) {
            const uint32_t src = static_cast<uint32_t>(__builtin_ctzll(behind));
            const uint32_t all = lane_of(n, src), x = w - (lane_of(upto, src) - all);
            r.runs = __builtin_amdgcn_readfirstlane(all / heads);
            r.b = b0 + src;
            r.h = __builtin_amdgcn_readfirstlane(x / r.runs);
            r.split = x - r.h * r.runs;
            r.live = true;
            return r;
        }
        base = lane_of(upto, 63);
    }
    return r;
}

// The first step of a pair's k-th run: its steps are cut evenly into its runs.
__device__ __forceinline__ uint32_t run_begin(uint32_t steps, uint32_t k, uint32_t runs) {
    const uint64_t at = static_cast<uint64_t>(steps) * k;
    if (at <= 0xffffffffu) return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at) / runs);
    return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at / runs));
}

// Records of (b, h), which the first launch has noted for pairs that see any key.
__device__ __forceinline__ void find_records(const PartArgs& a, uint32_t bh, uint32_t b, uint32_t& first, uint32_t& runs) {
    const uint2 at = *reinterpret_cast<const uint2*>(a.runs + 2 * static_cast<size_t>(bh));
    first = at.x;
    runs = part_length(a, b) != 0 ? at.y : 0u;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ uint4 stream16(const void* p) {
    typedef unsigned int u4v __attribute__((ext_vector_type(4)));
    const u4v t = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(p));
    return make_uint4(t.x, t.y, t.z, t.w);
}
__device__ __forceinline__ uint2 stream8(const void* p) {
    typedef unsigned int u2v __attribute__((ext_vector_type(2)));
    const u2v t = __builtin_nontemporal_load(reinterpret_cast<const u2v*>(p));
    return make_uint2(t.x, t.y);
}

// Waves per SIMD that an instance is compiled for.
template <uint32_t D, bool QF32, bool KF16, bool VF16>
constexpr uint32_t part_waves_per_eu() {
    return D == 256 && (QF32 || KF16 || VF16) ? 1u : 2u;
}

template <uint32_t D, bool QF32, bool KF16, bool VF16, bool SCORED>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(part_waves_per_eu<D, QF32, KF16, VF16>())))
part_kernel(PartArgs a) {
    constexpr uint32_t NB = D / 32;  // q8_0 blocks per row
    constexpr uint32_t NC = D / 64;
    constexpr uint32_t NM = D / 16;  // 16-dim tiles of V
    using ScaleVec = typename std::conditional<NB == 4, uint32_t, uint2>::type;  // NB / 2 fp16 scales
    extern __shared__ float smem[];  // cross-wave merge; while stepping, each wave's scales

    const Run run = find_run(a, blockIdx.x);
    if (!run.live) return;  // workgroup-uniform
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63, g4 = lane >> 4, n = lane & 15;
    const uint32_t b = run.b, h = run.h;
    const Geo& geo = a.g;
    const uint32_t L = part_length(a, b);
    const Visible vis = visible_steps(L, a.tokens, a.window, a.sinks);
    const uint32_t from = run_begin(vis.steps(), run.split, run.runs), to = run_begin(vis.steps(), run.split + 1, run.runs);
    if (run.split == 0 && threadIdx.x == 0)
        *reinterpret_cast<uint2*>(a.runs + 2 * (static_cast<size_t>(b) * geo.kv_heads + h)) = make_uint2(blockIdx.x, run.runs);

    // Column n: token n / heads at position at_n (none: sees no key), query head n % heads.
    const bool col = n < a.cols;
    const uint32_t tok = col ? n / a.heads : 0u;
    const uint32_t head = h * a.heads + (col ? n - tok * a.heads : 0u);
    const bool placed = col && L + tok >= a.tokens;
    const uint32_t past = placed ? L + tok - a.tokens + 1 : 0u;  // keys up to the token's own
    const uint32_t low = a.window != 0 && past > a.window ? past - a.window : 0u;

    // Query fragments (B operand): lane (g4, n) holds dims 32 blk + 8 g4 .. + 7 of column n.
    half8 qf[NB];
    half8 ql[QF32 ? NB : 1];
    {
        const size_t row = ((static_cast<size_t>(b) * a.tokens + tok) * a.q_heads + head) * D + 8 * g4;
#pragma unroll
        for (uint32_t blk = 0; blk < NB; ++blk) {
            if constexpr (QF32) {
                const float* p = static_cast<const float*>(a.q) + row + 32 * blk;
                const float4 x0 = *reinterpret_cast<const float4*>(p), x1 = *reinterpret_cast<const float4*>(p + 4);
                const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    qf[blk][i] = static_cast<_Float16>(x[i]);
                    ql[blk][i] = static_cast<_Float16>(x[i] - static_cast<float>(qf[blk][i]));
                }
            } else {
                qf[blk] = *reinterpret_cast<const half8*>(static_cast<const _Float16*>(a.q) + row + 32 * blk);
            }
        }
    }

    // Registers of one step.  K's are loaded again for the next step as soon as the scores
    // have read them, V's after the values: half a step is always in flight, and no second
    // set of registers is held.
    uint4 kreg[2][NC][KF16 ? 2 : 1];
    typename std::conditional<VF16, uint4, uint2>::type vreg[NM];
    ScaleVec ksc{}, vsc{};
    constexpr uint32_t KE = KF16 ? 2 : 1, VE = VF16 ? 2 : 1;
    auto row_at = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t tok0 = vis.step(i) * kChunk;
        uint32_t page = 0, tp = tok0;
        if (geo.layout == MIIKV_LAYOUT_PAGED) {
            const uint32_t e = tok0 / geo.page_tokens;
            tp = tok0 - e * geo.page_tokens;
            page = min(static_cast<uint32_t>(scalar_load(geo.table + static_cast<size_t>(b) * geo.table_stride + e)),
                       geo.num_pages - 1);
        }
        return (static_cast<size_t>(page) * geo.kv_heads + h) * geo.page_tokens + tp;
    };
    auto load_k = [&](size_t row) __attribute__((always_inline)) {
        const int8_t* kb = geo.k_codes + row * (D * KE);
        if constexpr (!KF16) ksc = *reinterpret_cast<const ScaleVec*>(geo.k_scales + row * NB + lane * (NB / 2));
#pragma unroll
        for (uint32_t J = 0; J < 2; ++J)
#pragma unroll
            for (uint32_t c = 0; c < NC; ++c)
#pragma unroll
                for (uint32_t e = 0; e < KE; ++e)
                    kreg[J][c][e] = stream16(kb + KE * (J * 16 * D + c * 1024 + g4 * 256 + n * 16) + 16 * e);
    };
    auto load_v = [&](size_t row) __attribute__((always_inline)) {
        const int8_t* vb = geo.v_codes + row * (D * VE);
        if constexpr (!VF16) vsc = *reinterpret_cast<const ScaleVec*>(geo.v_scales + row * NB + lane * (NB / 2));
#pragma unroll
        for (uint32_t mt = 0; mt < NM; ++mt) {
            if constexpr (VF16) vreg[mt] = stream16(vb + 2 * ((16 * mt + n) * 32 + g4 * 8));
            else vreg[mt] = stream8(vb + (16 * mt + n) * 32 + g4 * 8);
        }
    };

    // p = 2^(s - ref); ref is `shift` below the column's running maximum.
    float ref = -INFINITY, l_run = 0.0f;
    int shift = VF16 ? 14 : kMaxShift;
    bool fresh = true;  // no key seen by this wave yet
    float4v O[NM];
#pragma unroll
    for (uint32_t mt = 0; mt < NM; ++mt) O[mt] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    uint16_t* s_sc = reinterpret_cast<uint16_t*>(smem) + wave * (2 * kChunk * NB);
    const size_t pair = static_cast<size_t>(b) * geo.kv_heads + h;

    uint32_t i = from + wave;
    size_t row = 0;
    if (i < to) {
        row = row_at(i);
        load_k(row);
        load_v(row);
    }
    for (; i < to; i += kWaves) {
        const uint32_t tok0 = vis.step(i) * kChunk;
        const bool next = i + kWaves < to;
        if (next) row = row_at(i + kWaves);
        // Every column sees every key of the step, or there is something to mask.
        const bool whole = tok0 + kChunk + a.tokens <= L + 1 &&
                           (a.window == 0 || tok0 + kChunk <= a.sinks || tok0 + a.window >= L);
        asm volatile("" ::: "memory");  // the previous step's reads of the scales stay before it
        if constexpr (!KF16) *reinterpret_cast<ScaleVec*>(s_sc + lane * (NB / 2)) = ksc;
        asm volatile("" ::: "memory");
        // Scores S^T[key][column], one MFMA per 32-value block and its scale in fp32.
        float s[2][4];
#pragma unroll
        for (uint32_t J = 0; J < 2; ++J) {
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (KF16) {
                float4v c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t blk = 0; blk < NB; ++blk) {
                    const half8 k = __builtin_bit_cast(half8, kreg[J][blk / 2][KF16 ? blk % 2 : 0]);
                    c = mfma_16x16x32(k, qf[blk], c);
                    if constexpr (QF32) c = mfma_16x16x32(k, ql[QF32 ? blk : 0], c);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = c[k];
            } else {
                uint4 w[NB / 2];  // scales of keys 16 J + 4 g4 + k, all blocks
#pragma unroll
                for (uint32_t x = 0; x < NB / 2; ++x)
                    w[x] = *reinterpret_cast<const uint4*>(s_sc + (16 * J + 4 * g4) * NB + 8 * x);
                const uint16_t* sc = reinterpret_cast<const uint16_t*>(&w[0]);
#pragma unroll
                for (uint32_t blk = 0; blk < NB; ++blk) {
                    const uint4 kw = kreg[J][blk / 2][0];
                    const half8 k = blk % 2 == 0 ? codes8_to_half8(kw.x, kw.y) : codes8_to_half8(kw.z, kw.w);
                    float4v c = mfma_16x16x32(k, qf[blk], float4v{0.0f, 0.0f, 0.0f, 0.0f});
                    if constexpr (QF32) c = mfma_16x16x32(k, ql[QF32 ? blk : 0], c);
#pragma unroll
                    for (int x = 0; x < 4; ++x) acc[x] = fmaf(c[x], f16_bits_to_f32(sc[x * NB + blk]), acc[x]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) s[J][k] = acc[k] * a.scale_log2;
        }
        if (!whole) {
#pragma unroll
            for (uint32_t J = 0; J < 2; ++J)
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t t = tok0 + 16 * J + 4 * g4 + k;
                    if (t >= past || (t < low && t >= a.sinks)) s[J][k] = -INFINITY;
                }
        }
        if constexpr (SCORED) {
            if (col) {
                float* to = a.logits + (pair * a.cols + n) * a.logit_keys + tok0 + 4 * g4;
#pragma unroll
                for (uint32_t J = 0; J < 2; ++J)
                    *reinterpret_cast<float4*>(to + 16 * J) = make_float4(s[J][0], s[J][1], s[J][2], s[J][3]);
            }
        }
        if (next) load_k(row);
        // V's scales: those of keys that no column sees may hold anything, non-finite values
        // too; the largest of the others bounds `shift`.
        if constexpr (!VF16) {
            ScaleVec x = vsc;
            if (!whole) {
                const uint32_t t = tok0 + lane / 2;
                if (t >= L || (t < vis.lo && t >= a.sinks)) x = ScaleVec{};
            }
            asm volatile("" ::: "memory");
            *reinterpret_cast<ScaleVec*>(s_sc + kChunk * NB + lane * (NB / 2)) = x;
            asm volatile("" ::: "memory");
            // positive fp16 numbers are ordered as their bits (a sign counts as large)
            const uint32_t* xw = reinterpret_cast<const uint32_t*>(&x);
            uint32_t bits = 0;
#pragma unroll
            for (uint32_t w = 0; w < NB / 4; ++w) bits = max(bits, max(xw[w] & 0xffffu, xw[w] >> 16));
            // a scale of exponent field f is below 2^(f - 14)
            if (__any(static_cast<int>(bits >> 10) - 14 + shift > 15)) {
                uint32_t top = bits;
#pragma unroll
                for (uint32_t off = 1; off < 64; off <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), off, 64)));
                const int fits = max(kMinShift, 15 + 14 - static_cast<int>(__builtin_amdgcn_readfirstlane(top) >> 10));
                if (fits < shift) {
                    const float f = exp2_fast(static_cast<float>(fits - shift));
                    ref += static_cast<float>(shift - fits);
                    shift = fits;
                    if (!fresh) {
                        l_run *= f;
#pragma unroll
                        for (uint32_t mt = 0; mt < NM; ++mt) O[mt] *= f;
                    }
                }
            }
        }
        // Online softmax: the running maximum, rescaled where it grows.
        float top = s[0][0];
#pragma unroll
        for (uint32_t J = 0; J < 2; ++J)
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) top = fmaxf(top, s[J][k]);
        top = rows_reduce(top, MaxOp{}) - static_cast<float>(shift);
        if (__any(top > ref)) {
            const float to_ref = fmaxf(ref, top);
            if (!fresh) {
                const float f = ref == -INFINITY ? 0.0f : exp2_fast(ref - to_ref);
                l_run *= f;
#pragma unroll
                for (uint32_t mt = 0; mt < NM; ++mt) O[mt] *= f;
            }
            ref = to_ref;
        }
        fresh = false;
        const float use = ref == -INFINITY ? 0.0f : ref;  // a column that saw no key yet
        float p[8];
#pragma unroll
        for (uint32_t x = 0; x < 8; ++x) {
            p[x] = exp2_fast(s[x / 4][x % 4] - use);
            l_run += p[x];
        }
        // O^T += V^T P^T; element 8 g4 + x of the MFMA's K axis is key 16 (x / 4) + 4 g4 + x % 4,
        // the order of V's bytes.
        if constexpr (VF16) {
            half8 hi, lo;
#pragma unroll
            for (uint32_t x = 0; x < 8; ++x) {
                hi[x] = static_cast<_Float16>(p[x]);
                lo[x] = static_cast<_Float16>(p[x] - static_cast<float>(hi[x]));
            }
#pragma unroll
            for (uint32_t mt = 0; mt < NM; ++mt) {
                half8 v = __builtin_bit_cast(half8, vreg[mt]);
                if (!whole) {
#pragma unroll
                    for (uint32_t x = 0; x < 8; ++x) {
                        const uint32_t t = tok0 + 16 * (x / 4) + 4 * g4 + x % 4;
                        if (t >= L || (t < vis.lo && t >= a.sinks)) v[x] = static_cast<_Float16>(0.0f);
                    }
                }
                O[mt] = mfma_16x16x32(v, hi, O[mt]);
                O[mt] = mfma_16x16x32(v, lo, O[mt]);
            }
        } else {
            uint4 w[2][NB / 2];
#pragma unroll
            for (uint32_t J = 0; J < 2; ++J)
#pragma unroll
                for (uint32_t x = 0; x < NB / 2; ++x)
                    w[J][x] = *reinterpret_cast<const uint4*>(s_sc + kChunk * NB + (16 * J + 4 * g4) * NB + 8 * x);
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(&w[0][0]);
#pragma unroll
            for (uint32_t blk = 0; blk < NB; ++blk) {
                half8 hi, lo;
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x) {
                    float ps = p[x] * f16_bits_to_f32(sc[(x / 4) * 4 * NB + (x % 4) * NB + blk]);
                    // both parts come from the rounded product: hi taken from the exact one (a
                    // fused multiply and conversion) now and then rounds the other way, and lo
                    // does not make up for it (outputs 5e-6 off)
                    asm("" : "+v"(ps));
                    hi[x] = static_cast<_Float16>(ps);
                    lo[x] = static_cast<_Float16>(ps - static_cast<float>(hi[x]));
                }
#pragma unroll
                for (uint32_t mt = 2 * blk; mt < 2 * blk + 2; ++mt) {
                    const uint2 vw = __builtin_bit_cast(uint2, vreg[mt]);
                    const half8 v = codes8_to_half8(vw.x, vw.y);
                    O[mt] = mfma_16x16x32(v, hi, O[mt]);
                    O[mt] = mfma_16x16x32(v, lo, O[mt]);
                }
            }
        }
        if (next) load_v(row);
    }
    l_run = rows_reduce(l_run, AddOp{});

    // Merge of the four waves: O^T of column n, dims 16 mt + 4 g4 + i.
    __syncthreads();  // the scales' LDS is reused
    float* s_m = smem;                 // [kWaves][16]
    float* s_l = smem + kWaves * 16;   // [kWaves][16]
    float* s_o = smem + kWaves * 32;   // [kWaves][cols][D]
    if (col) {
        if (g4 == 0) {
            s_m[wave * 16 + n] = ref;
            s_l[wave * 16 + n] = l_run;
        }
#pragma unroll
        for (uint32_t mt = 0; mt < NM; ++mt)
            *reinterpret_cast<float4*>(s_o + (static_cast<size_t>(wave) * a.cols + n) * D + 16 * mt + 4 * g4) =
                make_float4(O[mt][0], O[mt][1], O[mt][2], O[mt][3]);
    }
    __syncthreads();
    float* rec = a.part + static_cast<size_t>(blockIdx.x) * part_record(a.cols, D);
    for (uint32_t e4 = threadIdx.x; e4 < a.cols * D / 4; e4 += 64 * kWaves) {
        const uint32_t c = 4 * e4 / D;
        float m = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) m = fmaxf(m, s_m[w * 16 + c]);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            const float mw = s_m[w * 16 + c];
            const float f = mw == -INFINITY ? 0.0f : exp2_fast(mw - m);
            const float4 o = *reinterpret_cast<const float4*>(s_o + static_cast<size_t>(w) * a.cols * D + 4 * e4);
            l += s_l[w * 16 + c] * f;
            acc.x += o.x * f;
            acc.y += o.y * f;
            acc.z += o.z * f;
            acc.w += o.w * f;
        }
        *reinterpret_cast<float4*>(rec + 4 * e4) = acc;
        if (4 * e4 % D == 0) {
            rec[a.cols * D + c] = m;
            rec[a.cols * D + a.cols + c] = l;
        }
    }
}

// Merge of (b, h)'s records, 32 outputs of one column per wave: lane (rg = lane / 8, q = lane
// % 8) folds records rg, rg + 8, .. for outputs 4q .. 4q + 3, then the 8 groups meet in a
// fixed butterfly.  Up to kAhead records of a lane are read at once.
constexpr uint32_t kAhead = 8;
template <uint32_t D>
__device__ void merge_records(const PartArgs& a) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t blocks = a.cols * D / 32;
    const uint32_t x = blockIdx.x * kWaves + (threadIdx.x >> 6);
    const uint32_t bh = x / blocks;
    if (bh >= a.batch * a.g.kv_heads) return;  // wave-uniform
    const uint32_t b = bh / a.g.kv_heads, h = bh % a.g.kv_heads;
    const uint32_t q = lane & 7, rg = lane >> 3;
    const uint32_t e = (x % blocks) * 32 + 4 * q, c = e / D;
    const uint32_t tok = c / a.heads, head = h * a.heads + c % a.heads;
    const size_t at = ((static_cast<size_t>(b) * a.tokens + tok) * a.q_heads + head) * D + e % D;
    float4 gv = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.gate != nullptr) gv = *reinterpret_cast<const float4*>(a.gate + at);
    uint32_t first, runs;
    find_records(a, bh, b, first, runs);
    const uint32_t rec = part_record(a.cols, D);
    const float* base = a.part + static_cast<size_t>(first) * rec;
    float m = -INFINITY, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto fold = [&](float m2, float l2, float4 o) {
        const float mn = fmaxf(m, m2);
        const float f1 = m == -INFINITY ? 0.0f : exp2_fast(m - mn), f2 = m2 == -INFINITY ? 0.0f : exp2_fast(m2 - mn);
        m = mn;
        l = l * f1 + l2 * f2;
        acc.x = acc.x * f1 + o.x * f2;
        acc.y = acc.y * f1 + o.y * f2;
        acc.z = acc.z * f1 + o.z * f2;
        acc.w = acc.w * f1 + o.w * f2;
    };
    for (uint32_t r0 = rg; r0 < runs; r0 += 8 * kAhead) {
        float ms[kAhead], ls[kAhead];
        float4 os[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            ms[j] = -INFINITY;
            ls[j] = 0.0f;
            os[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r0 + 8 * j < runs) {
                const float* r = base + static_cast<size_t>(r0 + 8 * j) * rec;
                ms[j] = r[a.cols * D + c];
                ls[j] = r[a.cols * D + a.cols + c];
                os[j] = *reinterpret_cast<const float4*>(r + e);
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) fold(ms[j], ls[j], os[j]);
    }
#pragma unroll
    for (uint32_t off = 8; off < 64; off <<= 1) {
        const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
        const float4 o = make_float4(__shfl_xor(acc.x, off), __shfl_xor(acc.y, off), __shfl_xor(acc.z, off), __shfl_xor(acc.w, off));
        fold(m2, l2, o);
    }
    if (rg != 0) return;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;  // a token that sees no key: zeros
    const float4 o = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (a.out != nullptr) *reinterpret_cast<float4*>(a.out + at) = o;
    if (a.gated_out != nullptr)
        *reinterpret_cast<float4*>(a.gated_out + at) =
            make_float4(o.x / (1.0f + expf(-gv.x)), o.y / (1.0f + expf(-gv.y)), o.z / (1.0f + expf(-gv.z)), o.w / (1.0f + expf(-gv.w)));
}

// Weights of kWeightKeys keys of one (b, h): the columns' merged m and l from the records,
// then each key's probabilities from its scores, added in column order.
template <uint32_t D>
__device__ void add_weights(const PartArgs& a, uint32_t x) {
    const uint32_t blocks = (a.max_context + kWeightKeys - 1) / kWeightKeys;
    const uint32_t bh = x / blocks, key = (x % blocks) * kWeightKeys + threadIdx.x;
    const uint32_t b = bh / a.g.kv_heads;
    const uint32_t L = part_length(a, b);
    if ((x % blocks) * kWeightKeys >= L) return;  // workgroup-uniform
    // the scores go out ahead of the records
    float s[16];
    const bool live = key < L;
    const float* row = a.logits + static_cast<size_t>(bh) * a.cols * a.logit_keys + (live ? key : 0u);
#pragma unroll
    for (uint32_t c = 0; c < 16; ++c) s[c] = c < a.cols ? row[static_cast<size_t>(c) * a.logit_keys] : -INFINITY;
    float* to = a.weights + static_cast<size_t>(bh) * a.weight_stride + (live ? key : 0u);
    const float before = *to;
    // Thread (rg, c) folds records rg, rg + 16, ..; then the four of a wave meet in a fixed butterfly, and the waves.
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    const uint32_t c = threadIdx.x & 15, rg = threadIdx.x >> 4;
    uint32_t first, runs;
    find_records(a, bh, b, first, runs);
    const uint32_t rec = part_record(a.cols, D);
    float m = -INFINITY, l = 0.0f;
    auto fold = [](float& m1, float& l1, float m2, float l2) {
        const float mn = fmaxf(m1, m2);
        l1 = l1 * (m1 == -INFINITY ? 0.0f : exp2_fast(m1 - mn)) + l2 * (m2 == -INFINITY ? 0.0f : exp2_fast(m2 - mn));
        m1 = mn;
    };
    constexpr uint32_t kDepth = 4;  // records read at a time
    if (c < a.cols)
        for (uint32_t r = rg; r < runs; r += 16 * kDepth) {
            float ms[kDepth], ls[kDepth];
#pragma unroll
            for (uint32_t j = 0; j < kDepth; ++j) {
                const float* p = a.part + static_cast<size_t>(first + min(r + 16 * j, runs - 1)) * rec + a.cols * D;
                ms[j] = p[c];
                ls[j] = p[a.cols + c];
            }
#pragma unroll
            for (uint32_t j = 0; j < kDepth; ++j)
                if (r + 16 * j < runs) fold(m, l, ms[j], ls[j]);
        }
#pragma unroll
    for (uint32_t off = 16; off < 64; off <<= 1) {
        const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
        fold(m, l, m2, l2);
    }
    if (threadIdx.x % 64 < 16) {
        s_m[threadIdx.x / 64][c] = m;
        s_l[threadIdx.x / 64][c] = l;
    }
    __syncthreads();
    __shared__ float s_ref[16], s_inv[16];
    if (threadIdx.x < 16) {
#pragma unroll
        for (uint32_t w = 1; w < kWaves; ++w) fold(m, l, s_m[w][c], s_l[w][c]);
        s_ref[c] = m == -INFINITY ? 0.0f : m;
        s_inv[c] = l > 0.0f ? 1.0f / l : 0.0f;
    }
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < 16; ++k)
        if (k < a.cols) sum += exp2_fast(s[k] - s_ref[k]) * s_inv[k];
    if (live) *to = before + sum;
}

template <uint32_t D, bool SCORED>
__global__ void __launch_bounds__(256) part_finish_kernel(PartArgs a) {
    if constexpr (SCORED) {
        if (blockIdx.x >= a.combine_wgs) {
            add_weights<D>(a, blockIdx.x - a.combine_wgs);
            return;
        }
    }
    merge_records<D>(a);
}

struct PartPlan {
    uint64_t run_bytes;
    uint64_t wgs;        // of the first launch: an upper bound on the runs
    uint64_t part_bytes;
    uint64_t logit_bytes;
    uint32_t logit_keys;
};

uint64_t up256(uint64_t x) { return (x + 255) / 256 * 256; }

PartPlan part_plan(const miikv_view* v, uint32_t q_heads, uint32_t batch, uint32_t tokens, uint32_t max_context,
                   uint32_t window, uint32_t sinks, bool scored) {
    PartPlan p{};
    const uint64_t pairs = static_cast<uint64_t>(batch) * v->kv_heads;
    const uint64_t most = most_visible_steps(max_context, tokens, window, sinks);
    // the runs: at most the slots and one partial run per pair, or one step per wave
    p.wgs = std::min<uint64_t>(kTargetWgs + pairs, pairs * ((most + kWaves - 1) / kWaves));
    const uint32_t cols = q_heads / v->kv_heads * tokens;
    p.run_bytes = up256(pairs * 2 * sizeof(uint32_t));
    p.part_bytes = up256(p.wgs * part_record(cols, v->head_dim) * sizeof(float));
    p.logit_keys = (max_context + kChunk - 1) / kChunk * kChunk;
    p.logit_bytes = scored ? up256(pairs * cols * p.logit_keys * sizeof(float)) : 0u;
    return p;
}

// Whether the sizes are ones that the kernels serve: a status.
int part_sizes(const miikv_view* v, uint32_t q_heads, uint32_t batch, uint32_t tokens, uint32_t max_context) {
    const int st = validate_view(v);
    if (st != MIIKV_OK) return st;
    if (batch == 0 || tokens == 0 || q_heads == 0 || q_heads % v->kv_heads != 0) return MIIKV_EINVAL;
    if (static_cast<uint64_t>(q_heads / v->kv_heads) * tokens > 16) return MIIKV_EUNSUPPORTED;
    if (max_context == 0 || max_context > view_seq_capacity(v) || max_context > 0x7fffffffu) return MIIKV_EINVAL;
    if (v->layout == MIIKV_LAYOUT_CONTIGUOUS && batch != 1) return MIIKV_EINVAL;
    if (batch > 65535u || static_cast<uint64_t>(batch) * v->kv_heads > 0xfffffu) return MIIKV_EINVAL;
    return MIIKV_OK;
}

template <uint32_t D, bool SCORED>
void launch_part(const PartArgs& a, bool qf32, bool kf, bool vf, dim3 grid, dim3 finish, size_t lds, hipStream_t s) {
    const auto go = [&](auto f, auto k, auto v) {
        hipLaunchKernelGGL((part_kernel<D, decltype(f)::value, decltype(k)::value, decltype(v)::value, SCORED>), grid,
                           dim3(64 * kWaves), lds, s, a);
    };
    const auto with_v = [&](auto f, auto k) { vf ? go(f, k, std::true_type{}) : go(f, k, std::false_type{}); };
    const auto with_k = [&](auto f) { kf ? with_v(f, std::true_type{}) : with_v(f, std::false_type{}); };
    qf32 ? with_k(std::true_type{}) : with_k(std::false_type{});
    hipLaunchKernelGGL((part_finish_kernel<D, SCORED>), finish, dim3(256), 0, s, a);
}

miikv_status part_impl(const miikv_view* view, const void* q, uint32_t q_dtype, uint32_t q_heads, float scale,
                       uint32_t batch, uint32_t tokens, const uint32_t* d_lengths, const miikv_decode_state* state,
                       uint32_t max_context, uint32_t window, uint32_t sinks, float* weights, uint64_t weight_stride,
                       bool scored, float* out, const float* gate, float* gated_out, void* workspace,
                       uint64_t workspace_bytes, void* stream) {
    const int st = part_sizes(view, q_heads, batch, tokens, max_context);
    if (st != MIIKV_OK) return st;
    if (q == nullptr || !std::isfinite(scale) || (q_dtype != MIIKV_DTYPE_F16 && q_dtype != MIIKV_DTYPE_F32))
        return MIIKV_EINVAL;
    if (d_lengths == nullptr && (state == nullptr || batch != 1)) return MIIKV_EINVAL;
    if (out == nullptr && gated_out == nullptr) return MIIKV_EINVAL;
    if ((gate == nullptr) != (gated_out == nullptr)) return MIIKV_EINVAL;
    if (scored && (weights == nullptr || weight_stride < max_context)) return MIIKV_EINVAL;
    if (!aligned16(q) || !aligned16(out) || !aligned16(gate) || !aligned16(gated_out) || !aligned16(workspace) ||
        !aligned16(view->k_codes) || !aligned16(view->v_codes) || !aligned16(view->k_scales) || !aligned16(view->v_scales))
        return MIIKV_EINVAL;
    if (window >= max_context) window = 0;  // hides nothing
    sinks = std::min(sinks, max_context);
    const PartPlan p = part_plan(view, q_heads, batch, tokens, max_context, window, sinks, scored);
    if (workspace == nullptr || workspace_bytes < p.run_bytes + p.part_bytes + p.logit_bytes) return MIIKV_EWORKSPACE;

    PartArgs a{};
    a.g = make_geo(*view);
    a.q = q;
    a.q_heads = q_heads;
    a.heads = q_heads / view->kv_heads;
    a.tokens = tokens;
    a.cols = a.heads * tokens;
    a.scale_log2 = scale * kLog2eF;
    a.len_ptr = d_lengths != nullptr ? d_lengths : &state->position;
    a.len_stride = d_lengths != nullptr ? 1u : 0u;
    a.len_add = d_lengths != nullptr ? 0u : 1u;
    a.max_context = max_context;
    a.window = window;
    a.sinks = sinks;
    a.batch = batch;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.runs = reinterpret_cast<uint32_t*>(ws);
    a.part = reinterpret_cast<float*>(ws + p.run_bytes);
    a.logits = reinterpret_cast<float*>(ws + p.run_bytes + p.part_bytes);
    a.logit_keys = p.logit_keys;
    a.weights = weights;
    a.weight_stride = weight_stride;
    a.out = out;
    a.gate = gate;
    a.gated_out = gated_out;
    const uint32_t D = view->head_dim;
    const uint64_t pairs = static_cast<uint64_t>(batch) * view->kv_heads;
    const uint64_t waves = pairs * (a.cols * D / 32);
    a.combine_wgs = static_cast<uint32_t>((waves + kWaves - 1) / kWaves);
    const uint64_t finish = a.combine_wgs + (scored ? pairs * ((max_context + kWeightKeys - 1) / kWeightKeys) : 0u);
    if (p.wgs > 0x7fffffffu || finish > 0x7fffffffu) return MIIKV_EINVAL;
    const size_t lds = std::max<size_t>((kWaves * 32 + static_cast<size_t>(kWaves) * a.cols * D) * sizeof(float),
                                        kWaves * 2 * kChunk * (D / 32) * sizeof(uint16_t));
    const bool f32 = q_dtype == MIIKV_DTYPE_F32, kf = mode_k_f16(view->quant_mode), vf = mode_v_f16(view->quant_mode);
    const dim3 grid(static_cast<uint32_t>(p.wgs)), fin(static_cast<uint32_t>(finish));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const auto with_dim = [&](auto sc) {
        constexpr bool SC = decltype(sc)::value;
        if (D == 128) launch_part<128, SC>(a, f32, kf, vf, grid, fin, lds, s);
        else launch_part<256, SC>(a, f32, kf, vf, grid, fin, lds, s);
    };
    if (scored) with_dim(std::true_type{});
    else with_dim(std::false_type{});
    return hip_status(hipGetLastError());
}

}  // namespace
}  // namespace miikv

using namespace miikv;

extern "C" uint64_t miikv_window_workspace_bytes(const miikv_view* view, uint32_t q_heads, uint32_t batch, uint32_t tokens,
                                                 uint32_t max_context, uint32_t window, uint32_t sinks) {
    if (part_sizes(view, q_heads, batch, tokens, max_context) != MIIKV_OK) return 0;
    if (window >= max_context) window = 0;
    const PartPlan p = part_plan(view, q_heads, batch, tokens, max_context, window, std::min(sinks, max_context), false);
    return p.run_bytes + p.part_bytes;
}

extern "C" miikv_status miikv_decode_attn_window(const miikv_view* view, const void* q, uint32_t q_dtype, uint32_t q_heads,
                                                 float scale, uint32_t batch, uint32_t tokens, const uint32_t* d_lengths,
                                                 const miikv_decode_state* decode_state, uint32_t max_context,
                                                 uint32_t window, uint32_t sinks, float* out, const float* gate,
                                                 float* gated_out, void* workspace, uint64_t workspace_bytes,
                                                 void* stream) {
    return part_impl(view, q, q_dtype, q_heads, scale, batch, tokens, d_lengths, decode_state, max_context, window, sinks,
                     nullptr, 0, false, out, gate, gated_out, workspace, workspace_bytes, stream);
}

extern "C" uint64_t miikv_scored_workspace_bytes(const miikv_view* view, uint32_t q_heads, uint32_t batch, uint32_t tokens,
                                                 uint32_t max_context) {
    if (part_sizes(view, q_heads, batch, tokens, max_context) != MIIKV_OK) return 0;
    const PartPlan p = part_plan(view, q_heads, batch, tokens, max_context, 0, 0, true);
    return p.run_bytes + p.part_bytes + p.logit_bytes;
}

extern "C" miikv_status miikv_decode_attn_scored(const miikv_view* view, const void* q, uint32_t q_dtype, uint32_t q_heads,
                                                 float scale, uint32_t batch, uint32_t tokens, const uint32_t* d_lengths,
                                                 const miikv_decode_state* decode_state, uint32_t max_context,
                                                 float* key_weights, uint64_t weight_stride, float* out, const float* gate,
                                                 float* gated_out, void* workspace, uint64_t workspace_bytes,
                                                 void* stream) {
    return part_impl(view, q, q_dtype, q_heads, scale, batch, tokens, d_lengths, decode_state, max_context, 0, 0,
                     key_weights, weight_stride, true, out, gate, gated_out, workspace, workspace_bytes, stream);
}
