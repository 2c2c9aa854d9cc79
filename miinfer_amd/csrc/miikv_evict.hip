// Eviction: of every (sequence, kv head) the keys with the largest accumulated weight stay,
// and their rows move together (gfx950).
//
// With L keys, a budget of n and L > n: the first `sinks` and the last `recent` keys stay,
// and of those between the n - sinks - recent with the largest weights; of equal weights
// the first ones.  Kept key i of the ascending list moves to position i.
//
// select_kernel finds the list: the weight that is just kept by a radix select over the
// weights' ordered bits (four digits of 8 bits, counts in LDS), then each wave's place in
// the list from counts of its own stretch of keys.  It also moves the weights.
// move_kernel moves the rows: codes are copied as they are, nothing is quantised again.
//
// In place, position i's source is at or behind i, so rows that go forward in order never
// overwrite one that is still to move: a workgroup owns a slice of every row (some bytes of
// each token, which no other workgroup touches), reads kMoveInPlace tokens, waits until all of
// them have arrived, and writes them.  To other pages every tile is independent.
//
// Bound: the cache's lines that hold a kept row.  A K line of 128 bytes holds 8 tokens'
// runs of 16 bytes and a V line 4 dims of 32 tokens, so where one key in eight stays nearly
// all lines of the old context are read (16384 keys of 8 heads to 4096, head_dim 128: 9.4 us for 45 MB;
// 12 sequences to 2048, head_dim 256: 40 us for 171 MB).  Of V a thread gathers single bytes.
#include "miikv_part.hpp"

#include <type_traits>

namespace miikv {
namespace {

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kSelectWaves = kSelectThreads / 64;
constexpr uint32_t kCopies = 16;  // histograms, one per lane % 16: weights share their top digits
constexpr uint32_t kCopyStride = kCopies + 1;  // words from a digit's counts to the next one's; odd, for the sums' reads
constexpr uint32_t kMoveTokens = 256;    // destination tokens moved at a time, to other pages
// In place, one turn after another.  (16384 keys of 8 heads to 4096, select and move: 256 at a time in slices of two
// runs and 32 dims 54.5 us; 1024 at a time 36.7; and slices of one run and 8 dims 23.3.)
constexpr uint32_t kMoveInPlace = 1024;

struct EvictArgs {
    Geo g;
    const int32_t* dst_table;  // null: in place
    uint32_t dst_stride;
    const float* weights;
    uint64_t weight_stride;
    float* weights_out;  // nullable
    uint64_t weight_out_stride;
    const uint32_t* lengths;
    uint32_t* new_lengths;
    int32_t* kept;
    uint32_t batch;
    uint32_t max_context;
    uint32_t sinks, recent, budget;
};

__device__ __forceinline__ uint32_t evict_length(const EvictArgs& a, uint32_t b) { return min(a.lengths[b], a.max_context); }

// Set bits of `mask` below this lane.
__device__ __forceinline__ uint32_t lanes_before(unsigned long long mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0u));
}

// Weights in the order of unsigned numbers; a NaN counts as less than any number.
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);  // -0 equals 0
    return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

// One workgroup of a (sequence, kv head).  Its keys lie in registers, kPer of each thread, a wave's
// kPer * 64 one behind another: a context of up to kSegment keys between the first and the last ones
// is read once, a longer one segment by segment in every pass.  Places behind the context count as
// key 0, the least there is: they come last of all and more keys than stay are real, so none is chosen.
//
// Bound: instructions of one compute unit, 256 cycles for each one that every key of 16384 needs,
// and the latency of the two reads and the barriers.  (For 16384 keys of 8 heads: the weights read anew
// in every pass, one at a time, 31.4 us; held in registers 19; a wave's keys one
// behind another, weights moved from registers 12.8; passes left out where all that share the digits stay 12.1.)
constexpr uint32_t kPer = 16;
constexpr uint32_t kSegment = kPer * kSelectThreads;

__device__ __forceinline__ void load_weights(const float* w, uint32_t first, uint32_t hi, float (&x)[kPer], uint32_t (&key)[kPer]) {
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) x[j] = w[min(first + j * 64, hi - 1)];
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) key[j] = first + j * 64 < hi ? ordered(x[j]) : 0u;
}

__global__ void __launch_bounds__(kSelectThreads) select_kernel(EvictArgs a) {
    const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t L = evict_length(a, b), n = a.budget;
    const size_t row = static_cast<size_t>(b) * a.g.kv_heads + h;
    const float* w = a.weights + row * a.weight_stride;
    float* out = a.weights_out == nullptr ? nullptr : a.weights_out + row * a.weight_out_stride;
    const bool moves = out != nullptr, same_row = out == w;
    int32_t* kept = a.kept + row * n;
    if (L <= n) {
        for (uint32_t i = tid; i < n; i += kSelectThreads) kept[i] = i < L ? static_cast<int32_t>(i) : -1;
        if (moves && !same_row)
            for (uint32_t i = tid; i < L; i += kSelectThreads) out[i] = w[i];
        return;
    }
    __shared__ uint32_t s_hist[4][256 * kCopyStride];  // [pass][digit][copy]: equal digits of a wave on kCopies banks
    __shared__ uint32_t s_count[4][256];
    __shared__ uint2 s_total[2][kSelectWaves];  // keys above and at the limit, of a wave; segments in turn
    const uint32_t lo = a.sinks, hi = L - a.recent, need = n - a.sinks - a.recent;
    for (uint32_t i = tid; i < a.sinks; i += kSelectThreads) {
        kept[i] = static_cast<int32_t>(i);
        if (moves && !same_row) out[i] = w[i];
    }
    for (uint32_t i = tid; i < a.recent; i += kSelectThreads) kept[n - a.recent + i] = static_cast<int32_t>(hi + i);
    if (need != 0) {  // and then hi - lo > need
        const uint32_t first = lo + wave * (kPer * 64) + lane;
        float x[kPer];
        uint32_t key[kPer];
        const bool once = hi - lo <= kSegment;
        for (uint32_t i = tid; i < 4 * 256 * kCopyStride; i += kSelectThreads) (&s_hist[0][0])[i] = 0;
        load_weights(w, first, hi, x, key);
        __syncthreads();
        uint32_t prefix = 0, k = need, low = 0;  // the limit's digits so far; keys of them that stay; bits not looked at
#pragma unroll
        for (uint32_t pass = 0; pass < 4; ++pass) {
            const uint32_t shift = 24 - 8 * pass;
            uint32_t* const hist = &s_hist[pass][lane % kCopies];
            for (uint32_t from = 0; from < hi - lo; from += kSegment) {
                if (!once) load_weights(w, first + from, hi, x, key);
#pragma unroll
                for (uint32_t j = 0; j < kPer; ++j)
                    if (pass == 0 || key[j] >> ((shift + 8) & 31) == prefix)
                        atomicAdd(hist + ((key[j] >> shift) & 255u) * kCopyStride, 1u);
            }
            __syncthreads();
            if (tid < 256) {
                uint32_t sum = 0;
#pragma unroll
                for (uint32_t c = 0; c < kCopies; ++c) sum += s_hist[pass][tid * kCopyStride + c];
                s_count[pass][tid] = sum;
            }
            __syncthreads();
            // Every wave finds the digit.  Lane l: digits 255 - 4l down to 252 - 4l.
            uint32_t c[4], sum = 0, digit = 0, before = 0, here = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) sum += c[j] = s_count[pass][255 - 4 * lane - j];
            uint32_t above = sum_to_lane(sum) - sum;
            const bool mine = above < k && k <= above + sum;  // of exactly one lane
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                if (above < k) {
                    digit = 255 - 4 * lane - j;
                    before = above;
                    here = c[j];
                }
                above += c[j];
            }
            const uint32_t from_lane = static_cast<uint32_t>(__builtin_ctzll(__ballot(mine)));
            prefix = prefix << 8 | static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(digit), from_lane));
            k -= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before), from_lane));
            // All keys that share these digits stay: the others need not be told apart.
            if (k == static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(here), from_lane))) {
                low = shift;
                break;
            }
        }
        // Keys above `prefix` stay, and the first k of those equal to it.  In place, a weight's new
        // position is at or before its old one, and its segment has been read whole by then.
        uint32_t gt0 = 0, eq0 = 0;  // keys above and equal, of the segments before
        for (uint32_t from = 0, turn = 0; from < hi - lo; from += kSegment, turn ^= 1) {
            if (!once) load_weights(w, first + from, hi, x, key);
            uint32_t gt = 0, eq = 0;
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                gt += static_cast<uint32_t>(__popcll(__ballot((key[j] >> low) > prefix)));
                eq += static_cast<uint32_t>(__popcll(__ballot((key[j] >> low) == prefix)));
            }
            if (lane == 0) s_total[turn][wave] = make_uint2(gt, eq);
            __syncthreads();
            const uint2 mine = s_total[turn][lane % kSelectWaves];
            const uint32_t gi = sum_to_lane(lane < kSelectWaves ? mine.x : 0u), ei = sum_to_lane(lane < kSelectWaves ? mine.y : 0u);
            uint32_t gt_at = gt0 + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(gi), wave)) - gt;
            uint32_t eq_at = eq0 + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ei), wave)) - eq;
            gt0 += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(gi), 63));
            eq0 += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ei), 63));
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                const unsigned long long gts = __ballot((key[j] >> low) > prefix), eqs = __ballot((key[j] >> low) == prefix);
                if ((gts | eqs) != 0) {
                    const uint32_t eq_mine = eq_at + lanes_before(eqs);
                    const uint32_t to = a.sinks + gt_at + lanes_before(gts) + min(eq_mine, k);
                    if ((key[j] >> low) > prefix || ((key[j] >> low) == prefix && eq_mine < k)) {
                        kept[to] = static_cast<int32_t>(first + from + j * 64);
                        if (moves) out[to] = x[j];
                    }
                    gt_at += static_cast<uint32_t>(__popcll(gts));
                    eq_at += static_cast<uint32_t>(__popcll(eqs));
                }
            }
        }
    }
    if (!moves) return;
    // The last keys' weights; in place they go forward in order, all of a turn read before any is written.
    if (same_row) __syncthreads();
    for (uint32_t i0 = 0; i0 < a.recent; i0 += kSelectThreads) {
        const uint32_t i = i0 + tid;
        const float y = i < a.recent ? w[hi + i] : 0.0f;
        if (same_row) {
            wait_vmem();
            __syncthreads();
        }
        if (i < a.recent) out[n - a.recent + i] = y;
    }
    // in place: what stood behind the keys that stay is no weight of the keys to come
    if (same_row)
        for (uint32_t i = n + tid; i < L; i += kSelectThreads) out[i] = 0.0f;
}

typedef unsigned int u4v __attribute__((ext_vector_type(4)));

// Row (page * kv_heads + head) * page_tokens + slot of position `pos`.
__device__ __forceinline__ uint32_t row_of(const Geo& g, const int32_t* table, uint32_t pos, uint32_t h) {
    uint32_t page = 0, tp = pos;
    if (table != nullptr) {
        const uint32_t e = pos / g.page_tokens;
        tp = pos - e * g.page_tokens;
        page = min(static_cast<uint32_t>(table[e]), g.num_pages - 1);
    }
    return (page * g.kv_heads + h) * g.page_tokens + tp;
}

// Roles of a (sequence, kv head)'s workgroups: slices of K (one or two of a token's D / 16 runs of 8 + 8 dims), of
// V (8 or 32 dims), one of the scales.  In place, where a workgroup moves all tokens of its slice, slices are
// the smaller ones.
template <uint32_t D, bool INPLACE>
struct Roles {
    static constexpr uint32_t k_runs = INPLACE ? 1 : 2, v_dims = INPLACE ? 8 : 32;
    static constexpr uint32_t k = D / 16 / k_runs, v = D / v_dims, all = k + v + 1;
};
template <uint32_t D, bool KF16, bool VF16, bool INPLACE>
__global__ void __launch_bounds__(INPLACE ? kMoveInPlace : kMoveTokens) move_kernel(EvictArgs a) {
    constexpr uint32_t NB = D / 32;
    using Role = Roles<D, INPLACE>;
    constexpr uint32_t KE = KF16 ? 2 : 1;
    constexpr uint32_t kTok = INPLACE ? kMoveInPlace : kMoveTokens;
    const uint32_t role = blockIdx.x % Role::all, tile = blockIdx.x / Role::all;
    const uint32_t h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const uint32_t left = min(evict_length(a, b), a.budget);
    if (!INPLACE && tile == 0 && role == 0 && h == 0 && tid == 0) a.new_lengths[b] = left;
    const int32_t* kept = a.kept + (static_cast<size_t>(b) * a.g.kv_heads + h) * a.budget;
    const int32_t* src_table = a.g.layout == MIIKV_LAYOUT_PAGED ? a.g.table + static_cast<size_t>(b) * a.g.table_stride : nullptr;
    const int32_t* dst_table = INPLACE ? src_table : a.dst_table + static_cast<size_t>(b) * a.dst_stride;
    // Two buffers: a wave may write the next tile's rows while another still stores this one's.
    __shared__ uint32_t s_rows[2][2][kTok];
    uint32_t turn = 0;
    for (uint32_t t0 = tile * kTok; t0 < left; t0 += kTok, turn ^= 1) {
        uint32_t *s_src = s_rows[turn][0], *s_dst = s_rows[turn][1];
        const uint32_t i = t0 + tid;
        bool moves = false;
        if (i < left) {
            const uint32_t from = static_cast<uint32_t>(kept[i]);
            moves = !INPLACE || from != i;
            s_src[tid] = row_of(a.g, src_table, from, h);
            s_dst[tid] = row_of(a.g, dst_table, i, h);
        }
        if (!__syncthreads_or(moves) && INPLACE) continue;  // nothing of this tile moves
        const uint32_t count = min(kTok, left - t0);
        if (role < Role::k) {
            // token tid's runs of 16 * KE bytes, k_runs from number role * k_runs on: of chunk c = number / 4, g = number % 4
            u4v r[Role::k_runs][KE];
            const size_t off = static_cast<size_t>(role) * Role::k_runs * 256;
            if (tid < count) {
                const size_t row = s_src[tid];
                const int8_t* p = a.g.k_codes + KE * ((row & ~size_t{15}) * D + off + (row & 15) * 16);
#pragma unroll
                for (uint32_t u = 0; u < Role::k_runs; ++u)
#pragma unroll
                    for (uint32_t e = 0; e < KE; ++e) r[u][e] = *reinterpret_cast<const u4v*>(p + KE * u * 256 + 16 * e);
            }
            if constexpr (INPLACE) {
                wait_vmem();
                __syncthreads();
            }
            if (tid < count) {
                const size_t row = s_dst[tid];
                int8_t* p = a.g.k_codes + KE * ((row & ~size_t{15}) * D + off + (row & 15) * 16);
#pragma unroll
                for (uint32_t u = 0; u < Role::k_runs; ++u)
#pragma unroll
                    for (uint32_t e = 0; e < KE; ++e) *reinterpret_cast<u4v*>(p + KE * u * 256 + 16 * e) = r[u][e];
            }
        } else if (role < Role::k + Role::v) {
            // groups of 32 tokens x v_dims dims x 4 units of 8 tokens (16 (x / 4) + 4 G + x % 4)
            using Elem = typename std::conditional<VF16, uint16_t, uint8_t>::type;
            constexpr uint32_t kPer = VF16 ? 2 : 4;  // elements of a 32-bit word
            const uint32_t d0 = (role - Role::k) * Role::v_dims;
            const Elem* v = reinterpret_cast<const Elem*>(a.g.v_codes);
            constexpr uint32_t kUnits = Role::v_dims / 8;  // per thread
            uint32_t r[kUnits][8 / kPer];
#pragma unroll
            for (uint32_t j = 0; j < kUnits; ++j) {
                const uint32_t x = j * kTok + tid, G = x & 3, d = d0 + x / 4 % Role::v_dims, H = x / (4 * Role::v_dims);
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) {
                    const uint32_t t = min(32 * H + 16 * (k / 4) + 4 * G + k % 4, count - 1);
                    const size_t row = s_src[t];
                    const uint32_t s = static_cast<uint32_t>(row & 31);
                    const uint32_t e = v[(row & ~size_t{31}) * D + d * 32 + ((s >> 2) & 3) * 8 + (s >> 4) * 4 + (s & 3)];
                    if (k % kPer == 0) r[j][k / kPer] = e;
                    else r[j][k / kPer] |= e << (32 / kPer * (k % kPer));
                }
            }
            if constexpr (INPLACE) {
                wait_vmem();
                __syncthreads();
            }
#pragma unroll
            for (uint32_t j = 0; j < kUnits; ++j) {
                const uint32_t x = j * kTok + tid, G = x & 3, d = d0 + x / 4 % Role::v_dims, H = x / (4 * Role::v_dims);
                if (32 * H + 4 * G >= count) continue;
                const size_t row = s_dst[32 * H];  // a group's rows are consecutive
                Elem* to = reinterpret_cast<Elem*>(a.g.v_codes) + row * D + d * 32 + G * 8;
                if (32 * H + 16 + 4 * G + 3 < count) {
                    uint32_t* word = reinterpret_cast<uint32_t*>(to);
#pragma unroll
                    for (uint32_t k = 0; k < 8 / kPer; ++k) word[k] = r[j][k];
                } else {  // the last group: what is behind the kept rows stays as it was
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k)
                        if (32 * H + 16 * (k / 4) + 4 * G + k % 4 < count) to[k] = static_cast<Elem>(r[j][k / kPer] >> (32 / kPer * (k % kPer)));
                }
            }
        } else {
            using ScaleRow = typename std::conditional<NB == 4, uint2, uint4>::type;
            ScaleRow ks{}, vs{};
            if (tid < count) {
                if constexpr (!KF16) ks = *reinterpret_cast<const ScaleRow*>(a.g.k_scales + static_cast<size_t>(s_src[tid]) * NB);
                if constexpr (!VF16) vs = *reinterpret_cast<const ScaleRow*>(a.g.v_scales + static_cast<size_t>(s_src[tid]) * NB);
            }
            if constexpr (INPLACE) {
                wait_vmem();
                __syncthreads();
            }
            if (tid < count) {
                if constexpr (!KF16) *reinterpret_cast<ScaleRow*>(a.g.k_scales + static_cast<size_t>(s_dst[tid]) * NB) = ks;
                if constexpr (!VF16) *reinterpret_cast<ScaleRow*>(a.g.v_scales + static_cast<size_t>(s_dst[tid]) * NB) = vs;
            }
        }
        if constexpr (!INPLACE) break;
    }
    // `new_lengths` may be `lengths`: min(length, budget) is the same of the old and of the new one
    if (INPLACE && role == 0 && h == 0 && tid == 0) a.new_lengths[b] = left;
}

int evict_sizes(const miikv_view* v, uint32_t batch, uint32_t max_context, uint32_t budget) {
    const int st = validate_view(v);
    if (st != MIIKV_OK) return st;
    if (batch == 0 || batch > 65535u || v->kv_heads > 65535u || budget == 0 || budget > 0x7fffffffu) return MIIKV_EINVAL;
    if (max_context == 0 || max_context > view_seq_capacity(v) || max_context > 0x7fffffffu) return MIIKV_EINVAL;
    if (v->layout == MIIKV_LAYOUT_CONTIGUOUS && batch != 1) return MIIKV_EINVAL;
    return MIIKV_OK;
}

template <uint32_t D>
void launch_move(const EvictArgs& a, bool kf, bool vf, hipStream_t s) {
    const uint32_t most = a.max_context < a.budget ? a.max_context : a.budget;
    const uint32_t tiles = a.dst_table != nullptr ? (most + kMoveTokens - 1) / kMoveTokens : 1u;
    const auto go = [&](auto k, auto v, auto in) {
        const dim3 grid(Roles<D, decltype(in)::value>::all * tiles, a.g.kv_heads, a.batch);
        hipLaunchKernelGGL((move_kernel<D, decltype(k)::value, decltype(v)::value, decltype(in)::value>), grid, dim3(decltype(in)::value ? kMoveInPlace : kMoveTokens), 0, s, a);
    };
    const auto with_in = [&](auto k, auto v) { a.dst_table == nullptr ? go(k, v, std::true_type{}) : go(k, v, std::false_type{}); };
    const auto with_v = [&](auto k) { vf ? with_in(k, std::true_type{}) : with_in(k, std::false_type{}); };
    kf ? with_v(std::true_type{}) : with_v(std::false_type{});
}

}  // namespace
}  // namespace miikv

using namespace miikv;

extern "C" miikv_status miikv_evict(const miikv_view* view, const float* key_weights, uint64_t weight_stride,
                                    uint32_t batch, const uint32_t* d_lengths, uint32_t max_context, uint32_t sinks,
                                    uint32_t recent, uint32_t budget, const int32_t* dst_table, uint32_t dst_stride,
                                    int32_t* kept, uint32_t* d_new_lengths, float* weights_out,
                                    uint64_t weights_out_stride, void* stream) {
    const int st = evict_sizes(view, batch, max_context, budget);
    if (st != MIIKV_OK) return st;
    if (key_weights == nullptr || weight_stride < max_context || d_lengths == nullptr || kept == nullptr ||
        d_new_lengths == nullptr)
        return MIIKV_EINVAL;
    if (static_cast<uint64_t>(sinks) + recent > budget) return MIIKV_EINVAL;
    const uint32_t most = max_context < budget ? max_context : budget;
    if (weights_out == key_weights ? weights_out_stride != weight_stride : weights_out != nullptr && weights_out_stride < most)
        return MIIKV_EINVAL;
    if (weights_out != nullptr && weights_out != key_weights) {  // in place, or apart
        const uint64_t rows = static_cast<uint64_t>(batch) * view->kv_heads - 1;
        const uintptr_t in = reinterpret_cast<uintptr_t>(key_weights), to = reinterpret_cast<uintptr_t>(weights_out);
        if (in < to + 4 * (rows * weights_out_stride + most) && to < in + 4 * (rows * weight_stride + max_context)) return MIIKV_EINVAL;
    }
    if (dst_table != nullptr &&
        (view->layout != MIIKV_LAYOUT_PAGED || static_cast<uint64_t>(dst_stride) * view->page_tokens < most))
        return MIIKV_EINVAL;
    if (!aligned16(view->k_codes) || !aligned16(view->v_codes) || !aligned16(view->k_scales) || !aligned16(view->v_scales))
        return MIIKV_EINVAL;
    const uint64_t tiles = (static_cast<uint64_t>(most) + kMoveTokens - 1) / kMoveTokens;
    if (tiles * (view->head_dim / 16 + 1) > 0x7fffffffu) return MIIKV_EINVAL;
    EvictArgs a{};
    a.g = make_geo(*view);
    a.dst_table = dst_table;
    a.dst_stride = dst_stride;
    a.weights = key_weights;
    a.weight_stride = weight_stride;
    a.weights_out = weights_out;
    a.weight_out_stride = weights_out_stride;
    a.lengths = d_lengths;
    a.new_lengths = d_new_lengths;
    a.kept = kept;
    a.batch = batch;
    a.max_context = max_context;
    a.sinks = sinks;
    a.recent = recent;
    a.budget = budget;
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(select_kernel, dim3(view->kv_heads, batch), dim3(kSelectThreads), 0, s, a);
    const bool kf = mode_k_f16(view->quant_mode), vf = mode_v_f16(view->quant_mode);
    if (view->head_dim == 128) launch_move<128>(a, kf, vf, s);
    else launch_move<256>(a, kf, vf, s);
    return hip_status(hipGetLastError());
}
