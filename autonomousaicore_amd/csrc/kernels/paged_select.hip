// Choosing pages of a long cache for each query: bounds of the pages' keys, and the pages whose bounds promise most.
//
// bounds[page][kvh] holds, for each element, the least and the greatest value of the page's keys.  For a query q no key
// of the page has more than sum_d q_d (hi_d where q_d >= 0, else lo_d); a row's score of a page is the largest of
// its group's heads' sums.  Scores are compared with one another, so they are added in 64 bits, where a bf16
// product is exact and equal sums that 53 bits hold come out equal in any order: the choice does not depend on how such a sum is
// cut.  Longer ones are rounded, so that pages whose scores agree in nearly all of 53 bits may change places between the forms below.
//
// kv_bounds_k: a wave per page and key/value head that the batch's rows touch; lanes hold 16 bytes of a key (8 of codes), the
// wave's groups of lanes go over the keys in turn, with several loads in flight, and are joined at the end.  Prompts of 8 x 4096
// e2m1 rows of 8 heads of 128: 6.4 us, 2.0 TB/s; 32 rows: 6.5 us with the call, a launch's latency.
// kv_score_k: tiles of up to 32 (token, head) pairs of one sequence and key/value head, their q in LDS as doubles, over a run of
// pages; hd / 8 lanes hold a page's bounds in registers, all pages of a wave loaded at once, and go over the tile's rows.
// Where a query's element is negative it meets the page's least, else the greatest: a choice of bits, one product of
// 64 bits in place of two.  Sequences of 32 x 512 pages, 8 heads of 128: 13.9 us, 3.1 TB/s (a table entry and a page's bounds read for
// one step at a time: 24.8); bound by the chain of loads from the batch's offsets to the pages.
// kv_score_many_k: the same for chunks and large groups on the matrix units, also in 64 bits.
// kv_pick_k: a block per row and key/value head finds the score that separates the chosen pages (10 bits of
// their order at a time, from the first bit in which they differ) and writes the pages in order of position.  The scores stay
// in registers, a thread has neighbouring pages: 64 of 2048 pages 7.7 us, 32 x 8 rows' 64 of 512 5.2, steps of a block that wait for one
// another (read from memory at each step, the calls take 17.3 for 13.8 and 19.9 for 19.0).
#include <algorithm>

#include "../runtime/memory_pool.hpp"
#include "attention_paged.hpp"

namespace aic::hip {

namespace {

// ------------------------------------------------------------------------------ bounds
struct BoundArgs {
    PageView kv;
    const int64_t *offsets, *lens;
    int64_t T;
    int B;
    void* bounds;
    int64_t pages;  // at most so many are touched
};

// The pages that sequence b's rows are in: [first, first + count).
__device__ __forceinline__ int touched(const BoundArgs& a, int b, int& first, int& len) {
    const int64_t lo = min(max(a.offsets[b], int64_t{0}), a.T), hi = min(max(a.offsets[b + 1], lo), a.T);
    const int n = static_cast<int>(hi - lo);
    len = static_cast<int>(min(max(a.lens[b], int64_t{0}), kMaxLen));
    first = a.kv.page_index(max(len - n, 0));
    return n > 0 && len > 0 ? a.kv.page_index(len - 1) - first + 1 : 0;
}

// EPL neighbouring elements of a key as floats; of a NaN group anything, its byte tells.
template <typename CT, int EPL>
__device__ __forceinline__ void load_key(const char* p, uint32_t byte, float (&x)[EPL]) {
    if constexpr (kE2<CT>) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const float s = exp_scale(byte);
        e2m1_floats(w.x, s, reinterpret_cast<float(&)[8]>(x[0]));
        e2m1_floats(w.y, s, reinterpret_cast<float(&)[8]>(x[8]));
    } else if constexpr (kE4<CT>) {
        uint4 w = *reinterpret_cast<const uint4*>(p);
        if (__builtin_expect(byte >= kTopByte, 0)) w = e4m3_in_range(w, byte);
        const float s = exp_scale(byte);
        e4m3_floats(make_uint2(w.x, w.y), s, reinterpret_cast<float(&)[8]>(x[0]));
        e4m3_floats(make_uint2(w.z, w.w), s, reinterpret_cast<float(&)[8]>(x[8]));
    } else {
        typedef CT vec_t __attribute__((ext_vector_type(EPL)));
        const vec_t y = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
        for (int j = 0; j < EPL; ++j) x[j] = static_cast<float>(y[j]);
    }
}

// A bound as bf16: the least values towards -infinity, the greatest ones towards infinity.  Only of an e4m3 cache are there any between
// the type's numbers, below its least one, 2^-133: to the nearest, a bound could leave a key out.
template <bool UP>
__device__ __forceinline__ bf16 bound_bf16(float x) {
    const uint32_t u = __float_as_uint(x), away = UP ? x > 0.0f : x < 0.0f;
    return __builtin_bit_cast(bf16, static_cast<uint16_t>((u + (away ? 0xffffu : 0u)) >> 16));
}

// f, idempotent, over the lanes that stand at the same place of their groups of L.
template <int L, typename F>
__device__ __forceinline__ float across_groups(float x, F f) {
    if constexpr (L <= 8) x = f(x, dpp<0x128>(x));  // row_ror 8, 4, 2
    if constexpr (L <= 4) x = f(x, dpp<0x124>(x));
    if constexpr (L <= 2) x = f(x, dpp<0x122>(x));
    if constexpr (L <= 16) x = facing_op<16>(x, f);
    return facing_op<32>(x, f);
}

template <typename CT, int HD>
__global__ __launch_bounds__(kBlock) void kv_bounds_k(BoundArgs a) {
    constexpr int EPL = kE2<CT> ? 16 : kPer16<CT>, L = HD / EPL, RPS = 64 / L, U = kE2<CT> || kE4<CT> ? 4 : 8;  // lanes of a key, keys of a step, steps at a time
    const int lane = threadIdx.x & 63;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (w >= a.pages * a.kv.Hkv) return;
    const int kvh = static_cast<int>(w % a.kv.Hkv);
    double left = static_cast<double>(w / a.kv.Hkv);  // whole numbers below 2^53
    int b = -1, pi = 0, len = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {  // 64 sequences per step, their pages added up across lanes
        int first = 0, n = 0, mine = 0;
        if (b0 + lane < a.B) mine = touched(a, b0 + lane, first, n);
        const double upto = wave_running_sum(static_cast<double>(mine));
        const uint64_t past = __ballot(left < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            b = b0 + l;
            const int before = static_cast<int>(left - (upto - mine));  // in lane l: of its sequence's pages
            pi = __builtin_amdgcn_readlane(first, l) + __builtin_amdgcn_readlane(before, l);
            len = __builtin_amdgcn_readlane(n, l);
            break;
        }
        left -= __shfl(upto, 63, 64);
    }
    if (b < 0 || pi >= a.kv.ld_table) return;
    const int page = a.kv.table[b * a.kv.ld_table + pi];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.kv.n_pages)) return;
    const int64_t row0 = (static_cast<int64_t>(page) * a.kv.Hkv + kvh) * a.kv.ps;
    const int filled = static_cast<int>(min(static_cast<int64_t>(a.kv.ps), len - static_cast<int64_t>(pi) * a.kv.ps));
    const int grp = lane / L, d0 = lane % L * EPL;
    auto least = [](float x, float y) { return __builtin_elementwise_minimum(x, y); };  // a NaN stays
    auto most = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
    float lo[EPL], hi[EPL];
    uint32_t top_byte = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) lo[j] = INFINITY, hi[j] = -INFINITY;
    for (int r0 = 0; r0 < filled; r0 += U * RPS) {
        float x[U][EPL];
        uint32_t byte[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t row = row0 + min(r0 + i * RPS + grp, filled - 1);  // past the last key: the last one again
            byte[i] = 127;
            if constexpr (kE4<CT>) byte[i] = a.kv.ke[row];
            if constexpr (kE2<CT>) byte[i] = a.kv.ke[row * (HD / kGroup) + d0 / kGroup];
            top_byte = max(top_byte, byte[i]);
            load_key<CT, EPL>(a.kv.kp + row * kRowBytes<CT, HD> + d0 * 16 / kPer16<CT>, byte[i], x[i]);
        }
#pragma unroll
        for (int i = 0; i < U; i += 2)
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                lo[j] = least(least(lo[j], x[i][j]), x[i + 1][j]);
                hi[j] = most(most(hi[j], x[i][j]), x[i + 1][j]);
            }
    }
    if constexpr (kE2<CT>) {
        if (top_byte == kNanGroup)
#pragma unroll
            for (int j = 0; j < EPL; ++j) lo[j] = hi[j] = NAN;
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) lo[j] = across_groups<L>(lo[j], least), hi[j] = across_groups<L>(hi[j], most);
    if (grp < 2) {  // one group writes the least, the next one the greatest values
        using BT = std::conditional_t<std::is_same_v<CT, float>, float, bf16>;
        BT* out = static_cast<BT*>(a.bounds) + ((static_cast<int64_t>(page) * a.kv.Hkv + kvh) * 2 + grp) * HD + d0;
        constexpr int W = 16 / sizeof(BT);
        typedef BT vec_t __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int j = 0; j < EPL; j += W) {
            vec_t y;
#pragma unroll
            for (int u = 0; u < W; ++u) {
                if constexpr (kE4<CT>) y[u] = grp == 0 ? bound_bf16<false>(lo[j + u]) : bound_bf16<true>(hi[j + u]);
                else y[u] = static_cast<BT>(grp == 0 ? lo[j + u] : hi[j + u]);  // exact: each is a cached value
            }
            *reinterpret_cast<vec_t*>(out + j) = y;
        }
    }
}

// ------------------------------------------------------------------------------ scores
struct SelectArgs {
    PagedArgs a;        // kv, q, ldq, T, offsets, lens, B, H, G, vec_q
    const void* bounds;
    double* scores;     // [T][Hkv][n_pages]; null: every row takes all its pages
    int64_t n_pages;    // of the longest cache
    int first, last, n_sel;
    int32_t* picked;
    int64_t* picked_lens;
};
constexpr int kRows = 32;       // (token, head) pairs of a tile

__device__ __forceinline__ int pages_of(const PageView& kv, int pos) { return pos < 0 ? 0 : kv.page_index(pos) + 1; }

// Over groups of L lanes, in all of them.
template <int L>
__device__ __forceinline__ double group_sum(double x) {
    x += dpp<0xb1>(x);   // quad_perm 1 0 3 2
    x += dpp<0x4e>(x);   // quad_perm 2 3 0 1
    if constexpr (L >= 8) x += dpp<0x141>(x);   // row_half_mirror
    if constexpr (L >= 16) x += dpp<0x140>(x);  // row_mirror
    return x;
}

// Eight elements of a page's bounds, and of them those that a query's signs meet: the least where it is negative.
template <typename BT> struct Bounds8;
template <> struct Bounds8<bf16> {
    uint4 lo, hi;
    __device__ __forceinline__ void load(const bf16* p, int hd) {
        lo = *reinterpret_cast<const uint4*>(p);
        hi = *reinterpret_cast<const uint4*>(p + hd);
    }
    __device__ __forceinline__ void meet(const uint32_t (&neg)[8], float (&x)[8]) const {
        const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = (neg[2 * i] & 0xffffu) | (neg[2 * i + 1] & 0xffff0000u), w = (l[i] & m) | (h[i] & ~m);
            x[2 * i] = __uint_as_float(w << 16);
            x[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
        }
    }
};
template <> struct Bounds8<float> {
    uint4 lo[2], hi[2];
    __device__ __forceinline__ void load(const float* p, int hd) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo[i] = reinterpret_cast<const uint4*>(p)[i];
            hi[i] = reinterpret_cast<const uint4*>(p + hd)[i];
        }
    }
    __device__ __forceinline__ void meet(const uint32_t (&neg)[8], float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t l[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w}, h[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = __uint_as_float((l[j] & neg[4 * i + j]) | (h[j] & ~neg[4 * i + j]));
        }
    }
};

// Tiles of up to kRows (token, head) pairs of a sequence and key/value head.
struct ScoreTile {
    Seq sq;
    int b, kvh, t0, nt;  // first token and their number
    int pages;           // that the last of them has, in the workspace's scores
    int per;             // heads of the group at a time: all of them, unless they are more than kRows
};
// Tiles of `tokens` tokens; false: none, or nothing to choose from page `first` on.
__device__ __forceinline__ bool score_tile(const SelectArgs& s, int tokens, int first, ScoreTile& x) {
    const PagedArgs& a = s.a;
    const int Hkv = a.kv.Hkv, tile = static_cast<int>(blockIdx.x) / Hkv;
    x.kvh = static_cast<int>(blockIdx.x) % Hkv;
    // 64 sequences per step, the found one's description from its lane
    const int lane = threadIdx.x & 63, shift = __builtin_ctz(tokens);
    x.b = -1;
    int left = tile;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        Seq own{};
        if (b0 + lane < a.B) own = sequence(a, b0 + lane);
        const int tiles = (own.n >> shift) + ((own.n & (tokens - 1)) != 0), upto = wave_running_sum(tiles);
        const uint64_t past = __ballot(left < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto at = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            const auto row0 = static_cast<uint64_t>(own.row0);
            x.b = b0 + l;
            x.sq = {static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(at(static_cast<int>(row0 >> 32)))) << 32 |
                                         static_cast<uint32_t>(at(static_cast<int>(row0)))),
                    at(own.n), at(own.len)};
            x.t0 = (left - at(upto - tiles)) << shift;
            break;
        }
        left -= __builtin_amdgcn_readlane(upto, 63);
    }
    if (x.b < 0) return false;
    x.nt = min(tokens, x.sq.n - x.t0);
    x.per = min(a.G, kRows / tokens);
    // rows past the workspace's pages have no scores (kv_pick_k)
    x.pages = static_cast<int>(min(static_cast<int64_t>(pages_of(a.kv, x.sq.len - x.sq.n + x.t0 + x.nt - 1)), s.n_pages));
    return x.pages > s.n_sel && first < x.pages - s.last;
}
// The tile's queries of heads g0 .. g0 + ng of the group, row (token, head): [row][4][L] of two doubles, the rows' starts
// 16 bytes apart in the banks: a lane's eight neighbouring elements lie L doubles apart, and the same element of other rows in others.
template <int HD> constexpr int kQueryRow = HD / 2 + 1;
template <int HD> __device__ __forceinline__ int query_at(int d) { return ((d & 7) >> 1) * (HD / 8) + (d >> 3); }
template <typename T, int HD>
__device__ __forceinline__ void stage_queries(const SelectArgs& s, const ScoreTile& x, int g0, int ng, double2* qs) {
    const PagedArgs& a = s.a;
    for (int i = threadIdx.x; i < x.nt * ng * HD; i += kBlock) {
        const int r = i / HD, d = i % HD, t = r / ng;
        const float y = ld(static_cast<const T*>(a.q) + (x.sq.row0 + x.t0 + t) * a.ldq + static_cast<int64_t>(x.kvh * a.G + g0 + r - t * ng) * HD, d);
        reinterpret_cast<double*>(qs + r * kQueryRow<HD> + query_at<HD>(d))[d & 1] = static_cast<double>(y) + 0.0;  // -0 as 0
    }
}
// A page's score over the group's heads; best: over those of this chunk of them.
__device__ __forceinline__ void put_score(const SelectArgs& s, const ScoreTile& x, int t, int p, double best, bool valid, bool first_chunk) {
    // a NaN; a page that is none: chosen, and the row's attention is NaN
    if (best != best || !valid) best = INFINITY;
    double* out = s.scores + ((x.sq.row0 + x.t0 + t) * s.a.kv.Hkv + x.kvh) * s.n_pages + p;
    *out = first_chunk ? best : fmax(*out, best);
}

// A wave's NS steps of pages, all loaded at once.
template <typename BT, int HD, int NS>
struct ScorePages {
    static constexpr int L = HD / 8, PPS = 64 / L, PAGES = NS * PPS;  // lanes of a page, pages of a step and in all
    Bounds8<BT> bd[NS];
    bool valid[NS];
    __device__ __forceinline__ void load(const SelectArgs& s, const ScoreTile& x, int id) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            const int page = __shfl(id, k * PPS + lane / L, 64);
            valid[k] = static_cast<uint32_t>(page) < static_cast<uint32_t>(s.a.kv.n_pages);
            bd[k].load(static_cast<const BT*>(s.bounds) + (static_cast<int64_t>(valid[k] ? page : 0) * s.a.kv.Hkv + x.kvh) * 2 * HD + lane % L * 8, HD);
        }
    }
    __device__ __forceinline__ void score(const SelectArgs& s, const ScoreTile& x, const double2* qs, int p0, int g0, int ng) const {
        const int lane = threadIdx.x & 63, l = lane % L;
        for (int t = 0; t < x.nt; ++t) {
            double best[NS];
#pragma unroll
            for (int k = 0; k < NS; ++k) best[k] = -INFINITY;
            for (int g = 0; g < ng; ++g) {
                double q[8];
                uint32_t neg[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double2 y = qs[(t * ng + g) * kQueryRow<HD> + j * L + l];
                    q[2 * j] = y.x, q[2 * j + 1] = y.y;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) neg[j] = static_cast<uint32_t>(__double_as_longlong(q[j]) >> 63);
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    float y[8];
                    bd[k].meet(neg, y);
                    double sum = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum = fma(q[j], static_cast<double>(y[j]), sum);
                    sum = group_sum<L>(sum);
                    best[k] = sum > best[k] || sum != sum ? sum : best[k];
                }
            }
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const int p = p0 + k * PPS + lane / L;
                if (l == 0 && p < x.pages) put_score(s, x, t, p, best[k], valid[k], g0 == 0);
            }
        }
    }
};

// f(p0, id, g0, ng): the block's runs of 4 * PAGES pages, a wave's first page and its lanes' page ids, for each chunk of heads with its
// queries staged; load(id) before the queries are.
template <typename T, int HD, int PAGES, typename Load, typename F>
__device__ __forceinline__ void over_runs(const SelectArgs& s, const ScoreTile& x, double2* qs, Load load, F f) {
    const PagedArgs& a = s.a;
    const int lane = threadIdx.x & 63, mine = static_cast<int>(threadIdx.x >> 6) * PAGES;
    const int32_t* tr = a.kv.table + x.b * a.kv.ld_table;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * (4 * PAGES), stride = static_cast<int64_t>(gridDim.y) * (4 * PAGES);
    auto page_id = [&](int64_t p) { return lane < PAGES && p + lane < x.pages && p + lane < a.kv.ld_table ? tr[p + lane] : -1; };
    int id = page_id(first + mine);
    for (int64_t run = first; run < x.pages; run += stride) {
        const int p0 = static_cast<int>(run) + mine, now = id;
        load(now);
        id = page_id(run + stride + mine);
        for (int g0 = 0; g0 < a.G; g0 += x.per) {
            const int ng = min(x.per, a.G - g0);
            if (run == first || a.G > x.per) {  // else they are there
                if (run != first || g0 > 0) __syncthreads();
                stage_queries<T, HD>(s, x, g0, ng, qs);
                __syncthreads();
            }
            if (p0 < x.pages) f(p0, now, g0, ng);
        }
    }
}

template <typename T, typename BT, int HD, int NS>
__global__ __launch_bounds__(kBlock) void kv_score_k(SelectArgs s, int tokens) {
    using P = ScorePages<BT, HD, NS>;
    extern __shared__ __attribute__((aligned(16))) double2 qs[];
    ScoreTile x;
    if (!score_tile(s, tokens, static_cast<int>(blockIdx.y) * (4 * P::PAGES), x)) return;
    P pages;
    over_runs<T, HD, P::PAGES>(
        s, x, qs, [&](int id) { pages.load(s, x, id); }, [&](int p0, int, int g0, int ng) { pages.score(s, x, qs, p0, g0, ng); });
}

// The same for many pairs, on the matrix units: sum_d of q+ hi and of q- lo, K = 2 HD in 64 bits; 16 pages of a wave, lane
// (page, quarter of the columns).  An infinite bound would meet the zeros of the other sign: then as above.  512 rows of 32 heads over 8 on
// 512 pages: 103 us, the matrix units busy 58% of it with two waves to a SIMD (both 16-row tiles of 32 pairs at once, the bounds
// made 64 bits as they are used: the call 142 us for 114).
template <typename T, typename BT, int HD>
__global__ __launch_bounds__(kBlock) void kv_score_many_k(SelectArgs s, int tokens) {
    using Plain = ScorePages<BT, HD, HD / 32>;
    static_assert(Plain::PAGES == 16);
    typedef double f64x4 __attribute__((ext_vector_type(4)));
    constexpr int C = HD / 4, EV = 16 / sizeof(BT), NV = C / EV;  // columns of a lane, elements of a load, loads
    extern __shared__ __attribute__((aligned(16))) double2 qs[];
    ScoreTile x;
    if (!score_tile(s, tokens, static_cast<int>(blockIdx.y) * 64, x)) return;
    const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
    double* out = reinterpret_cast<double*>(qs + min(tokens * x.per, kRows) * kQueryRow<HD>) + static_cast<int>(threadIdx.x >> 6) * (kRows * 16);  // [row][16]
    uint4 lo[NV], hi[NV];
    bool valid = false;
    auto load = [&](int id) {
        const int page = __shfl(id, col, 64);
        valid = static_cast<uint32_t>(page) < static_cast<uint32_t>(s.a.kv.n_pages);
        const BT* p = static_cast<const BT*>(s.bounds) + (static_cast<int64_t>(valid ? page : 0) * s.a.kv.Hkv + x.kvh) * 2 * HD + quarter * C;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            lo[i] = reinterpret_cast<const uint4*>(p)[i];
            hi[i] = reinterpret_cast<const uint4*>(p + HD)[i];
        }
    };
    auto value = [](const uint4& w, int j) {  // element j of 16 bytes
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
        if constexpr (sizeof(BT) == 4) return static_cast<double>(__uint_as_float(v[j]));
        else return static_cast<double>(__uint_as_float(j & 1 ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16));
    };
    over_runs<T, HD, 16>(s, x, qs, load, [&](int p0, int id, int g0, int ng) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) bad |= non_finite_bits<BT>(lo[i]) | non_finite_bits<BT>(hi[i]);
        if (__builtin_expect(__ballot(bad != 0) != 0, 0)) {
            Plain pages;
            pages.load(s, x, id);
            pages.score(s, x, qs, p0, g0, ng);
            return;
        }
        // one 16-row tile after the other: the bounds stay in registers in 64 bits
        const int rows = x.nt * ng;
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 16) {
            f64x4 acc = {0.0, 0.0, 0.0, 0.0};
            const double2* q = qs + min(r0 + col, rows - 1) * kQueryRow<HD> + (quarter * C >> 3);
#pragma unroll
            for (int d = 0; d < C; d += 2) {
                const double2 y = q[((d & 7) >> 1) * (HD / 8) + (d >> 3)];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(u ? y.y : y.x));
                    const uint64_t neg = static_cast<uint64_t>(static_cast<int64_t>(bits) >> 63);
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(__longlong_as_double(static_cast<long long>(bits & neg)), value(lo[(d + u) / EV], (d + u) % EV), acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(__longlong_as_double(static_cast<long long>(bits & ~neg)), value(hi[(d + u) / EV], (d + u) % EV), acc, 0, 0, 0);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) out[(r0 + 4 * e + quarter) * 16 + col] = acc[e];  // row 4 e + quarter
        }
        // lane: page col of every fourth token
        wave_lds_fence();
        const int p = p0 + col;
        for (int t = quarter; t < x.nt; t += 4) {
            double best = -INFINITY;
            for (int g = 0; g < ng; ++g) {
                const double sum = out[(t * ng + g) * 16 + col];
                best = sum > best || sum != sum ? sum : best;
            }
            if (p < x.pages) put_score(s, x, t, p, best, valid, g0 == 0);
        }
        wave_lds_fence();
    });
}

// -------------------------------------------------------------------------------- pick
// Orders doubles as whole numbers do; -0 as 0.
__device__ __forceinline__ uint64_t order(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int kBins = 1024;

// K: pages of a thread, neighbouring ones, whose scores it keeps; 0: any number, read from memory each time.
template <int K>
__global__ __launch_bounds__(kBlock) void kv_pick_k(SelectArgs s) {
    const PagedArgs& a = s.a;
    const int Hkv = a.kv.Hkv, kvh = static_cast<int>(blockIdx.x) % Hkv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t t = blockIdx.x / static_cast<unsigned>(Hkv), at = t * Hkv + kvh;
    __shared__ uint4 bins[kBins / 4];
    __shared__ double ends[2][4];
    __shared__ int sums[3][4];
    __shared__ int cut_bin, cut_need, cut_count;

    const double* scores = s.scores + at * s.n_pages;
    double kept[K > 0 ? K : 1];
    if (K > 0 && s.scores) {  // on their way before the row is known; what lies behind its pages is not used
#pragma unroll
        for (int j = 0; j < K; ++j) kept[j] = tid * K + j < s.n_pages ? scores[tid * K + j] : 0.0;
    }
    // the row's sequence, by every wave for itself
    int own_b = -1, pos = -1;
    bool past = false;  // of a sequence longer than lengths reach, whose tiles have scored other positions
    for (int b0 = 0; b0 < a.B && own_b < 0; b0 += 256) {
        int64_t from[4], to[4], len[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = min(b0 + 64 * j + lane, a.B - 1);
            from[j] = a.offsets[i], to[j] = a.offsets[i + 1], len[j] = a.lens[i];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t here = __ballot(b0 + 64 * j + lane < a.B && from[j] <= t && t < to[j]);
            if (here) {
                const int l = __builtin_ctzll(here);
                const int64_t at_pos = len[j] - (to[j] - t);
                own_b = b0 + 64 * j + l;
                pos = __builtin_amdgcn_readlane(at_pos < 0 ? -1 : static_cast<int>(min(at_pos, kMaxLen)), l);
                past = pos >= 0 && __ballot(len[j] > kMaxLen) >> l & 1;
            }
        }
    }
    const bool nobody = own_b < 0;
    const int P = pages_of(a.kv, pos);
    int32_t* out = s.picked + at * s.n_sel;
    const int32_t* tr = a.kv.table + static_cast<int64_t>(nobody ? 0 : own_b) * a.kv.ld_table;
    auto id = [&](int p) { return p < a.kv.ld_table ? tr[p] : -1; };
    if (past || P > s.n_pages) {  // past max_len: a position without a place, so that the row's attention is NaN
        for (int i = tid; i < s.n_sel; i += kBlock) out[i] = -1;
        if (tid == 0) s.picked_lens[at] = 1;
        return;
    }
    if (P <= s.n_sel) {
        for (int i = tid; i < s.n_sel; i += kBlock) out[i] = i < P ? id(i) : -1;
        if (tid == 0) s.picked_lens[at] = nobody ? -1 : pos + 1;
        return;
    }

    // a thread's pages [q0, q1), of which those in [c0, c1) are free to choose
    const int run = K > 0 ? K : (P + kBlock - 1) / kBlock;
    auto at_most = [&](int64_t p) { return static_cast<int>(min(p, static_cast<int64_t>(P))); };
    const int q0 = at_most(static_cast<int64_t>(tid) * run), q1 = at_most(static_cast<int64_t>(tid + 1) * run), c0 = s.first, c1 = P - s.last;
    [[maybe_unused]] int32_t ids[K > 0 ? K : 1];
    uint64_t keys[K > 0 ? K : 1];
    if constexpr (K > 0) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            ids[j] = q0 + j < q1 ? id(q0 + j) : -1;
            keys[j] = order(kept[j]);
        }
    }
    // f(page, its score's order, j) of this thread's pages
    auto each = [&](auto f) {
        if constexpr (K > 0) {
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (q0 + j < q1) f(q0 + j, keys[j], j);
        } else {
            for (int p = q0; p < q1; ++p) f(p, order(scores[p]), 0);
        }
    };
    auto free = [&](int p) { return p >= c0 && p < c1; };

    // chosen: order >> shift above `prefix`, and of those at it the first `need`
    int need = s.n_sel - s.first - s.last;
    double lo = INFINITY, hi = -INFINITY;
    if constexpr (K > 0) {
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (q0 + j < q1 && free(q0 + j)) lo = fmin(lo, kept[j]), hi = fmax(hi, kept[j]);
    } else {
        for (int p = max(q0, c0); p < min(q1, c1); ++p) lo = fmin(lo, scores[p]), hi = fmax(hi, scores[p]);
    }
    lo = wave_all(lo, [](double x, double y) { return fmin(x, y); });
    hi = wave_all(hi, [](double x, double y) { return fmax(x, y); });
    if (lane == 0) ends[0][wave] = lo, ends[1][wave] = hi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) lo = fmin(lo, ends[0][w]), hi = fmax(hi, ends[1][w]);
    const uint64_t first_key = order(lo), last_key = order(hi);
    int shift = first_key == last_key ? 0 : 64 - __builtin_clzll(first_key ^ last_key);  // the bits below it differ
    uint64_t prefix = shift == 64 ? 0 : last_key >> shift;
    int count = c1 - c0;
    while (shift > 0 && count != need && need > 0) {
        const int next = max(shift - 10, 0), bits = shift - next;
        bins[tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        each([&](int p, uint64_t k, int) {
            if (free(p) && (shift == 64 ? 0 : k >> shift) == prefix) atomicAdd(reinterpret_cast<uint32_t*>(bins) + ((k >> next) & ((1u << bits) - 1)), 1u);
        });
        __syncthreads();
        // from the top: thread i has bins 1023 - 4 i and the three below
        const uint4 mine = bins[kBins / 4 - 1 - tid];
        const int total = static_cast<int>(mine.x + mine.y + mine.z + mine.w), upto = wave_running_sum(total);
        if (lane == 63) sums[2][wave] = upto;
        __syncthreads();
        int before = upto - total;
#pragma unroll
        for (int w = 0; w < 3; ++w) before += w < wave ? sums[2][w] : 0;
        if (before < need && need <= before + total) {
            const uint32_t n[4] = {mine.w, mine.z, mine.y, mine.x};
            int left = need - before, i = 0;
            while (i < 3 && left > static_cast<int>(n[i])) left -= static_cast<int>(n[i++]);
            cut_bin = kBins - 1 - (4 * tid + i), cut_need = left, cut_count = static_cast<int>(n[i]);
        }
        __syncthreads();
        prefix = shift == 64 ? static_cast<uint64_t>(cut_bin) : prefix << bits | static_cast<uint64_t>(cut_bin);
        need = cut_need, count = cut_count, shift = next;
    }

    // in order of position
    int ties = 0, sure = 0;
    each([&](int p, uint64_t k, int) {
        const uint64_t h = shift == 64 ? 0 : k >> shift;
        ties += free(p) && h == prefix;
        sure += !free(p) || h > prefix;
    });
    const int ties_upto = wave_running_sum(ties);
    if (lane == 63) sums[0][wave] = ties_upto;
    __syncthreads();
    int tie = ties_upto - ties;
#pragma unroll
    for (int w = 0; w < 3; ++w) tie += w < wave ? sums[0][w] : 0;
    const int mine = sure + min(ties, max(need - tie, 0)), upto = wave_running_sum(mine);
    if (lane == 63) sums[1][wave] = upto;
    __syncthreads();
    int place = upto - mine;
#pragma unroll
    for (int w = 0; w < 3; ++w) place += w < wave ? sums[1][w] : 0;
    each([&](int p, uint64_t k, int j) {
        bool take = true;
        if (free(p)) {
            const uint64_t h = shift == 64 ? 0 : k >> shift;
            take = h > prefix || (h == prefix && tie++ < need);
        }
        if (take) out[place++] = K > 0 ? ids[j] : id(p);
    });
    if (tid == 0) s.picked_lens[at] = static_cast<int64_t>(s.n_sel - 1) * a.kv.ps + (pos - (P - 1) * a.kv.ps) + 1;
}

// Blocks of kv_score_k: what the card holds at once, four to a CU, which go on to further runs of pages, their ids ahead (a block for every run,
// two rounds of them: 16.2 us for 13.9).
constexpr int64_t kScoreBlocks = 1024;
// Pairs of a tile from which on the matrix units score them, 16 rows of a product being there in any case.  The call: 512 tokens of 32 heads over 8
// on 512 pages, 113.9 us and 244 with kv_score_k; 2 x 8 tokens, 18.5 and 29.4; 16 x 5 tokens of 2 heads, 24.4 and 28.2; a token's 16 heads of a group,
// 32 sequences, 27.8 and 35.2; its 8, 40.3 and 38.4.  Tiles so few that a wave takes one step's pages (below) do not come here: one sequence of 512 pages,
// 32 heads over 8, 8 tokens, 20.4 so and 18.2 here, 4 tokens, 14.9 and 14.3, 2 tokens, 12.1 and 13.8.
constexpr int64_t kManyPairs = 9;
int64_t longest_pages(const KVPages& c, int64_t max_len) { return (max_len + c.page_size - 1) / c.page_size; }

void check_select(const KVPages& c, int64_t T, int64_t max_len) {
    check_cache_shape(c, "kv_select");
    AIC_CHECK(c.page_size >= 1 && c.page_size <= 65536, InvalidArgument, "kv_select: page_size must be 1 .. 65536, got ", c.page_size);
    AIC_CHECK(T >= 0 && T <= INT32_MAX, InvalidArgument, "kv_select: T must be 0 .. 2^31 - 1");
    AIC_CHECK(max_len >= 0 && max_len <= kMaxLen, InvalidArgument, "kv_select: max_len must be 0 .. ", kMaxLen);
}

}  // namespace

void kv_bounds(const KVPages& c, void* bounds, const int64_t* offsets, const int64_t* lens, int64_t B, int64_t T, hipStream_t s) {
    const PageView pv = page_view(c, "kv_bounds");
    AIC_CHECK(B >= 0 && T >= 0 && B <= INT32_MAX && T <= INT32_MAX, InvalidArgument, "kv_bounds: B and T must be 0 .. 2^31 - 1");
    if (B == 0 || T == 0) return;
    AIC_CHECK(bounds && offsets && lens, InvalidArgument, "kv_bounds: null pointer");
    AIC_CHECK(reinterpret_cast<uintptr_t>(bounds) % 16 == 0, InvalidArgument, "kv_bounds: the bounds must be 16-byte aligned");
    // n rows are in at most (n - 1) / page_size + 2 pages
    const BoundArgs a{pv, offsets, lens, T, static_cast<int>(B), bounds, T / c.page_size + 2 * std::min(B, T)};
    const int64_t blocks = (a.pages * c.kv_heads + 3) / 4;
    AIC_CHECK(blocks <= INT32_MAX, OutOfRange, "kv_bounds: too many rows in one call");
    auto run = [&](auto ct, auto hd) {
        kv_bounds_k<decltype(ct), decltype(hd)::value><<<static_cast<unsigned>(blocks), kBlock, 0, s>>>(a);
    };
    auto types = [&](auto hd) {
        if (c.type == DType::Float32) run(float{}, hd);
        else if (c.type == DType::BFloat16) run(bf16{}, hd);
        else if (c.type == DType::UInt8) run(uint8_t{}, hd);
        else run(e2m1x2{}, hd);
    };
    if (c.head_dim == 32) types(std::integral_constant<int, 32>{});
    else if (c.head_dim == 64) types(std::integral_constant<int, 64>{});
    else types(std::integral_constant<int, 128>{});
    AIC_LAUNCH_CHECK("kv_bounds");
}

int64_t kv_select_workspace(const KVPages& c, int64_t T, int64_t max_len) {
    check_select(c, T, max_len);
    const int64_t pages = longest_pages(c, max_len), rows = T * c.kv_heads;
    AIC_CHECK(pages == 0 || rows <= INT64_MAX / 8 / pages, OutOfRange, "kv_select: too many rows and pages in one call");
    return rows * pages * 8;
}

void kv_select(const KVPages& c, const void* bounds, const void* q, int64_t ld_q, const int64_t* offsets, const int64_t* lens, int64_t B,
               int64_t T, int64_t max_q, int64_t max_len, int64_t H, int64_t first, int64_t last, int64_t n_sel, int32_t* picked,
               int64_t* picked_lens, void* workspace, int64_t workspace_bytes, DType dt, hipStream_t s) {
    const int64_t most = kv_select_workspace(c, T, max_len);
    AIC_CHECK(B >= 0 && B <= INT32_MAX, InvalidArgument, "kv_select: B must be 0 .. 2^31 - 1");
    AIC_CHECK(max_q >= 0, InvalidArgument, "kv_select: max_q must not be negative");
    AIC_CHECK(dt == DType::Float32 || dt == DType::BFloat16, DTypeMismatch, "kv_select: queries are float32 or bfloat16");
    AIC_CHECK(c.type == dt || holds_codes(c.type), DTypeMismatch, "kv_select: queries of ", dtype_name(dt), " with a cache of ",
              dtype_name(c.type));
    AIC_CHECK(H >= 1 && H % c.kv_heads == 0, ShapeMismatch, "kv_select: ", H, " query heads over ", c.kv_heads, " key/value heads");
    AIC_CHECK(H <= 65536, InvalidArgument, "kv_select: more than 65536 query heads");
    AIC_CHECK(ld_q >= H * c.head_dim, InvalidArgument, "kv_select: leading dimension below heads * head_dim");
    AIC_CHECK(first >= 0 && last >= 1 && n_sel >= 1 && first <= n_sel && last <= n_sel - first && n_sel <= (1 << 24), InvalidArgument,
              "kv_select: n_sel must be up to 2^24 and hold the first ", first, " (from 0) and the last ", last, " (from 1) pages, got ", n_sel);
    AIC_CHECK(workspace_bytes >= 0, InvalidArgument, "kv_select: negative workspace size");
    const PageView pv = page_view(c, "kv_select");
    if (T == 0) return;
    AIC_CHECK(bounds && q && picked && picked_lens && (B == 0 || (offsets && lens)), InvalidArgument, "kv_select: null pointer");
    AIC_CHECK(reinterpret_cast<uintptr_t>(bounds) % 16 == 0, InvalidArgument, "kv_select: the bounds must be 16-byte aligned");
    const bool scored = B > 0 && longest_pages(c, max_len) > n_sel;
    const int64_t need = scored ? most : 0;
    const StreamScratchUse use(s);
    if (workspace) {
        AIC_CHECK(workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, InvalidArgument,
                  "kv_select: the workspace must be 16-byte aligned and hold ", need, " bytes, got ", workspace_bytes);
    } else if (need > 0) {
        AIC_CHECK(stream_scratch_ready(s), InvalidState, "kv_select: a captured call needs a workspace of its own");
        workspace = stream_scratch(static_cast<size_t>(need), s);
    }
    SelectArgs x{};
    x.a.kv = pv;
    x.a.q = q, x.a.ldq = ld_q, x.a.T = T;
    x.a.offsets = offsets, x.a.lens = lens;
    x.a.B = static_cast<int>(B), x.a.H = static_cast<int>(H), x.a.G = static_cast<int>(H / c.kv_heads);
    x.bounds = bounds;
    x.scores = scored ? static_cast<double*>(workspace) : nullptr;
    x.n_pages = longest_pages(c, max_len);
    x.first = static_cast<int>(first), x.last = static_cast<int>(last), x.n_sel = static_cast<int>(n_sel);
    x.picked = picked, x.picked_lens = picked_lens;
    const int64_t picks = T * c.kv_heads;
    AIC_CHECK(picks <= INT32_MAX, OutOfRange, "kv_select: too many rows in one call");
    if (scored) {
        int tokens = 32;
        while (tokens > 1 && (tokens * x.a.G > kRows || tokens / 2 >= std::min(max_q, T))) tokens /= 2;
        const int64_t tiles = (tokens == 1 ? T : (T + tokens - 1) / tokens + std::min(B, T)) * c.kv_heads;
        AIC_CHECK(tiles <= INT32_MAX, OutOfRange, "kv_select: too many rows in one call");
        const int64_t pairs = tokens * std::min(x.a.G, kRows / tokens);
        auto launch = [&](auto hd, auto steps) {
            constexpr int D = decltype(hd)::value, NS = decltype(steps)::value, per = 4 * NS * (512 / D);
            const size_t lds = static_cast<size_t>(pairs) * kQueryRow<D> * sizeof(double2);  // at most 33 KB
            const int64_t runs = (x.n_pages + per - 1) / per, most = std::max<int64_t>(kScoreBlocks / tiles, 1);
            const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(std::min<int64_t>({runs, most, 65535})));
            if (NS == D / 32 && pairs >= kManyPairs) {
                const size_t both = lds + 4 * kRows * 16 * sizeof(double);
                if (c.type == DType::Float32) kv_score_many_k<float, float, D><<<grid, kBlock, both, s>>>(x, tokens);
                else if (dt == DType::Float32) kv_score_many_k<float, bf16, D><<<grid, kBlock, both, s>>>(x, tokens);
                else kv_score_many_k<bf16, bf16, D><<<grid, kBlock, both, s>>>(x, tokens);
            } else if (c.type == DType::Float32) kv_score_k<float, float, D, NS><<<grid, kBlock, lds, s>>>(x, tokens);
            else if (dt == DType::Float32) kv_score_k<float, bf16, D, NS><<<grid, kBlock, lds, s>>>(x, tokens);
            else kv_score_k<bf16, bf16, D, NS><<<grid, kBlock, lds, s>>>(x, tokens);
        };
        auto run = [&](auto hd) {
            // 16 pages of a wave; one step's where that would leave CUs without a block: the call on 2048 pages of 2 heads, 64 blocks
            // 16.5, 256 13.8 us; 2 x 512 of 8 heads, 128 and 512 blocks, 11.5 and 11.5; 8 of them, 12.0 and 12.4; 32, 19.0 and 20.4
            constexpr int NS = decltype(hd)::value / 32;
            if (NS > 1 && tiles * ((x.n_pages + 63) / 64) < 256) launch(hd, std::integral_constant<int, 1>{});
            else launch(hd, std::integral_constant<int, NS>{});
        };
        if (c.head_dim == 32) run(std::integral_constant<int, 32>{});
        else if (c.head_dim == 64) run(std::integral_constant<int, 64>{});
        else run(std::integral_constant<int, 128>{});
        AIC_LAUNCH_CHECK("kv_select scores");
    }
    const auto grid = static_cast<unsigned>(picks);
    // the call, 2 kept, 8 kept and none: 512 pages, 32 x 8 rows, 19.0, 20.9 and 19.9 us; 2048 pages, 2 rows, 13.8 with 8 and 17.3 without,
    // 32 x 8 rows 46.3 and 50.6
    if (x.n_pages <= 2 * kBlock) kv_pick_k<2><<<grid, kBlock, 0, s>>>(x);
    else if (x.n_pages <= 8 * kBlock) kv_pick_k<8><<<grid, kBlock, 0, s>>>(x);
    else kv_pick_k<0><<<grid, kBlock, 0, s>>>(x);
    AIC_LAUNCH_CHECK("kv_select");
}

}  // namespace aic::hip
