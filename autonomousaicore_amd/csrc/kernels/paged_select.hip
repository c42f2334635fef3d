// Choosing pages of a long cache for each query: bounds of the pages' keys, and the pages whose bounds promise most.
//
// bounds[page][kvh] holds, for each element, the least and the greatest value of the page's keys.  For a query q no key
// of the page has more than sum_d max(q_d lo_d, q_d hi_d); a row's score of a page is the largest of
// its group's heads' sums.  Scores are compared with one another, so they are added in 64 bits, where a bf16
// product is exact and equal sums come out equal in any order that their digits allow: the choice does not
// depend on how the sum is cut.
//
// kv_bounds_k: a wave per page and key/value head that the batch's rows touch; lanes hold 16 bytes of a key (8 of codes), the
// wave's groups of lanes go over the keys in turn and are joined at the end.
// kv_score_k: tiles of up to 32 (token, head) pairs of one sequence and key/value head, their q in LDS as doubles, over a run of
// pages; hd / 8 lanes hold a page's bounds in registers and go over the tile's rows.
// kv_pick_k: a block per row and key/value head finds the score that separates the chosen pages (10 bits of
// their order at a time, from the first bit in which they differ) and writes the pages in order of position.
#include <algorithm>

#include "../runtime/memory_pool.hpp"
#include "attention_paged.hpp"

namespace aic::hip {

namespace {

template <typename T> using Bound = std::conditional_t<std::is_same_v<T, float>, float, bf16>;

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

// EPL neighbouring elements of a key as floats.
template <typename CT, int EPL>
__device__ __forceinline__ void load_key(const char* p, uint32_t byte, float (&x)[EPL]) {
    if constexpr (kE2<CT>) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const float s = exp_scale(byte);
        e2m1_floats(w.x, s, reinterpret_cast<float(&)[8]>(x[0]));
        e2m1_floats(w.y, s, reinterpret_cast<float(&)[8]>(x[8]));
        if (byte == kNanGroup)
#pragma unroll
            for (int j = 0; j < EPL; ++j) x[j] = NAN;
    } else if constexpr (kE4<CT>) {
        uint4 w = *reinterpret_cast<const uint4*>(p);
        if (byte >= kTopByte) w = e4m3_in_range(w, byte);
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

// The first one's NaN or the second's.
__device__ __forceinline__ float least(float x, float y) { return x < y || x != x ? x : y; }
__device__ __forceinline__ float most(float x, float y) { return x > y || x != x ? x : y; }

template <typename CT, int HD>
__global__ __launch_bounds__(kBlock) void kv_bounds_k(BoundArgs a) {
    constexpr int EPL = kE2<CT> ? 16 : kPer16<CT>, L = HD / EPL, RPS = 64 / L;  // lanes of a key, keys of a step
    const int lane = threadIdx.x & 63;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (w >= a.pages * a.kv.Hkv) return;
    const int kvh = static_cast<int>(w % a.kv.Hkv);
    int64_t left = w / a.kv.Hkv;
    int b = -1, pi = 0, len = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {  // 64 sequences per step, their pages added up across lanes
        int first = 0, n = 0, mine = 0;
        if (b0 + lane < a.B) mine = touched(a, b0 + lane, first, n);
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t x = __shfl_up(upto, o, 64);
            if (lane >= o) upto += x;
        }
        const uint64_t past = __ballot(left < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            b = b0 + l;
            pi = __shfl(first, l, 64) + static_cast<int>(left - (__shfl(upto, l, 64) - __shfl(mine, l, 64)));
            len = __shfl(n, l, 64);
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
    float lo[EPL], hi[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) lo[j] = INFINITY, hi[j] = -INFINITY;
    for (int r0 = 0; r0 < filled; r0 += 2 * RPS) {
        // two keys at a time: past the last one, the last one again
        float x[2][EPL];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t row = row0 + min(r0 + i * RPS + grp, filled - 1);
            uint32_t byte = 127;
            if constexpr (kE4<CT>) byte = a.kv.ke[row];
            if constexpr (kE2<CT>) byte = a.kv.ke[row * (HD / kGroup) + d0 / kGroup];
            load_key<CT, EPL>(a.kv.kp + row * kRowBytes<CT, HD> + d0 * 16 / kPer16<CT>, byte, x[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                lo[j] = least(lo[j], x[i][j]);
                hi[j] = most(hi[j], x[i][j]);
            }
    }
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const float x = __shfl_xor(lo[j], o, 64), y = __shfl_xor(hi[j], o, 64);
            lo[j] = least(lo[j], x);
            hi[j] = most(hi[j], y);
        }
    if (grp == 0) {
        using BT = Bound<CT>;
        BT* out = static_cast<BT*>(a.bounds) + (static_cast<int64_t>(page) * a.kv.Hkv + kvh) * 2 * HD + d0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {  // exact: a bound is a cached value
            st(out, j, lo[j]);
            st(out, HD + j, hi[j]);
        }
    }
}

// ------------------------------------------------------------------------------ scores
struct SelectArgs {
    PagedArgs a;        // kv, q, ldq, T, offsets, lens, B, H, G, vec_q
    const void* bounds;
    double* scores;     // [T][Hkv][n_pages]
    int64_t n_pages;    // of the longest cache
    int first, last, n_sel;
    int32_t* picked;
    int64_t* picked_lens;
};
constexpr int kRows = 32;    // (token, head) pairs of a tile
constexpr int kRun = 32;     // pages of a block

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

template <typename T, typename BT, int HD>
__global__ __launch_bounds__(kBlock) void kv_score_k(SelectArgs s, int tokens) {
    constexpr int L = HD / 8, PPS = 64 / L;  // lanes of a page, pages of a wave's step
    __shared__ __attribute__((aligned(16))) double qs[kRows][HD];
    const PagedArgs& a = s.a;
    const int Hkv = a.kv.Hkv, kvh = static_cast<int>(blockIdx.x) % Hkv, tile = static_cast<int>(blockIdx.x) / Hkv;
    int b, local;
    {
        // tiles of `tokens` tokens: find_tile counts rows of one head
        PagedArgs one = a;
        one.G = 1;
        bool found;
        if (tokens == 32) found = find_tile<32>(one, tile, b, local);
        else if (tokens == 16) found = find_tile<16>(one, tile, b, local);
        else if (tokens == 8) found = find_tile<8>(one, tile, b, local);
        else if (tokens == 4) found = find_tile<4>(one, tile, b, local);
        else if (tokens == 2) found = find_tile<2>(one, tile, b, local);
        else found = find_tile<1>(one, tile, b, local);
        if (!found) return;
    }
    const Seq sq = wave_sequence(a, b);
    const int t0 = local * tokens, nt = min(tokens, sq.n - t0);
    // the last row's pages; rows past the workspace's have no scores (kv_pick_k)
    const int most_pages = static_cast<int>(min(static_cast<int64_t>(pages_of(a.kv, sq.len - sq.n + t0 + nt - 1)), s.n_pages));
    const int first_run = static_cast<int>(blockIdx.y) * kRun;
    if (most_pages <= s.n_sel || first_run >= most_pages - s.last) return;  // nothing to choose here
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane / L, d0 = lane % L * 8;
    const int32_t* tr = a.kv.table + b * a.kv.ld_table;

    // heads of the group, kRows / tokens at a time (one chunk unless the group is larger than kRows)
    const int per = min(a.G, kRows / tokens);
    for (int g0 = 0; g0 < a.G; g0 += per) {
        const int ng = min(per, a.G - g0), rows = nt * ng;
        __syncthreads();
        for (int i = threadIdx.x; i < rows * HD; i += kBlock) {
            const int r = i / HD, d = i % HD;
            qs[r][d] = ld(static_cast<const T*>(a.q) + (sq.row0 + t0 + r / ng) * a.ldq + static_cast<int64_t>(kvh * a.G + g0 + r % ng) * HD, d);
        }
        __syncthreads();
        for (int64_t p0 = first_run; p0 < most_pages; p0 += static_cast<int64_t>(gridDim.y) * kRun)
        for (int p = static_cast<int>(p0) + wave * PPS + grp; p - grp < min(static_cast<int>(p0) + kRun, most_pages); p += 4 * PPS) {
            const int page = p < most_pages && p < a.kv.ld_table ? tr[p] : -1;
            const bool valid = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.n_pages);
            const BT* bp = static_cast<const BT*>(s.bounds) + (static_cast<int64_t>(valid ? page : 0) * Hkv + kvh) * 2 * HD + d0;
            double lo[8], hi[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) lo[j] = ld(bp, j), hi[j] = ld(bp + HD, j);
            for (int t = 0; t < nt; ++t) {
                double best = -INFINITY;
                for (int g = 0; g < ng; ++g) {
                    const double* q = &qs[t * ng + g][d0];
                    double sum = 0.0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum = fma(q[j], q[j] >= 0.0 ? hi[j] : lo[j], sum);
                    sum = group_sum<L>(sum);
                    best = sum > best || sum != sum ? sum : best;
                }
                if (best != best || !valid) best = INFINITY;  // also a page that is none: chosen, and the row's attention is NaN
                if (lane % L == 0 && p < most_pages) {
                    double* out = s.scores + ((sq.row0 + t0 + t) * Hkv + kvh) * s.n_pages + p;
                    *out = g0 > 0 ? fmax(*out, best) : best;
                }
            }
        }
    }
}

// -------------------------------------------------------------------------------- pick
// Orders doubles as whole numbers do; -0 as 0.
__device__ __forceinline__ uint64_t order(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int kBins = 1024;

__global__ __launch_bounds__(kBlock) void kv_pick_k(SelectArgs s) {
    const PagedArgs& a = s.a;
    const int Hkv = a.kv.Hkv, kvh = static_cast<int>(blockIdx.x) % Hkv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t t = blockIdx.x / static_cast<unsigned>(Hkv), at = t * Hkv + kvh;
    __shared__ uint32_t bins[kBins];
    __shared__ uint64_t ends[2][4];
    __shared__ int sums[2][4];
    __shared__ int cut_bin, cut_need, cut_count;

    int b = block_sequence(a.offsets, a.B, t);
    while (b >= 0 && b < a.B && t >= a.offsets[b + 1]) ++b;
    int32_t* out = s.picked + at * s.n_sel;
    const bool nobody = b < 0 || b >= a.B;
    const int64_t pos64 = nobody ? -1 : a.lens[b] - (a.offsets[b + 1] - t);
    const int pos = pos64 < 0 || pos64 > kMaxLen ? -1 : static_cast<int>(pos64), P = pages_of(a.kv, pos);
    const int32_t* tr = a.kv.table + static_cast<int64_t>(nobody ? 0 : b) * a.kv.ld_table;
    auto id = [&](int p) { return p < a.kv.ld_table ? tr[p] : -1; };
    if (P > s.n_pages) {  // past max_len: a position without a place, so that the row's attention is NaN
        for (int i = tid; i < s.n_sel; i += kBlock) out[i] = -1;
        if (tid == 0) s.picked_lens[at] = 1;
        return;
    }
    if (P <= s.n_sel) {
        for (int i = tid; i < s.n_sel; i += kBlock) out[i] = i < P ? id(i) : -1;
        if (tid == 0) s.picked_lens[at] = nobody ? -1 : pos + 1;
        return;
    }

    const int c0 = s.first, c1 = P - s.last;
    int need = s.n_sel - s.first - s.last;
    const double* scores = s.scores + at * s.n_pages;
    // chosen: order >> shift above `prefix`, and of those at it the first `need`
    uint64_t lo = ~0ull, hi = 0;
    for (int p = c0 + tid; p < c1; p += kBlock) {
        const uint64_t k = order(scores[p]);
        lo = min(lo, k), hi = max(hi, k);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t x = __shfl_xor(static_cast<unsigned long long>(lo), o, 64), y = __shfl_xor(static_cast<unsigned long long>(hi), o, 64);
        lo = min(lo, x), hi = max(hi, y);
    }
    if (lane == 0) ends[0][wave] = lo, ends[1][wave] = hi;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) lo = min(lo, ends[0][w]), hi = max(hi, ends[1][w]);
    int shift = lo == hi ? 0 : 64 - __builtin_clzll(lo ^ hi);  // the bits below it differ
    uint64_t prefix = shift == 64 ? 0 : hi >> shift;
    int count = c1 - c0;
    while (shift > 0 && count != need && need > 0) {
        const int next = max(shift - 10, 0), bits = shift - next;
        for (int i = tid; i < kBins; i += kBlock) bins[i] = 0;
        __syncthreads();
        for (int p = c0 + tid; p < c1; p += kBlock) {
            const uint64_t k = order(scores[p]);
            if ((shift == 64 ? 0 : k >> shift) == prefix) atomicAdd(&bins[(k >> next) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // lane l: bins 16 l .. 16 l + 15, from the top
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) mine += bins[kBins - 1 - (16 * lane + i)];
            const int upto = wave_running_sum(static_cast<int>(mine)), before = upto - static_cast<int>(mine);
            if (before < need && need <= upto) {
                int left = need - before;
                for (int i = 0; i < 16; ++i) {
                    const int bin = kBins - 1 - (16 * lane + i), n = static_cast<int>(bins[bin]);
                    if (left <= n) {
                        cut_bin = bin, cut_need = left, cut_count = n;
                        break;
                    }
                    left -= n;
                }
            }
        }
        __syncthreads();
        prefix = shift == 64 ? static_cast<uint64_t>(cut_bin) : prefix << bits | static_cast<uint64_t>(cut_bin);
        need = cut_need, count = cut_count, shift = next;
    }

    // in order of position: a run of pages per thread
    const int run = (P + kBlock - 1) / kBlock, q0 = min(tid * run, P), q1 = min(q0 + run, P);
    auto head = [&](int p) { return order(scores[p]) >> shift; };
    auto free = [&](int p) { return p >= c0 && p < c1; };
    int ties = 0, sure = 0;
    for (int p = q0; p < q1; ++p) {
        if (!free(p)) {
            ++sure;
        } else {
            const uint64_t h = shift == 64 ? 0 : head(p);
            ties += h == prefix;
            sure += h > prefix;
        }
    }
    const int ties_upto = wave_running_sum(ties);
    if (lane == 63) sums[0][wave] = ties_upto;
    __syncthreads();
    int tie = ties_upto - ties;
    for (int w = 0; w < wave; ++w) tie += sums[0][w];
    const int mine = sure + min(ties, max(need - tie, 0)), upto = wave_running_sum(mine);
    if (lane == 63) sums[1][wave] = upto;
    __syncthreads();
    int place = upto - mine;
    for (int w = 0; w < wave; ++w) place += sums[1][w];
    for (int p = q0; p < q1; ++p) {
        bool take = true;
        if (free(p)) {
            const uint64_t h = shift == 64 ? 0 : head(p);
            take = h > prefix || (h == prefix && tie++ < need);
        }
        if (take) out[place++] = id(p);
    }
    if (tid == 0) s.picked_lens[at] = static_cast<int64_t>(s.n_sel - 1) * a.kv.ps + (pos - (P - 1) * a.kv.ps) + 1;
}

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
    const int64_t need = kv_select_workspace(c, T, max_len);
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
    x.scores = static_cast<double*>(workspace);
    x.n_pages = longest_pages(c, max_len);
    x.first = static_cast<int>(first), x.last = static_cast<int>(last), x.n_sel = static_cast<int>(n_sel);
    x.picked = picked, x.picked_lens = picked_lens;
    const int64_t picks = T * c.kv_heads;
    AIC_CHECK(picks <= INT32_MAX, OutOfRange, "kv_select: too many rows in one call");
    if (B > 0 && x.n_pages > n_sel) {
        int tokens = 32;
        while (tokens > 1 && (tokens * x.a.G > kRows || tokens / 2 >= std::min(max_q, T))) tokens /= 2;
        const int64_t tiles = (T + tokens - 1) / tokens + std::min(B, T), runs = (x.n_pages + kRun - 1) / kRun;
        AIC_CHECK(tiles * c.kv_heads <= INT32_MAX, OutOfRange, "kv_select: too many rows in one call");
        const dim3 grid(static_cast<unsigned>(tiles * c.kv_heads), static_cast<unsigned>(std::min<int64_t>(runs, 65535)));
        auto run = [&](auto hd) {
            constexpr int D = decltype(hd)::value;
            if (c.type == DType::Float32) kv_score_k<float, float, D><<<grid, kBlock, 0, s>>>(x, tokens);
            else if (dt == DType::Float32) kv_score_k<float, bf16, D><<<grid, kBlock, 0, s>>>(x, tokens);
            else kv_score_k<bf16, bf16, D><<<grid, kBlock, 0, s>>>(x, tokens);
        };
        if (c.head_dim == 32) run(std::integral_constant<int, 32>{});
        else if (c.head_dim == 64) run(std::integral_constant<int, 64>{});
        else run(std::integral_constant<int, 128>{});
        AIC_LAUNCH_CHECK("kv_select scores");
    }
    kv_pick_k<<<static_cast<unsigned>(picks), kBlock, 0, s>>>(x);
    AIC_LAUNCH_CHECK("kv_select");
}

}  // namespace aic::hip
