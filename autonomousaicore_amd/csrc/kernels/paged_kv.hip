// Writing rows of new keys and values into a paged cache, and reading cached rows back.
//
// Both are one pass over packed rows: sequence b's rows offsets[b] .. offsets[b+1] stand at the last
// positions of its lens[b] cached tokens.  A block takes a few rows, finds their places once, and its
// threads then carry 16-byte units of the cache, up to four each with all loads in flight together: a
// thread that went from the offsets to the page table to its row by itself waited for four loads one
// after the other (prompts of 8 x 2048 rows of 8 heads of 128 into e4m3: 24.1 us so, 16.4 us; 16 x 4096 rows
// back: 101 us, 58.8 us).  A head's amax is an exchange among its hd / 16 lanes.  Bound by memory: 4.0 TB/s
// and 4.3 TB/s there, a large copy's 5.0.
#include <algorithm>
#include <type_traits>

#include "paged_kv.hpp"
#include "wave_dpp.hpp"

namespace aic::hip {

void check_cache_shape(const KVPages& c, const char* what) {
    AIC_CHECK(c.type == DType::Float32 || c.type == DType::BFloat16 || c.type == DType::UInt8 || c.type == DType::UInt4, DTypeMismatch, what,
              ": a cache holds float32, bfloat16, e4m3 (uint8) or e2m1 (uint4)");
    AIC_CHECK(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128, InvalidArgument, what,
              ": head_dim must be 32, 64 or 128, got ", c.head_dim);
    AIC_CHECK(c.kv_heads >= 1 && c.kv_heads <= 4096, InvalidArgument, what, ": kv_heads must be 1 .. 4096, got ",
              c.kv_heads);
}

PageView page_view(const KVPages& c, const char* what) {
    check_cache_shape(c, what);
    AIC_CHECK(c.page_size >= 1 && c.page_size <= 65536, InvalidArgument, what, ": page_size must be 1 .. 65536, got ",
              c.page_size);
    AIC_CHECK(c.n_pages >= 1 && c.n_pages <= INT32_MAX, InvalidArgument, what, ": n_pages must be 1 .. 2^31 - 1, got ",
              c.n_pages);
    AIC_CHECK(c.ld_table >= 1, InvalidArgument, what, ": ld_table must be positive, got ", c.ld_table);
    AIC_CHECK(c.k_pages && c.v_pages && c.page_table, InvalidArgument, what, ": null cache pointer");
    AIC_CHECK(!holds_codes(c.type) || (c.k_exps && c.v_exps), InvalidArgument, what,
              ": a cache of codes needs k_exps and v_exps");
    // a head's exponents are read as one word
    AIC_CHECK(c.type != DType::UInt4 || (reinterpret_cast<uintptr_t>(c.k_exps) | reinterpret_cast<uintptr_t>(c.v_exps)) % 4 == 0,
              InvalidArgument, what, ": the exponents of an e2m1 cache must be 4-byte aligned");
    AIC_CHECK((reinterpret_cast<uintptr_t>(c.k_pages) | reinterpret_cast<uintptr_t>(c.v_pages)) % 16 == 0,
              InvalidArgument, what, ": the pools must be 16-byte aligned");
    PageView v{};
    v.kp = static_cast<char*>(c.k_pages);
    v.vp = static_cast<char*>(c.v_pages);
    v.ke = c.k_exps;
    v.ve = c.v_exps;
    v.table = c.page_table;
    v.ld_table = c.ld_table;
    v.n_pages = static_cast<int32_t>(c.n_pages);
    v.ps = static_cast<int32_t>(c.page_size);
    v.Hkv = static_cast<int32_t>(c.kv_heads);
    int l = 0;
    while ((int64_t{1} << l) < c.page_size) ++l;
    v.shift = 31 + l;  // mul * ps - 2^shift < ps <= 2^l: exact for 31-bit positions
    v.mul = static_cast<uint32_t>(((uint64_t{1} << v.shift) + c.page_size - 1) / c.page_size);
    return v;
}

namespace {

// N neighbouring elements of a row as floats; vec: 16-byte aligned.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, bool vec, float (&v)[N]) {
    constexpr int W = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(W)));
    if (vec && N % W == 0) {
#pragma unroll
        for (int i = 0; i < N / W; ++i) {
            const vec_t x = reinterpret_cast<const vec_t*>(p)[i];
#pragma unroll
            for (int j = 0; j < W; ++j) v[i * W + j] = static_cast<float>(x[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = static_cast<float>(p[j]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, bool vec, const float (&v)[N]) {
    constexpr int W = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(W)));
    if (vec && N % W == 0) {
#pragma unroll
        for (int i = 0; i < N / W; ++i) {
            vec_t x;
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = static_cast<T>(v[i * W + j]);  // bf16: to nearest even
            reinterpret_cast<vec_t*>(p)[i] = x;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) p[j] = static_cast<T>(v[j]);
    }
}

constexpr int kMaxRows = 256;   // rows per block

// A batch's rows cut into blocks of `rows` rows x ncol units (2 Hkv heads of hd * size / 16 units); wide
// rows are shared by the blocks of the grid's second dimension.
struct Cut {
    const int64_t *offsets, *lens;
    int64_t T;
    int B, rows, ncol;
    uint32_t mul;  // unit / ncol = unit * mul >> 32, exact for several rows' 1024 units; 0: one row
};

constexpr int kPastAll = -2;    // a position past 2^31 - 1

// The places of the block's rows: page * Hkv * ps + slot, -1: none, -2: a row of no sequence.  where: their positions, -1
// before 0 and for rows of no sequence, or kPastAll.
__device__ __forceinline__ void block_places(const PageView& pv, const Cut& c, int64_t t0, int64_t (&at)[kMaxRows], int* where = nullptr) {
    const int b0 = block_sequence(c.offsets, c.B, t0);
    const int r = static_cast<int>(threadIdx.x);
    if (r < c.rows) {
        int64_t place = -2;
        int b = b0, p = -1;
        const int64_t t = t0 + r;
        int64_t end = b < c.B ? c.offsets[b + 1] : 0;
        while (b < c.B && t >= end) {
            ++b;
            if (b < c.B) end = c.offsets[b + 1];
        }
        if (t < c.T && b >= 0 && b < c.B) {
            const int64_t pos = c.lens[b] - (end - t);
            place = -1;
            if (pos > INT32_MAX) p = kPastAll;
            else if (pos >= 0) {
                const int64_t row = pv.row(pv.table + b * pv.ld_table, static_cast<int>(pos), 0);
                if (row >= 0) place = row;
                p = static_cast<int>(pos);
            }
        }
        at[r] = place;
        if (where) where[r] = p;
    }
    __syncthreads();
}

// Row of unit u of the block.
__device__ __forceinline__ int row_of_unit(const Cut& c, int u) {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(u)) * c.mul) >> 32);
}
// Unit u of the block: row r, k or v, head, first element.
struct Unit {
    int r, kv, h, d;
};
template <int HD, int EPU>
__device__ __forceinline__ Unit unit(const PageView& pv, const Cut& c, int u) {
    constexpr int LPR = HD / EPU;
    Unit x;
    x.r = row_of_unit(c, u);
    const int col = u - x.r * c.ncol, hh = col / LPR;
    x.kv = hh >= pv.Hkv;
    x.h = x.kv ? hh - pv.Hkv : hh;
    x.d = col % LPR * EPU;
    return x;
}

// amax of a row's head -> the exponent e with the least 2^e >= amax / 448 (0 for a zero row, at
// least -126): amax = 1.m 2^(E - 127) and 448 = 1.75 2^8, so e = E - 135, one more where 1.m > 1.75.
__device__ __forceinline__ int row_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u == 0) return 0;
    const int e = static_cast<int>(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -126);
}

// e4m3 has no infinity: held as NaN, and no part of the amax.
__device__ __forceinline__ void finite_or_nan(float& x, float& amax) {
    const bool fine = fabsf(x) < INFINITY;
    amax = fine ? fmaxf(amax, fabsf(x)) : amax;
    x = fine ? x : NAN;
}
// Over a head's lanes: 2, 4 or 8 neighbours of 16 elements.
template <int HD>
__device__ __forceinline__ float head_amax(float amax) {
    amax = fmaxf(amax, dpp<0xb1>(amax));
    if constexpr (HD >= 64) amax = fmaxf(amax, dpp<0x4e>(amax));
    if constexpr (HD >= 128) amax = fmaxf(amax, dpp<0x141>(amax));
    return amax;
}
// Eight elements as codes: one rounding, to nearest even; |x| inv <= 448.
__device__ __forceinline__ uint2 e4m3_codes(const float (&x)[8], float inv) {
    int q[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        q[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inv, x[4 * j + 1] * inv, 0, false);
        q[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inv, x[4 * j + 3] * inv, q[j], true);
    }
    return make_uint2(static_cast<uint32_t>(q[0]), static_cast<uint32_t>(q[1]));
}

template <typename T, typename CT, int HD, int U>
__global__ __launch_bounds__(kBlock) void kv_write_k(PageView pv, Cut c, const T* __restrict__ k, const T* __restrict__ v,
                                                     int64_t ld, bool vec) {
    constexpr int EPU = kPer16<CT>;
    __shared__ int64_t at[kMaxRows];
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.rows;
    const int u0 = static_cast<int>(blockIdx.y) * (kBlock * U) + static_cast<int>(threadIdx.x);
    float x[U][EPU];
    // the rows' data does not wait for their places
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = u0 + i * kBlock;
        const Unit w = unit<HD, EPU>(pv, c, min(u, c.rows * c.ncol - 1));
        const int64_t t = min(t0 + w.r, c.T - 1);
        load_row<T, EPU>((w.kv ? v : k) + t * ld + w.h * HD + w.d, vec, x[i]);
    }
    block_places(pv, c, t0, at);
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = u0 + i * kBlock;
        const bool mine = u < c.rows * c.ncol;
        const Unit w = unit<HD, EPU>(pv, c, mine ? u : c.rows * c.ncol - 1);
        const int64_t place = at[w.r], row = place + static_cast<int64_t>(w.h) * pv.ps;
        const bool go = mine && place >= 0;
        char* pool = w.kv ? pv.vp : pv.kp;
        if constexpr (kE2<CT>) {
            uint32_t amax = 0;  // a unit is a group
#pragma unroll
            for (int j = 0; j < EPU; ++j) amax = max(amax, __float_as_uint(x[i][j]) & 0x7fffffffu);
            const uint32_t byte = group_byte(amax);
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = e2m1_codes(reinterpret_cast<const float(&)[8]>(x[i][8 * j]), byte);
            if (go) {
                *reinterpret_cast<uint4*>(pool + row * (HD / 2) + w.d / 2) = make_uint4(q[0], q[1], q[2], q[3]);
                (w.kv ? pv.ve : pv.ke)[row * (HD / kGroup) + w.d / kGroup] = static_cast<uint8_t>(byte);
            }
        } else if constexpr (kE4<CT>) {
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < EPU; ++j) finite_or_nan(x[i][j], amax);
            const int e = row_exponent(head_amax<HD>(amax));
            const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            const uint2 q0 = e4m3_codes(reinterpret_cast<const float(&)[8]>(x[i][0]), inv);
            const uint2 q1 = e4m3_codes(reinterpret_cast<const float(&)[8]>(x[i][8]), inv);
            if (go) {
                *reinterpret_cast<uint4*>(pool + row * HD + w.d) = make_uint4(q0.x, q0.y, q1.x, q1.y);
                if (w.d == 0) (w.kv ? pv.ve : pv.ke)[row] = static_cast<uint8_t>(e + 127);
            }
        } else {
            if (go) store_row<CT, EPU>(reinterpret_cast<CT*>(pool) + row * HD + w.d, true, x[i]);
        }
    }
}

// Elements of a unit of kv_read: 16 bytes of the cache, of e2m1 half as many (32 elements, four stores 64 bytes apart, would
// leave a store's lanes 16 bytes of every 64: prompts of 8 x 2048 rows of 8 heads of 128 21.0 us for 14.5, 3.8 TB/s).
template <typename CT> constexpr int kRead = kE2<CT> ? 16 : kPer16<CT>;

// Appending with the rotation on the way: a unit is 16 elements of a head, i .. i + 7 of its first half and the same of its second,
// so that a thread holds the pairs that turn together, and the head's hd / 16 lanes hold it whole.  Prompts of 8 x 2048 rows of 16 and 8
// heads of 128 into e2m1: 31.4 us, 4.6 TB/s of a large copy's 5.0 (two units per thread; one 32.7, four 33.0 us).  Columns of a row: H heads of
// q, then Hkv of k, then Hkv of v.
struct Turn {
    const void *q, *k, *v;
    void* q_out;
    int64_t ld_q, ld_qo, ld_kv;
    const float *cos_t, *sin_t;
    int64_t n_pos;
    int H;
    bool vec_q, vec_qo, vec_kv, vec_t;
};
template <typename T, typename CT, int HD, int U>
__global__ __launch_bounds__(kBlock) void kv_append_k(PageView pv, Cut c, Turn a) {
    // y1 = x1 c - x2 s, y2 = x1 s + x2 c: four products and two sums in fp32, each rounded
#pragma clang fp contract(off)
    constexpr int LPH = HD / 16;
    __shared__ int64_t at[kMaxRows];
    __shared__ int pos[kMaxRows];
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.rows;
    const int u0 = static_cast<int>(blockIdx.y) * (kBlock * U) + static_cast<int>(threadIdx.x);
    const int last = c.rows * c.ncol - 1, heads = a.H + pv.Hkv;
    float x1[U][8], x2[U][8];
    // the rows' data does not wait for their places
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = min(u0 + i * kBlock, last), r = row_of_unit(c, u), col = u - r * c.ncol, hh = col / LPH, d = col % LPH * 8;
        const int64_t t = min(t0 + r, c.T - 1);
        const bool q = hh < a.H;
        const int h = q ? hh : hh < heads ? hh - a.H : hh - heads;
        const T* p = static_cast<const T*>(q ? a.q : hh < heads ? a.k : a.v) + t * (q ? a.ld_q : a.ld_kv) + static_cast<int64_t>(h) * HD + d;
        load_row<T, 8>(p, q ? a.vec_q : a.vec_kv, x1[i]);
        load_row<T, 8>(p + HD / 2, q ? a.vec_q : a.vec_kv, x2[i]);
    }
    block_places(pv, c, t0, at, pos);
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = u0 + i * kBlock, uu = min(u, last), r = row_of_unit(c, uu), col = uu - r * c.ncol, hh = col / LPH, d = col % LPH * 8;
        const bool q = hh < a.H, mine = u <= last;
        const int h = q ? hh : hh < heads ? hh - a.H : hh - heads;
        const int p = pos[r];
        const bool turned = p != -1, past = p == kPastAll || p >= a.n_pos;
        if (hh < heads && turned) {
            float cs[8], sn[8];
            const int64_t row = static_cast<int64_t>(past ? 0 : p) * (HD / 2) + d;
            load_row<float, 8>(a.cos_t + row, a.vec_t, cs);
            load_row<float, 8>(a.sin_t + row, a.vec_t, sn);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y1 = x1[i][j] * cs[j] - x2[i][j] * sn[j], y2 = x1[i][j] * sn[j] + x2[i][j] * cs[j];
                x1[i][j] = past ? NAN : y1;
                x2[i][j] = past ? NAN : y2;
            }
        }
        if (q) {
            if (mine && turned) {
                T* o = static_cast<T*>(a.q_out) + (t0 + r) * a.ld_qo + static_cast<int64_t>(h) * HD + d;
                store_row<T, 8>(o, a.vec_qo, x1[i]);
                store_row<T, 8>(o + HD / 2, a.vec_qo, x2[i]);
            }
        }
        const bool v = hh >= heads, go = mine && !q && at[r] >= 0 && !past;
        const int64_t row = at[r] + static_cast<int64_t>(h) * pv.ps;
        char* pool = v ? pv.vp : pv.kp;
        uint8_t* exps = v ? pv.ve : pv.ke;
        if constexpr (kE4<CT>) {
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                finite_or_nan(x1[i][j], amax);
                finite_or_nan(x2[i][j], amax);
            }
            const int e = row_exponent(head_amax<HD>(amax));
            const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            if (go) {
                *reinterpret_cast<uint2*>(pool + row * HD + d) = e4m3_codes(x1[i], inv);
                *reinterpret_cast<uint2*>(pool + row * HD + HD / 2 + d) = e4m3_codes(x2[i], inv);
                if (d == 0) exps[row] = static_cast<uint8_t>(e + 127);
            }
        } else if constexpr (kE2<CT>) {
            uint32_t m1 = 0, m2 = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m1 = max(m1, __float_as_uint(x1[i][j]) & 0x7fffffffu);
                m2 = max(m2, __float_as_uint(x2[i][j]) & 0x7fffffffu);
            }
            if constexpr (HD == 32) m1 = m2 = max(m1, m2);  // one group: two lanes
            m1 = max(m1, dpp<0xb1>(m1)), m2 = max(m2, dpp<0xb1>(m2));
            if constexpr (HD > 32) m1 = max(m1, dpp<0x4e>(m1)), m2 = max(m2, dpp<0x4e>(m2));  // four lanes of each half
            const uint32_t b1 = group_byte(m1), b2 = group_byte(m2);
            if (go) {
                *reinterpret_cast<uint32_t*>(pool + row * (HD / 2) + d / 2) = e2m1_codes(x1[i], b1);
                *reinterpret_cast<uint32_t*>(pool + row * (HD / 2) + (HD / 2 + d) / 2) = e2m1_codes(x2[i], b2);
                if (d % kGroup == 0) {
                    exps[row * (HD / kGroup) + d / kGroup] = static_cast<uint8_t>(b1);
                    if constexpr (HD > 32) exps[row * (HD / kGroup) + (HD / 2 + d) / kGroup] = static_cast<uint8_t>(b2);
                }
            }
        } else if (go) {
            CT* o = reinterpret_cast<CT*>(pool) + row * HD + d;
            store_row<CT, 8>(o, true, x1[i]);
            store_row<CT, 8>(o + HD / 2, true, x2[i]);
        }
    }
}

template <typename T, typename CT, int HD, int U>
__global__ __launch_bounds__(kBlock) void kv_read_k(PageView pv, Cut c, T* __restrict__ k, T* __restrict__ v, int64_t ld, bool vec) {
    constexpr int EPU = kRead<CT>;
    using raw_t = std::conditional_t<EPU == kPer16<CT>, uint4, uint2>;
    __shared__ int64_t at[kMaxRows];
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.rows;
    const int u0 = static_cast<int>(blockIdx.y) * (kBlock * U) + static_cast<int>(threadIdx.x);
    block_places(pv, c, t0, at);
    raw_t raw[U];
    uint32_t ex[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const Unit w = unit<HD, EPU>(pv, c, min(u0 + i * kBlock, c.rows * c.ncol - 1));
        const int64_t place = at[w.r], row = place + static_cast<int64_t>(w.h) * pv.ps;
        raw[i] = raw_t{};
        ex[i] = 127;
        if (place >= 0) {
            raw[i] = *reinterpret_cast<const raw_t*>((w.kv ? pv.vp : pv.kp) + row * static_cast<int64_t>(kRowBytes<CT, HD>) + w.d * 16 / kPer16<CT>);
            if constexpr (kE4<CT>) ex[i] = (w.kv ? pv.ve : pv.ke)[row];
            if constexpr (kE2<CT>) ex[i] = (w.kv ? pv.ve : pv.ke)[row * (HD / kGroup) + w.d / kGroup];
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = u0 + i * kBlock;
        if (u >= c.rows * c.ncol) return;
        const Unit w = unit<HD, EPU>(pv, c, u);
        if (at[w.r] == -2) continue;
        float x[EPU];
        if constexpr (kE2<CT>) {
            const float s = exp_scale(ex[i]);
            e2m1_floats(raw[i].x, s, reinterpret_cast<float(&)[8]>(x[0]));
            e2m1_floats(raw[i].y, s, reinterpret_cast<float(&)[8]>(x[8]));
            if (__builtin_expect(ex[i] == kNanGroup, 0)) {
#pragma unroll
                for (int j = 0; j < EPU; ++j) x[j] = NAN;
            }
        } else if constexpr (kE4<CT>) {
            const float s = exp_scale(ex[i]);
            if (__builtin_expect(ex[i] >= kTopByte, 0)) raw[i] = e4m3_in_range(raw[i], ex[i]);
            float a[8], b[8];
            e4m3_floats(make_uint2(raw[i].x, raw[i].y), s, a);
            e4m3_floats(make_uint2(raw[i].z, raw[i].w), s, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = a[j], x[8 + j] = b[j];
        } else {
            typedef CT vec_t __attribute__((ext_vector_type(EPU)));
            const vec_t y = __builtin_bit_cast(vec_t, raw[i]);
#pragma unroll
            for (int j = 0; j < EPU; ++j) x[j] = static_cast<float>(y[j]);
        }
        store_row<T, EPU>((w.kv ? v : k) + (t0 + w.r) * ld + w.h * HD + w.d, vec, x);
    }
}

template <typename F>
void by_head_dim(int64_t hd, F&& f) {
    if (hd == 32) f(std::integral_constant<int, 32>{});
    else if (hd == 64) f(std::integral_constant<int, 64>{});
    else f(std::integral_constant<int, 128>{});
}

void check_rows(const char* what, const KVPages& c, const void* k, const void* v, int64_t ld, const int64_t* offsets,
                const int64_t* lens, int64_t B, int64_t T, DType dt) {
    AIC_CHECK(dt == DType::Float32 || dt == DType::BFloat16, DTypeMismatch, what, ": rows are float32 or bfloat16");
    AIC_CHECK(c.type == dt || holds_codes(c.type), DTypeMismatch, what, ": rows of ", dtype_name(dt),
              " with a cache of ", dtype_name(c.type));
    AIC_CHECK(B >= 0 && T >= 0 && B <= INT32_MAX && T <= INT32_MAX, InvalidArgument, what, ": B and T must be 0 .. 2^31 - 1");
    AIC_CHECK(ld >= c.kv_heads * c.head_dim, InvalidArgument, what, ": leading dimension ", ld, " below kv_heads * head_dim");
    AIC_CHECK(B == 0 || T == 0 || (k && v && offsets && lens), InvalidArgument, what, ": null pointer");
}

bool aligned16(const void* k, const void* v, int64_t ld, int64_t size) {
    return (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 && ld * size % 16 == 0;
}

// `most` units per thread, or one where that leaves the card mostly empty (a decode step's few rows).  f(cut, grid, few)
template <typename F>
void cut_rows(int64_t ncol, int64_t most, const int64_t* offsets, const int64_t* lens, int64_t B, int64_t T, F&& f) {
    const bool few = T * ncol < kBlock * most * 256;
    const int64_t per = kBlock * (few ? 1 : most);
    Cut cut{offsets, lens, T, static_cast<int>(B), static_cast<int>(std::clamp<int64_t>(per / ncol, 1, kMaxRows)), static_cast<int>(ncol), 0};
    if (cut.rows > 1) cut.mul = static_cast<uint32_t>(((uint64_t{1} << 32) + ncol - 1) / ncol);
    const int64_t blocks = (T + cut.rows - 1) / cut.rows, shares = (cut.rows * ncol + per - 1) / per;
    AIC_CHECK(blocks <= INT32_MAX && shares <= 65535, OutOfRange, "too many rows or heads in one call");
    f(cut, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(shares)), few);
}

// f(row type, cache type)
template <typename F>
void by_types(const KVPages& c, DType dt, F&& f) {
    if (dt == DType::Float32 && c.type == DType::Float32) f(float{}, float{});
    else if (dt == DType::Float32 && c.type == DType::UInt8) f(float{}, uint8_t{});
    else if (dt == DType::Float32) f(float{}, e2m1x2{});
    else if (c.type == DType::BFloat16) f(bf16{}, bf16{});
    else if (c.type == DType::UInt8) f(bf16{}, uint8_t{});
    else f(bf16{}, e2m1x2{});
}

// Four units per thread; of 32 elements, which take twice the registers, two (four: the same 13.1 us for prompts of 8 x 2048 rows).
template <bool READ, typename F>
void launch_rows(const KVPages& c, const int64_t* offsets, const int64_t* lens, int64_t B, int64_t T, DType dt, F&& f) {
    by_types(c, dt, [&](auto t, auto ct) {
        using CT = decltype(ct);
        constexpr int per = READ ? kRead<CT> : kPer16<CT>, most = per == 32 ? 2 : 4;
        cut_rows(2 * c.kv_heads * (c.head_dim / per), most, offsets, lens, B, T, [&](const Cut& cut, dim3 grid, bool few) {
            by_head_dim(c.head_dim, [&](auto hd) {
                if (few) f(t, ct, hd, std::integral_constant<int, 1>{}, grid, cut);
                else f(t, ct, hd, std::integral_constant<int, most>{}, grid, cut);
            });
        });
    });
}

}  // namespace

void kv_write(const KVPages& c, const void* k, const void* v, int64_t ld, const int64_t* offsets, const int64_t* lens,
              int64_t B, int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_write", c, k, v, ld, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_write");
    if (B == 0 || T == 0) return;
    const bool vec = aligned16(k, v, ld, static_cast<int64_t>(dtype_size(dt)));
    launch_rows<false>(c, offsets, lens, B, T, dt, [&](auto t, auto ct, auto hd, auto u, dim3 grid, const Cut& cut) {
        using X = decltype(t);
        kv_write_k<X, decltype(ct), decltype(hd)::value, decltype(u)::value><<<grid, kBlock, 0, s>>>(
            pv, cut, static_cast<const X*>(k), static_cast<const X*>(v), ld, vec);
    });
    AIC_LAUNCH_CHECK("kv_write");
}

void kv_append_rope(const KVPages& c, const void* q, int64_t ld_q, void* q_out, int64_t ld_qo, int64_t H, const void* k, const void* v,
                    int64_t ld_kv, const float* cos_t, const float* sin_t, int64_t n_pos, const int64_t* offsets, const int64_t* lens,
                    int64_t B, int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_append", c, k, v, ld_kv, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_append");
    AIC_CHECK(H >= 0 && H <= 65536, InvalidArgument, "kv_append: H must be 0 .. 65536, got ", H);
    AIC_CHECK(H == 0 || (ld_q >= H * c.head_dim && ld_qo >= H * c.head_dim), InvalidArgument,
              "kv_append: leading dimension of q below H * head_dim");
    AIC_CHECK(n_pos >= 1, InvalidArgument, "kv_append: n_pos must be positive, got ", n_pos);
    if (B == 0 || T == 0) return;
    AIC_CHECK(cos_t && sin_t && (H == 0 || (q && q_out)), InvalidArgument, "kv_append: null pointer");
    AIC_CHECK(H == 0 || q != q_out || ld_q == ld_qo, InvalidArgument, "kv_append: q_out in the place of q needs its leading dimension");
    const int64_t size = static_cast<int64_t>(dtype_size(dt));
    const Turn a{q, k, v, q_out, ld_q, ld_qo, ld_kv, cos_t, sin_t, n_pos, static_cast<int>(H), aligned16(q, q, ld_q, size),
                 aligned16(q_out, q_out, ld_qo, size), aligned16(k, v, ld_kv, size), aligned16(cos_t, sin_t, 4, 4)};
    cut_rows((H + 2 * c.kv_heads) * (c.head_dim / 16), 2, offsets, lens, B, T, [&](const Cut& cut, dim3 grid, bool few) {
        by_types(c, dt, [&](auto t, auto ct) {
            by_head_dim(c.head_dim, [&](auto hd) {
                using X = decltype(t);
                using C = decltype(ct);
                constexpr int D = decltype(hd)::value;
                if (few) kv_append_k<X, C, D, 1><<<grid, kBlock, 0, s>>>(pv, cut, a);
                else kv_append_k<X, C, D, 2><<<grid, kBlock, 0, s>>>(pv, cut, a);
            });
        });
    });
    AIC_LAUNCH_CHECK("kv_append");
}

void kv_read(const KVPages& c, void* k, void* v, int64_t ld, const int64_t* offsets, const int64_t* lens, int64_t B,
             int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_read", c, k, v, ld, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_read");
    if (B == 0 || T == 0) return;
    const bool vec = aligned16(k, v, ld, static_cast<int64_t>(dtype_size(dt)));
    launch_rows<true>(c, offsets, lens, B, T, dt, [&](auto t, auto ct, auto hd, auto u, dim3 grid, const Cut& cut) {
        using X = decltype(t);
        kv_read_k<X, decltype(ct), decltype(hd)::value, decltype(u)::value><<<grid, kBlock, 0, s>>>(
            pv, cut, static_cast<X*>(k), static_cast<X*>(v), ld, vec);
    });
    AIC_LAUNCH_CHECK("kv_read");
}

}  // namespace aic::hip
