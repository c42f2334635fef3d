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
    AIC_CHECK(c.type == DType::Float32 || c.type == DType::BFloat16 || c.type == DType::UInt8, DTypeMismatch, what,
              ": a cache holds float32, bfloat16 or e4m3 (uint8)");
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
    AIC_CHECK(c.type != DType::UInt8 || (c.k_exps && c.v_exps), InvalidArgument, what,
              ": an e4m3 cache needs k_exps and v_exps");
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

// The places of the block's rows: page * Hkv * ps + slot, -1: none, -2: a row of no sequence.
__device__ __forceinline__ void block_places(const PageView& pv, const Cut& c, int64_t t0, int64_t (&at)[kMaxRows]) {
    const int b0 = block_sequence(c.offsets, c.B, t0);
    const int r = static_cast<int>(threadIdx.x);
    if (r < c.rows) {
        int64_t place = -2;
        int b = b0;
        const int64_t t = t0 + r;
        int64_t end = b < c.B ? c.offsets[b + 1] : 0;
        while (b < c.B && t >= end) {
            ++b;
            if (b < c.B) end = c.offsets[b + 1];
        }
        if (t < c.T && b >= 0 && b < c.B) {
            const int64_t pos = c.lens[b] - (end - t);
            place = -1;
            if (pos >= 0 && pos <= INT32_MAX) {
                const int64_t row = pv.row(pv.table + b * pv.ld_table, static_cast<int>(pos), 0);
                if (row >= 0) place = row;
            }
        }
        at[r] = place;
    }
    __syncthreads();
}

// Unit u of the block: row r, k or v, head, first element.
struct Unit {
    int r, kv, h, d;
};
template <int HD, int EPU>
__device__ __forceinline__ Unit unit(const PageView& pv, const Cut& c, int u) {
    constexpr int LPR = HD / EPU;
    Unit x;
    x.r = static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(u)) * c.mul) >> 32);
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

template <typename T, typename CT, int HD, int U>
__global__ __launch_bounds__(kBlock) void kv_write_k(PageView pv, Cut c, const T* __restrict__ k, const T* __restrict__ v,
                                                     int64_t ld, bool vec) {
    constexpr int EPU = 16 / sizeof(CT);
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
        if constexpr (sizeof(CT) == 1) {
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < EPU; ++j) {
                const bool fine = fabsf(x[i][j]) < INFINITY;  // e4m3 has no infinity: held as NaN
                amax = fine ? fmaxf(amax, fabsf(x[i][j])) : amax;
                x[i][j] = fine ? x[i][j] : NAN;
            }
            amax = fmaxf(amax, dpp<0xb1>(amax));  // the head's lanes: 2, 4 or 8 neighbours
            if constexpr (HD >= 64) amax = fmaxf(amax, dpp<0x4e>(amax));
            if constexpr (HD >= 128) amax = fmaxf(amax, dpp<0x141>(amax));
            const int e = row_exponent(amax);
            const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            int q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // one rounding, to nearest even; |x| inv <= 448
                q[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[i][4 * j] * inv, x[i][4 * j + 1] * inv, 0, false);
                q[j] = __builtin_amdgcn_cvt_pk_fp8_f32(x[i][4 * j + 2] * inv, x[i][4 * j + 3] * inv, q[j], true);
            }
            if (go) {
                *reinterpret_cast<int4*>(pool + row * HD + w.d) = make_int4(q[0], q[1], q[2], q[3]);
                if (w.d == 0) (w.kv ? pv.ve : pv.ke)[row] = static_cast<uint8_t>(e + 127);
            }
        } else {
            if (go) store_row<CT, EPU>(reinterpret_cast<CT*>(pool) + row * HD + w.d, true, x[i]);
        }
    }
}

template <typename T, typename CT, int HD, int U>
__global__ __launch_bounds__(kBlock) void kv_read_k(PageView pv, Cut c, T* __restrict__ k, T* __restrict__ v, int64_t ld, bool vec) {
    constexpr int EPU = 16 / sizeof(CT);
    __shared__ int64_t at[kMaxRows];
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * c.rows;
    const int u0 = static_cast<int>(blockIdx.y) * (kBlock * U) + static_cast<int>(threadIdx.x);
    block_places(pv, c, t0, at);
    uint4 raw[U];
    uint32_t ex[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const Unit w = unit<HD, EPU>(pv, c, min(u0 + i * kBlock, c.rows * c.ncol - 1));
        const int64_t place = at[w.r], row = place + static_cast<int64_t>(w.h) * pv.ps;
        raw[i] = make_uint4(0, 0, 0, 0);
        ex[i] = 127;
        if (place >= 0) {
            raw[i] = *reinterpret_cast<const uint4*>((w.kv ? pv.vp : pv.kp) + row * static_cast<int64_t>(HD * sizeof(CT)) + w.d * sizeof(CT));
            if constexpr (sizeof(CT) == 1) ex[i] = (w.kv ? pv.ve : pv.ke)[row];
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = u0 + i * kBlock;
        if (u >= c.rows * c.ncol) return;
        const Unit w = unit<HD, EPU>(pv, c, u);
        if (at[w.r] == -2) continue;
        float x[EPU];
        if constexpr (sizeof(CT) == 1) {
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
    AIC_CHECK(c.type == dt || c.type == DType::UInt8, DTypeMismatch, what, ": rows of ", dtype_name(dt),
              " with a cache of ", dtype_name(c.type));
    AIC_CHECK(B >= 0 && T >= 0 && B <= INT32_MAX && T <= INT32_MAX, InvalidArgument, what, ": B and T must be 0 .. 2^31 - 1");
    AIC_CHECK(ld >= c.kv_heads * c.head_dim, InvalidArgument, what, ": leading dimension ", ld, " below kv_heads * head_dim");
    AIC_CHECK(B == 0 || T == 0 || (k && v && offsets && lens), InvalidArgument, what, ": null pointer");
}

bool aligned16(const void* k, const void* v, int64_t ld, int64_t size) {
    return (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 && ld * size % 16 == 0;
}

// Four units per thread, or one where that leaves the card mostly empty (a decode step's few rows).
template <typename F>
void launch_rows(const KVPages& c, const int64_t* offsets, const int64_t* lens, int64_t B, int64_t T, DType dt, F&& f) {
    const int64_t ncol = 2 * c.kv_heads * (c.head_dim * static_cast<int64_t>(dtype_size(c.type)) / 16);
    const bool few = T * ncol < kBlock * 4 * 256;
    const int64_t per = kBlock * (few ? 1 : 4);
    Cut cut{offsets, lens, T, static_cast<int>(B), static_cast<int>(std::clamp<int64_t>(per / ncol, 1, kMaxRows)), static_cast<int>(ncol), 0};
    if (cut.rows > 1) cut.mul = static_cast<uint32_t>(((uint64_t{1} << 32) + ncol - 1) / ncol);
    const int64_t blocks = (T + cut.rows - 1) / cut.rows, shares = (cut.rows * ncol + per - 1) / per;
    AIC_CHECK(blocks <= INT32_MAX && shares <= 65535, OutOfRange, "too many rows or heads in one call");
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(shares));
    auto types = [&](auto hd, auto u) {
        if (dt == DType::Float32 && c.type == DType::Float32) f(float{}, float{}, hd, u, grid, cut);
        else if (dt == DType::Float32) f(float{}, uint8_t{}, hd, u, grid, cut);
        else if (c.type == DType::BFloat16) f(bf16{}, bf16{}, hd, u, grid, cut);
        else f(bf16{}, uint8_t{}, hd, u, grid, cut);
    };
    by_head_dim(c.head_dim, [&](auto hd) {
        if (few) types(hd, std::integral_constant<int, 1>{});
        else types(hd, std::integral_constant<int, 4>{});
    });
}

}  // namespace

void kv_write(const KVPages& c, const void* k, const void* v, int64_t ld, const int64_t* offsets, const int64_t* lens,
              int64_t B, int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_write", c, k, v, ld, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_write");
    if (B == 0 || T == 0) return;
    const bool vec = aligned16(k, v, ld, static_cast<int64_t>(dtype_size(dt)));
    launch_rows(c, offsets, lens, B, T, dt, [&](auto t, auto ct, auto hd, auto u, dim3 grid, const Cut& cut) {
        using X = decltype(t);
        kv_write_k<X, decltype(ct), decltype(hd)::value, decltype(u)::value><<<grid, kBlock, 0, s>>>(
            pv, cut, static_cast<const X*>(k), static_cast<const X*>(v), ld, vec);
    });
    AIC_LAUNCH_CHECK("kv_write");
}

void kv_read(const KVPages& c, void* k, void* v, int64_t ld, const int64_t* offsets, const int64_t* lens, int64_t B,
             int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_read", c, k, v, ld, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_read");
    if (B == 0 || T == 0) return;
    const bool vec = aligned16(k, v, ld, static_cast<int64_t>(dtype_size(dt)));
    launch_rows(c, offsets, lens, B, T, dt, [&](auto t, auto ct, auto hd, auto u, dim3 grid, const Cut& cut) {
        using X = decltype(t);
        kv_read_k<X, decltype(ct), decltype(hd)::value, decltype(u)::value><<<grid, kBlock, 0, s>>>(
            pv, cut, static_cast<X*>(k), static_cast<X*>(v), ld, vec);
    });
    AIC_LAUNCH_CHECK("kv_read");
}

}  // namespace aic::hip
