// Writing rows of new keys and values into a paged cache, and reading cached rows back.
//
// Both are one pass over packed rows: sequence b's rows offsets[b] .. offsets[b+1] stand at the last
// positions of its lens[b] cached tokens.  A thread carries eight elements of one (row, head), so a
// bf16 row is read in 16-byte pieces, its head's amax is one exchange among hd / 8 lanes, and codes
// are written 8 bytes at a time.  Bound by memory.
#include "paged_kv.hpp"

namespace aic::hip {

PageView page_view(const KVPages& c, const char* what) {
    AIC_CHECK(c.type == DType::Float32 || c.type == DType::BFloat16 || c.type == DType::UInt8, DTypeMismatch, what,
              ": a cache holds float32, bfloat16 or e4m3 (uint8)");
    AIC_CHECK(c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128, InvalidArgument, what,
              ": head_dim must be 32, 64 or 128, got ", c.head_dim);
    AIC_CHECK(c.kv_heads >= 1 && c.kv_heads <= 4096, InvalidArgument, what, ": kv_heads must be 1 .. 4096, got ",
              c.kv_heads);
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

template <typename T> struct Oct;  // eight elements of a row
template <> struct Oct<float> {
    static __device__ __forceinline__ void load(const float* p, bool vec, float (&v)[8]) {
        if (vec) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = p[j];
        }
    }
    static __device__ __forceinline__ void store(float* p, bool vec, const float (&v)[8]) {
        if (vec) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = v[j];
        }
    }
};
template <> struct Oct<bf16> {
    static __device__ __forceinline__ void load(const bf16* p, bool vec, float (&v)[8]) {
        if (vec) {
            const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = bf2f(a[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = bf2f(p[j]);
        }
    }
    static __device__ __forceinline__ void store(bf16* p, bool vec, const float (&v)[8]) {
        if (vec) {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                      pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = f2bf(v[j]);
        }
    }
};

// One thread's eight elements: packed row t, k or v, head h, elements 8c ..
struct Piece {
    int64_t t = 0, row = -1;
    int kv = 0, h = 0, c = 0;
    bool live = false;  // row t belongs to a sequence
};

template <int HD>
__device__ __forceinline__ Piece piece(const PageView& pv, const int64_t* offsets, const int64_t* lens, int B, int64_t T) {
    constexpr int LPR = HD / 8;
    const int64_t per_row = 2LL * pv.Hkv * LPR, first = static_cast<int64_t>(blockIdx.x) * kBlock;
    const int b0 = block_sequence(offsets, B, first / per_row);
    const int64_t i = first + threadIdx.x;
    Piece p;
    p.t = i / per_row;
    const int r = static_cast<int>(i - p.t * per_row);
    p.c = r % LPR;
    p.h = (r / LPR) % pv.Hkv;
    p.kv = r / LPR / pv.Hkv;
    if (p.t >= T) return p;
    int b = b0;
    while (b < B && p.t >= offsets[b + 1]) ++b;
    if (b < 0 || b >= B) return p;
    p.live = true;
    const int64_t pos = lens[b] - (offsets[b + 1] - p.t);
    if (pos < 0 || pos > INT32_MAX) return p;
    p.row = pv.row(pv.table + b * pv.ld_table, static_cast<int>(pos), p.h);
    return p;
}

// amax of a row's head -> the exponent e with the least 2^e >= amax / 448 (0 for a zero row, at
// least -126): amax = 1.m 2^(E - 127) and 448 = 1.75 2^8, so e = E - 135, one more where 1.m > 1.75.
__device__ __forceinline__ int row_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u == 0) return 0;
    const int e = static_cast<int>(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -126);
}

template <typename T, typename CT, int HD>
__global__ __launch_bounds__(kBlock) void kv_write_k(PageView pv, const T* __restrict__ k, const T* __restrict__ v, int64_t ld,
                                                     const int64_t* __restrict__ offsets, const int64_t* __restrict__ lens,
                                                     int B, int64_t rows, bool vec) {
    const Piece p = piece<HD>(pv, offsets, lens, B, rows);
    float x[8] = {};
    if (p.row >= 0) Oct<T>::load((p.kv ? v : k) + p.t * ld + p.h * HD + p.c * 8, vec, x);
    if constexpr (sizeof(CT) == 1) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (!(fabsf(x[j]) < INFINITY)) x[j] = NAN;  // e4m3 has no infinity: held as NaN
            else amax = fmaxf(amax, fabsf(x[j]));
        }
#pragma unroll
        for (int o = HD / 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, kWave));  // lanes of the row's head
        const int e = row_exponent(amax);
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        int w[2] = {0, 0};
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // one rounding, to nearest even; |x| inv <= 448
            w[u] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * u] * inv, x[4 * u + 1] * inv, w[u], false);
            w[u] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * u + 2] * inv, x[4 * u + 3] * inv, w[u], true);
        }
        if (p.row < 0) return;
        *reinterpret_cast<int2*>((p.kv ? pv.vp : pv.kp) + p.row * HD + p.c * 8) = make_int2(w[0], w[1]);
        if (p.c == 0) (p.kv ? pv.ve : pv.ke)[p.row] = static_cast<uint8_t>(e + 127);
    } else {
        if (p.row < 0) return;
        Oct<CT>::store(reinterpret_cast<CT*>(p.kv ? pv.vp : pv.kp) + p.row * HD + p.c * 8, true, x);
    }
}

template <typename T, typename CT, int HD>
__global__ __launch_bounds__(kBlock) void kv_read_k(PageView pv, T* __restrict__ k, T* __restrict__ v, int64_t ld,
                                                    const int64_t* __restrict__ offsets, const int64_t* __restrict__ lens, int B,
                                                    int64_t rows, bool vec) {
    const Piece p = piece<HD>(pv, offsets, lens, B, rows);
    if (!p.live) return;
    float x[8] = {};
    if (p.row >= 0) {
        const char* pool = p.kv ? pv.vp : pv.kp;
        if constexpr (sizeof(CT) == 1)
            e4m3_floats(*reinterpret_cast<const uint2*>(pool + p.row * HD + p.c * 8),
                        exp_scale((p.kv ? pv.ve : pv.ke)[p.row]), x);
        else Oct<CT>::load(reinterpret_cast<const CT*>(pool) + p.row * HD + p.c * 8, true, x);
    }
    Oct<T>::store((p.kv ? v : k) + p.t * ld + p.h * HD + p.c * 8, vec, x);
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

template <typename F>
void launch_rows(const KVPages& c, int64_t B, int64_t T, DType dt, F&& f) {
    const int64_t blocks = (T * 2 * c.kv_heads * (c.head_dim / 8) + kBlock - 1) / kBlock;
    AIC_CHECK(blocks <= INT32_MAX, OutOfRange, "too many rows in one call");
    by_head_dim(c.head_dim, [&](auto hd) {
        const auto g = static_cast<unsigned>(blocks);
        if (dt == DType::Float32 && c.type == DType::Float32) f(float{}, float{}, hd, g);
        else if (dt == DType::Float32) f(float{}, uint8_t{}, hd, g);
        else if (c.type == DType::BFloat16) f(bf16{}, bf16{}, hd, g);
        else f(bf16{}, uint8_t{}, hd, g);
    });
}

}  // namespace

void kv_write(const KVPages& c, const void* k, const void* v, int64_t ld, const int64_t* offsets, const int64_t* lens,
              int64_t B, int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_write", c, k, v, ld, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_write");
    if (B == 0 || T == 0) return;
    const bool vec = aligned16(k, v, ld, static_cast<int64_t>(dtype_size(dt)));
    launch_rows(c, B, T, dt, [&](auto t, auto ct, auto hd, unsigned grid) {
        using X = decltype(t);
        kv_write_k<X, decltype(ct), decltype(hd)::value><<<grid, kBlock, 0, s>>>(
            pv, static_cast<const X*>(k), static_cast<const X*>(v), ld, offsets, lens, static_cast<int>(B), T, vec);
    });
    AIC_LAUNCH_CHECK("kv_write");
}

void kv_read(const KVPages& c, void* k, void* v, int64_t ld, const int64_t* offsets, const int64_t* lens, int64_t B,
             int64_t T, DType dt, hipStream_t s) {
    check_rows("kv_read", c, k, v, ld, offsets, lens, B, T, dt);
    const PageView pv = page_view(c, "kv_read");
    if (B == 0 || T == 0) return;
    const bool vec = aligned16(k, v, ld, static_cast<int64_t>(dtype_size(dt)));
    launch_rows(c, B, T, dt, [&](auto t, auto ct, auto hd, unsigned grid) {
        using X = decltype(t);
        kv_read_k<X, decltype(ct), decltype(hd)::value><<<grid, kBlock, 0, s>>>(
            pv, static_cast<X*>(k), static_cast<X*>(v), ld, offsets, lens, static_cast<int>(B), T, vec);
    });
    AIC_LAUNCH_CHECK("kv_read");
}

}  // namespace aic::hip
