// What the bf16 flash attention kernels share: swizzled [rows][head_dim] tiles in LDS, the MFMA
// fragments read from them, waits, and the stores of a transposed accumulator.
#pragma once

#include "common.hpp"

namespace aic::hip {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLazyRescale = 8.0f;  // log2 units

typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16_t;

// ---------------------------------------------------------------------------------------
// [rows][HD] bf16 tiles in LDS, 16-byte chunks XOR-swizzled per row.  The swizzle depends
// on row % 16 only and makes both read patterns bank-conflict free: a ds_read_b128 phase
// (16 consecutive rows, one logical chunk) touches 16 distinct bank slots, and each half of
// a ds_read_b64_tr_b16 (4 consecutive rows x 64 bytes) covers the banks exactly once.
// ---------------------------------------------------------------------------------------
template <int HD>
__device__ __forceinline__ int swz(int row) {
    if constexpr (HD == 128) return 4 * (row & 3) | ((row >> 2) & 3);
    else if constexpr (HD == 32) return (row >> 2) & 3;
    else return 4 * ((row >> 1) & 1) | ((row >> 2) & 3);
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4)); }

// MFMA operand fragments of a swizzled [rows][HD] tile, addressed through per-lane byte
// offsets computed once per kernel (every read is then a register base plus an immediate).
//   row(t, rb, kk): lane = row rb + lane%32 (rb a multiple of 32), 8 values of k step kk
//                   along head_dim (ds_read_b128).
//   tr(t, ob, ks):  lane = head_dim column 32ob + lane%32, 8 values along rows in the
//                   permuted order of a 16-row step ks (elements 0..3: rows 16ks + 4h + 0..3,
//                   elements 4..7: rows 16ks + 8 + 4h + 0..3, h = lane / 32), read with two
//                   ds_read_b64_tr_b16: within a group of 16 lanes, output lane i slot j takes
//                   element i % 4 of the 4 values at source lane 4j + i / 4, so source lane
//                   s = 4j + q addresses row (base + j), columns cb' + 4q .. +3.
template <int HD>
struct Frags {
    static constexpr int KS = HD / 16, OB = HD / 32, RB = HD * 2;  // RB: bytes per row
    int row_off[KS];
    int tr_off[OB][2];
    __device__ __forceinline__ void init(int lane = threadIdx.x & 63) {
        const int h = lane >> 5, r = lane & 31;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) row_off[kk] = r * RB + (((2 * kk + h) ^ swz<HD>(r)) << 4);
        const int g = lane >> 4, s = lane & 15, j = s >> 2, q = s & 3;
#pragma unroll
        for (int ob = 0; ob < OB; ++ob)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = 8 * u + 4 * h + j;
                const int col = 32 * ob + 16 * (g & 1) + 4 * q;
                tr_off[ob][u] = row * RB + (((col >> 3) ^ swz<HD>(row)) << 4) + (col & 7) * 2;
            }
    }
    __device__ __forceinline__ bf16x8 row(const char* t, int rb, int kk) const {
        return *reinterpret_cast<const bf16x8*>(t + rb * RB + row_off[kk]);
    }
    __device__ __forceinline__ bf16x8 tr(const char* t, int ob, int ks) const {
        const v4i16_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(t + 16 * ks * RB + tr_off[ob][0]));
        const v4i16_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(t + 16 * ks * RB + tr_off[ob][1]));
        const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
        return __builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, y.x, y.y));
    }
};

__device__ __forceinline__ bf16x8 pack_bf16x8(const f32x16& a, int off) {
    return __builtin_bit_cast(bf16x8, make_uint4(pack_bf16x2(a[off], a[off + 1]), pack_bf16x2(a[off + 2], a[off + 3]),
                                                 pack_bf16x2(a[off + 4], a[off + 5]),
                                                 pack_bf16x2(a[off + 6], a[off + 7])));
}

__device__ __forceinline__ uint4 ldg16(const bf16* p, bool ok) {
    return ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ void zero(f32x16& a) {
#pragma unroll
    for (int e = 0; e < 16; ++e) a[e] = 0.0f;
}

// Writes a [32 rows of head_dim] x [lane = token] accumulator block as token rows.
__device__ __forceinline__ void store_t(bf16* row_ptr, const f32x16& acc, int ob, float mul) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int d0 = ob * 32 + 8 * g + 4 * h;
        *reinterpret_cast<uint2*>(row_ptr + d0) =
            make_uint2(pack_bf16x2(acc[4 * g] * mul, acc[4 * g + 1] * mul),
                       pack_bf16x2(acc[4 * g + 2] * mul, acc[4 * g + 3] * mul));
    }
}

}  // namespace

}  // namespace aic::hip
