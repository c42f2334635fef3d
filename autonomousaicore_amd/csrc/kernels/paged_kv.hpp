// The paged key/value cache as its kernels see it (paged_kv.hip, attention_paged.hip).
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace aic::hip {

// Pools [n_pages][Hkv][ps][hd]: a page holds each head's rows one after another, so that the rows
// of a head that one block reads are whole runs of ps * hd elements.  e4m3 pools carry one byte per
// (page, head, slot): the row is code * 2^(byte - 127).  Powers of two cost no precision that the
// codes have (e4m3 is a floating format: moving a row by up to one binade leaves its relative steps),
// make the values exact in bf16 (from 2^-124 on, where the codes' last digit meets bf16's), and go through the hardware's
// scaled conversion for free.
struct PageView {
    char *kp, *vp;
    uint8_t *ke, *ve;
    const int32_t* table;
    int64_t ld_table;
    int32_t n_pages, ps, Hkv;
    uint32_t mul;  // position / ps = position * mul >> shift, exact below 2^31
    int shift;

    __device__ __forceinline__ int page_index(int pos) const {
        return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(pos)) * mul) >> shift);
    }
    // Row index (in rows of hd elements) of position pos of the sequence whose table row is `tr`, head
    // h; -1 where the table has no valid page there.
    __device__ __forceinline__ int64_t row(const int32_t* tr, int pos, int h) const {
        const int pi = page_index(pos);
        const int page = pi < ld_table ? tr[pi] : -1;
        if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(n_pages)) return -1;
        return (static_cast<int64_t>(page) * Hkv + h) * ps + (pos - pi * ps);
    }
};

// Type, heads and head_dim checked: what sizes are made of.  `what` names the entry in the messages.
void check_cache_shape(const KVPages& c, const char* what);
// All arguments checked, and the view made of them.
PageView page_view(const KVPages& c, const char* what);

constexpr int kBlock = 256;

// Block-wide: how many of offsets[0 .. B-1] are <= t, minus one: the sequence of packed row t, or one
// before it in a run of empty sequences.  One parallel load instead of a chain of dependent ones.
__device__ __forceinline__ int block_sequence(const int64_t* offsets, int B, int64_t t) {
    int n = 0;
    for (int i0 = 0; i0 < B; i0 += kBlock) {
        const int i = i0 + static_cast<int>(threadIdx.x);
        n += __syncthreads_count(i < B && offsets[i] <= t);
    }
    return n - 1;
}

// The eight e4m3 codes of w times the power of two s, as floats: element j in byte j.
__device__ __forceinline__ void e4m3_floats(uint2 w, float s, float (&v)[8]) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w.x, s, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w.x, s, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w.y, s, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w.y, s, true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}
// The same as bf16, to nearest even where code * s has bits below 2^-133.
__device__ __forceinline__ uint4 e4m3_bf16(uint2 w, float s) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, true)));
}
// The largest number that codes and both types share is 240 * 2^120.  From exponent byte kTopByte (2^120) on, a row's larger codes
// are past it: 256 * 2^120 is 2^128, the code nearest to numbers past 248 * 2^120.  They are read as 240 * 2^120, so that finite
// numbers stay finite.  Four codes of a row with such a byte, brought into the range; NaN stays.
constexpr uint32_t kTopByte = 247;
__device__ __forceinline__ uint32_t e4m3_in_range(uint32_t w, uint32_t byte) {
    const uint32_t top = 0x77u - 8u * (min(byte, 254u) - kTopByte);  // 8 codes to a binade
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        const uint32_t c = w >> i & 0x7fu;
        w = c > top && c != 0x7fu ? (w & ~(0x7fu << i)) | top << i : w;
    }
    return w;
}
__device__ __forceinline__ uint4 e4m3_in_range(uint4 w, uint32_t byte) {
    return make_uint4(e4m3_in_range(w.x, byte), e4m3_in_range(w.y, byte), e4m3_in_range(w.z, byte), e4m3_in_range(w.w, byte));
}
// 2^(b - 127) of a stored exponent byte (1 .. 254; 0 and 255 cannot be written and read as 2^-126, 2^127).
__device__ __forceinline__ float exp_scale(uint32_t b) {
    return __uint_as_float(min(max(b, 1u), 254u) << 23);
}

}  // namespace aic::hip
