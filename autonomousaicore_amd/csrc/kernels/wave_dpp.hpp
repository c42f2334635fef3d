// Reductions and scans over a wave of 64 lanes in registers: DPP moves inside rows of 16 lanes and gfx950's
// v_permlane16_swap / v_permlane32_swap across them.  A step costs a few cycles where a ds_bpermute
// (what __shfl_xor becomes) costs about a hundred, which counts where a kernel is a chain of them.
#pragma once

#include "common.hpp"

namespace aic::hip {

typedef uint32_t u32_pair __attribute__((ext_vector_type(2)));

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {  // lanes without a source: 0
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, true));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(dpp<CTRL, ROWS>(__float_as_uint(x)));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int dpp(int x) {
    return static_cast<int>(dpp<CTRL, ROWS>(static_cast<uint32_t>(x)));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
    const uint32_t lo = dpp<CTRL, ROWS>(static_cast<uint32_t>(u)), hi = dpp<CTRL, ROWS>(static_cast<uint32_t>(u >> 32));
    return __longlong_as_double(static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo));
}
// The two values of the rows of 16 (N = 16) or halves (N = 32) that face each other, in every lane of both.
template <int N>
__device__ __forceinline__ u32_pair facing(uint32_t x) {
    if constexpr (N == 16) return __builtin_bit_cast(u32_pair, __builtin_amdgcn_permlane16_swap(x, x, false, false));
    else return __builtin_bit_cast(u32_pair, __builtin_amdgcn_permlane32_swap(x, x, false, false));
}

template <int N, typename F>
__device__ __forceinline__ float facing_op(float x, F f) {
    const u32_pair p = facing<N>(__float_as_uint(x));
    return f(__uint_as_float(p.x), __uint_as_float(p.y));
}
template <int N, typename F>
__device__ __forceinline__ int facing_op(int x, F f) {
    const u32_pair p = facing<N>(static_cast<uint32_t>(x));
    return f(static_cast<int>(p.x), static_cast<int>(p.y));
}
template <int N, typename F>
__device__ __forceinline__ double facing_op(double x, F f) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
    const u32_pair lo = facing<N>(static_cast<uint32_t>(u)), hi = facing<N>(static_cast<uint32_t>(u >> 32));
    return f(__longlong_as_double(static_cast<int64_t>((static_cast<uint64_t>(hi.x) << 32) | lo.x)),
             __longlong_as_double(static_cast<int64_t>((static_cast<uint64_t>(hi.y) << 32) | lo.y)));
}

// f over all 64 lanes, in every lane; f associative and commutative.  Neighbours, pairs of a quad, then mirrored
// halves of 8 and of 16 lanes (whose groups already agree), then the rows and halves that face each other.
template <typename T, typename F>
__device__ __forceinline__ T wave_all(T x, F f) {
    x = f(x, dpp<0xb1>(x));   // quad_perm 1 0 3 2
    x = f(x, dpp<0x4e>(x));   // quad_perm 2 3 0 1
    x = f(x, dpp<0x141>(x));  // row_half_mirror
    x = f(x, dpp<0x140>(x));  // row_mirror
    x = facing_op<16>(x, f);
    return facing_op<32>(x, f);
}
// Inclusive running sum over the lanes.
template <typename T>
__device__ __forceinline__ T wave_running_sum(T x) {
    x += dpp<0x111>(x);  // row_shr 1, 2, 4, 8
    x += dpp<0x112>(x);
    x += dpp<0x114>(x);
    x += dpp<0x118>(x);
    x += dpp<0x142, 0xa>(x);  // the last lane of row 0 (2) to row 1 (3)
    x += dpp<0x143, 0xc>(x);  // lane 31 to the upper half
    return x;
}

}  // namespace aic::hip
