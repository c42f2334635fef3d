// Attention over the paged cache, fp32 queries: up to 4 query rows per key/value head (single tokens, a few
// drafted ones).
//
// The formulas are attention_paged.hip's.  A tile of the matrix pipe has 32 rows: with one row in it,
// 128 steps of 64 cycles per 32 keys of 128 cost more than the keys' bytes.  Here hd / 4 lanes hold one key's four values each, q alike; a
// score is four products and a sum over those lanes, which leaves it in all of them, so that the same
// lanes weigh their four values of v without an exchange.  Each group of lanes keeps maximum, sum and
// output of its own keys; they are joined once at the end.  The waves of a block take batches of keys in
// turn and share nothing until then; 8 loads of 1 KB of K and of V per wave are in flight, with enough waves
// per CU to cover them (30 single tokens of 16 heads of 128 on 1000 keys: 66 us, 4.8 TB/s; 16 loads: 71 us; on e4m3
// caches of 4000, where each value is converted, 148 us).  Bound by the bytes of the cache for one and two rows, by the
// vector instructions behind them; tiles of 8 rows would take 24.5 us for 30 tokens of 16 heads of 64 over 2 on 1000
// keys, and the matrix pipe 20.9 us (59 and 52 us for 30 sequences of 7 rows of 12 heads; the other way round, 26 and
// 30 us, for 10 of them).
#include <type_traits>

#include "attention_paged.hpp"

namespace aic::hip {

namespace {

// The sum over groups of L neighbouring lanes, in all of them.
template <int L>
__device__ __forceinline__ float group_sum(float x) {
    x += dpp<0xb1>(x);   // quad_perm 1 0 3 2
    x += dpp<0x4e>(x);   // quad_perm 2 3 0 1
    x += dpp<0x141>(x);  // row_half_mirror
    if constexpr (L >= 16) x += dpp<0x140>(x);  // row_mirror
    if constexpr (L >= 32) x = facing_op<16>(x, [](float a, float b) { return a + b; });
    return x;
}
// f over the lanes that stand at the same place of their groups of L.
template <int L, typename F>
__device__ __forceinline__ float across_groups(float x, F f) {
    if constexpr (L <= 8) x = f(x, dpp<0x128>(x));  // row_ror 8
    if constexpr (L <= 16) x = facing_op<16>(x, f);
    return facing_op<32>(x, f);
}

// Four neighbouring elements of a cached row.
template <typename CT> using Quad = std::conditional_t<kE2<CT>, uint16_t, std::conditional_t<kE4<CT>, uint32_t, float4>>;
__device__ __forceinline__ float4 floats(float4 x, uint32_t) { return x; }
__device__ __forceinline__ float4 floats(uint16_t x, uint32_t e) {
    const float s = exp_scale(e);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, s, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x, s, 1);
    const bool none = e == kNanGroup;
    return make_float4(none ? NAN : a[0], none ? NAN : a[1], none ? NAN : b[0], none ? NAN : b[1]);
}
__device__ __forceinline__ float4 floats(uint32_t x, uint32_t e) {
    const float s = exp_scale(e);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, s, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, s, true);
    return make_float4(a[0], a[1], b[0], b[1]);
}

// RM: rows of a tile.
template <typename CT, int HD, int RM, typename A>
__device__ __forceinline__ bool f32_few_pass(const A& a, int tid, int block, float down) {
    constexpr int L = HD / 4, KI = 64 / L, NI = 8, KB = NI * KI;  // a batch: NI loads of KI keys
    static_assert(KB <= 64, "a lane per key looks its page up");
    __shared__ float2 mls[4][RM];
    __shared__ float os[4][RM][HD];
    const int rest = block / grid_heads(a);
    const int split = rest % a.nsplit, tile = rest / a.nsplit;
    int b, local;
    if (!find_tile<RM>(a, tile, b, local)) return false;
    const int kvh = kv_head(a, b, block % grid_heads(a));
    const Seq sq = wave_sequence(a, b);
    if (std::is_same_v<A, PickedArgs> && sq.n == 0) return false;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = lane / L, d0 = 4 * (lane % L);
    const int rows = sq.n * a.G, r0 = local * RM;

    const int first_pos = sq.len - sq.n + r0 / a.G, last_pos = sq.len - sq.n + (min(r0 + RM, rows) - 1) / a.G;
    int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0, k_hi = last_pos + 1;
    k_lo &= ~63;
    part_of_keys(k_lo, k_hi, split, a.nsplit);

    int lo[RM];         // first key that row r sees
    uint32_t span[RM];  // keys from there on that it sees, up to this split's last
    float4 q[RM], o[RM];
    float m[RM], l[RM];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        const bool real = r0 + r < rows;
        const int tok = (r0 + r) / a.G, pos = real ? sq.len - sq.n + tok : -1;
        lo[r] = a.window > 0 ? max(0, max(pos, 0) - a.window + 1) : 0;
        span[r] = static_cast<uint32_t>(max(min(pos, k_hi - 1) - lo[r] + 1, 0));
        const float* p = static_cast<const float*>(a.q) + (sq.row0 + tok) * a.ldq + static_cast<int64_t>(kvh * a.G + (r0 + r) % a.G) * HD + d0;
        q[r] = !real ? make_float4(0, 0, 0, 0) : a.vec_q ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
        o[r] = make_float4(0, 0, 0, 0);
        m[r] = -INFINITY;
        l[r] = 0.0f;
    }

    if (k_lo < k_hi) {
        const int32_t* tr = a.kv.table + b * a.kv.ld_table;
        // the cached row of a batch's key `lane`; keys past the last are read as the last one: hidden below
        auto row_of = [&](int k0) { return a.kv.row(tr, min(k0 + min(lane, KB - 1), k_hi - 1), kvh); };
        int64_t row = row_of(k_lo + wave * KB);
        for (int k0 = k_lo + wave * KB; k0 < k_hi; k0 += 4 * KB) {
            Quad<CT> kx[NI], vx[NI];
            [[maybe_unused]] uint32_t ke[NI], ve[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int64_t at = __shfl(row, i * KI + grp, 64);
                const char* none = reinterpret_cast<const char*>(&kNoPage);
                const int64_t byte = at * kRowBytes<CT, HD> + d0 * 16 / kPer16<CT>;
                kx[i] = *reinterpret_cast<const Quad<CT>*>(at >= 0 ? a.kv.kp + byte : none);
                vx[i] = *reinterpret_cast<const Quad<CT>*>(at >= 0 ? a.kv.vp + byte : none);
                if constexpr (kE2<CT>) {
                    ke[i] = at >= 0 ? a.kv.ke[at * (HD / kGroup) + d0 / kGroup] : kNanGroup;
                    ve[i] = at >= 0 ? a.kv.ve[at * (HD / kGroup) + d0 / kGroup] : kNanGroup;
                } else if constexpr (kE4<CT>) {
                    ke[i] = at >= 0 ? a.kv.ke[at] : 127;
                    ve[i] = at >= 0 ? a.kv.ve[at] : 127;
                } else {
                    ke[i] = ve[i] = 0;
                }
            }
            row = row_of(k0 + 4 * KB);
            if constexpr (kE4<CT>) {
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < NI; ++i) most = max(most, max(ke[i], ve[i]));
                if (__builtin_expect(most >= kTopByte, 0)) {
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        if (ke[i] >= kTopByte) kx[i] = e4m3_in_range(kx[i], ke[i]);
                        if (ve[i] >= kTopByte) vx[i] = e4m3_in_range(vx[i], ve[i]);
                    }
                }
            }
            const bool open = k0 + KB - 1 <= first_pos && k0 + KB <= k_hi && (a.window <= 0 || k0 > last_pos - a.window);
#pragma unroll
            for (int r = 0; r < RM; ++r) {
                float s[NI], mx = m[r];
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const float4 k = floats(kx[i], ke[i]);
                    s[i] = group_sum<L>(fmaf(k.x, q[r].x, fmaf(k.y, q[r].y, fmaf(k.z, q[r].z, k.w * q[r].w))));
                    if (!open) s[i] = static_cast<uint32_t>(k0 + i * KI + grp - lo[r]) < span[r] ? s[i] : -INFINITY;
                    mx = fmaxf(mx, s[i]);
                }
                // keys that this group's row has seen only scores of -infinity from count from zero; alpha is 1 exactly where the
                // maximum stands (an fma with off would leave off's rounding error in it, once per batch of keys)
                const float off = mx == -INFINITY ? -down : fmaf(-mx, a.c, -down);
                const float alpha = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[r] - mx) * a.c);
                m[r] = mx;
                // the batch by itself first: added one by one, keys lighter than half a step of the sum would all be lost
                float lb = 0.0f;
                float4 ob = make_float4(0, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const float w = weight(s[i], a.c, off);
                    const float4 v = floats(vx[i], ve[i]);
                    lb += w;
                    const float4 y = make_float4(fmaf(w, v.x, ob.x), fmaf(w, v.y, ob.y), fmaf(w, v.z, ob.z), fmaf(w, v.w, ob.w));
                    // a hidden key adds nothing, also where its v is an infinity or NaN
                    const bool seen = open || static_cast<uint32_t>(k0 + i * KI + grp - lo[r]) < span[r];
                    ob.x = seen ? y.x : ob.x, ob.y = seen ? y.y : ob.y, ob.z = seen ? y.z : ob.z, ob.w = seen ? y.w : ob.w;
                }
                l[r] = fmaf(l[r], alpha, lb);
                o[r] = make_float4(fmaf(o[r].x, alpha, ob.x), fmaf(o[r].y, alpha, ob.y), fmaf(o[r].z, alpha, ob.z), fmaf(o[r].w, alpha, ob.w));
            }
        }
    }
    // the groups of a wave, then the waves: M = max m_i, o = sum 2^((m_i - M) c) o_i, l alike.  True where a sum of this thread's has
    // left fp32's range.
    const bool again = down > 0.0f;
    bool over = false;
    auto add = [](float x, float y) { return x + y; };
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        const float M = across_groups<L>(m[r], [](float x, float y) { return fmaxf(x, y); });
        const float f = __builtin_amdgcn_exp2f((m[r] - (M == -INFINITY ? 0.0f : M)) * a.c);
        const float lw = across_groups<L>(l[r] * f, add);
        const float4 x = make_float4(across_groups<L>(o[r].x * f, add), across_groups<L>(o[r].y * f, add),
                                     across_groups<L>(o[r].z * f, add), across_groups<L>(o[r].w * f, add));
        if (lane == 0) mls[wave][r] = make_float2(M, lw);
        if (lane < L) *reinterpret_cast<float4*>(&os[wave][r][d0]) = x;
    }
    __syncthreads();
    for (int i = tid; i < RM * HD; i += 256) {
        const int r = i / HD, d = i % HD;
        if (r0 + r >= rows) break;
        const int tok = (r0 + r) / a.G, head = kvh * a.G + (r0 + r) % a.G, pos = sq.len - sq.n + tok;
        const int64_t t = sq.row0 + tok;
        const int first = a.window > 0 ? max(0, max(pos, 0) - a.window + 1) : 0, last = min(pos, k_hi - 1);
        const bool empty = last < first || last < k_lo;
        float M = -INFINITY, lw = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, mls[w][r].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f((mls[w][r].x - (M == -INFINITY ? 0.0f : M)) * a.c);
            lw = fmaf(f, mls[w][r].y, lw);
            x = fmaf(f, os[w][r][d], x);
        }
        Range range;
        range.look(x);
        over |= !empty && range.left(lw);
        const float y = empty ? 0.0f : x * (1.0f / lw);  // lw == 0: only scores of -infinity, 0 / 0 = NaN
        float* to;
        if (a.nsplit > 1) {
            const int64_t at = (static_cast<int64_t>(split) * a.T + t) * a.H + head;
            if (d == 0 && !again) a.part_ml[at] = make_float2(M, empty ? 0.0f : lw == 0.0f ? -1.0f : lw);
            to = a.part_o + at * HD + d;
        } else {
            if (a.lse && d == 0 && !again) a.lse[t * a.H + head] = empty ? -INFINITY : log_sum(M, lw, a.c);
            to = static_cast<float*>(a.o) + t * a.ldo + static_cast<int64_t>(head) * HD + d;
        }
        if (!again || !(fabsf(*to) < INFINITY)) *to = y;
    }
    return over;
}

template <typename CT, int HD, int RM, typename A>
__global__ __launch_bounds__(256) void attn_paged_f32_few_k(A a) {
    one_or_two_passes(a, [](const A& args, int tid, int block, float down) { return f32_few_pass<CT, HD, RM>(args, tid, block, down); });
}

}  // namespace

// Row tiles of 1, 2 or 4 rows for up to 4 rows, 0: for the matrix pipe.
int f32_few_rows(int64_t max_q, int64_t G) {
    const int64_t rows = max_q * G;
    return rows > 4 ? 0 : rows > 2 ? 4 : rows > 1 ? 2 : 1;
}

template <typename A>
void attn_paged_f32_few(const A& a, int rows, DType type, int head_dim, unsigned blocks, hipStream_t s) {
    auto run = [&](auto ct, auto hd) {
        using C = decltype(ct);
        constexpr int D = decltype(hd)::value;
        if (rows == 1) attn_paged_f32_few_k<C, D, 1><<<blocks, 256, 0, s>>>(a);
        else if (rows == 2) attn_paged_f32_few_k<C, D, 2><<<blocks, 256, 0, s>>>(a);
        else attn_paged_f32_few_k<C, D, 4><<<blocks, 256, 0, s>>>(a);
        AIC_LAUNCH_CHECK("attn_paged few, fp32");
    };
    by_cache_type<float>(type, [&](auto ct) {
        if (head_dim == 32) run(ct, std::integral_constant<int, 32>{});
        else if (head_dim == 64) run(ct, std::integral_constant<int, 64>{});
        else run(ct, std::integral_constant<int, 128>{});
    });
}

template void attn_paged_f32_few(const PagedArgs&, int, DType, int, unsigned, hipStream_t);
template void attn_paged_f32_few(const PickedArgs&, int, DType, int, unsigned, hipStream_t);

}  // namespace aic::hip
