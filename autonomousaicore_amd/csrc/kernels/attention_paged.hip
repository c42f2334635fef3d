// Attention of a chunk of new tokens per sequence over the paged key/value cache.
//
// Sequence b's queries are the packed rows offsets[b] .. offsets[b+1]; row i of n stands at position
// pos = lens[b] - n + i and sees the cached keys max(0, pos - window + 1) .. pos (window 0: from 0).
//   s_j = scale q . k_j,   o = sum_j softmax(s)_j v_j,   lse = log sum_j exp s_j
// in one pass over the keys with the running maximum and sum in fp32.  The G = H / Hkv query heads of
// one key/value head share its rows: a tile's query rows are (token, head) pairs, row r being token
// r / G and head kvh G + r % G, so the cache is read once per key/value head.
//
// A wave holds 32 query rows; scores come out as S^T = K Q^T, so a lane owns one query row (its half
// of the wave splits the keys), maximum and sum need one exchange with lane ^ 32, and P feeds
// O^T += V^T P^T from the accumulator registers.  fp32 runs v_mfma_f32_32x32x2_f32 and keeps P in
// fp32; bf16 runs v_mfma_f32_32x32x16_bf16 with P rounded to bf16 (each weight off by at most 2^-8 of
// itself, as an output is by its own rounding; the sum l adds them unrounded).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_tiles.hpp"
#include "paged_kv.hpp"
#include "../runtime/memory_pool.hpp"

namespace aic::hip {

namespace {

struct PagedArgs {
    PageView kv;
    const void* q;
    void* o;
    float* lse;
    int64_t ldq, ldo, T;
    const int64_t *offsets, *lens;
    int B, H, G, window;
    float c;         // scale in log2 units
    int chunk;       // keys of one split (0: one split over all of them)
    int nsplit;
    float2* part_ml;  // [nsplit][T][H]: maximum, sum (-1: only scores of -infinity)
    float* part_o;    // [nsplit][T][H][hd]
    bool vec_q, vec_o;
};

// All ones: a NaN in fp32, bf16 and e4m3.  Keys whose page id is out of range are read from here, so
// that exactly the queries that would see them become NaN.
__device__ const uint4 kNoPage = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};

constexpr int64_t kMaxLen = INT32_MAX - 4095;  // positions and a tile past them fit in 32 bits

// Weights are held times 2^-40: at most 2^8 2^-40 each, so that the sums over 2^31 keys stay below
// the largest v, and a finite v never overflows before the division by l.  Exact, and it costs weights
// below 2^-86 of the maximum.  bf16 takes it in exp2's argument, whose last bits (2^-19 there) are far below
// the weight's rounding; fp32 multiplies.
constexpr float kDown = 40.0f;
template <typename T>
__device__ __forceinline__ float weight(float s, float c, float off) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(fmaf(s, c, off - kDown));
    else return __builtin_amdgcn_exp2f(fmaf(s, c, off)) * 0x1p-40f;
}
__device__ __forceinline__ float log_sum(float m, float l, float c) { return (m * c + log2f(l * 0x1p40f)) * kLn2; }

struct Seq {
    int64_t row0;  // first packed row
    int n, len;    // queries, cached keys
};
__device__ __forceinline__ Seq sequence(const PagedArgs& a, int b) {
    const int64_t lo = min(max(a.offsets[b], int64_t{0}), a.T), hi = min(max(a.offsets[b + 1], lo), a.T);
    return {lo, static_cast<int>(hi - lo), static_cast<int>(min(max(a.lens[b], int64_t{0}), kMaxLen))};
}

// Tile `tile` of the batch cut into tiles of R query rows: its sequence and the tile's place in it.
// Every wave finds it by itself: 64 sequences per step, their tile counts added up across lanes.
template <int R>
__device__ __forceinline__ bool find_tile(const PagedArgs& a, int tile, int& b, int& local) {
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        int tiles = 0;
        if (b0 + lane < a.B) tiles = static_cast<int>((static_cast<int64_t>(sequence(a, b0 + lane).n) * a.G + R - 1) / R);
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o, 64);
            if (lane >= o) upto += x;
        }
        const uint64_t past = __ballot(tile < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            b = __builtin_amdgcn_readfirstlane(b0 + l);
            local = __builtin_amdgcn_readfirstlane(tile - (__shfl(upto, l, 64) - __shfl(tiles, l, 64)));
            return true;
        }
        tile -= __shfl(upto, 63, 64);
    }
    return false;
}

// ------------------------------------------------------------------------------- tiles
// [KT][HD] tiles of T in LDS, 16-byte chunks swizzled per row.
template <typename T, int HD>
__device__ __forceinline__ int chunk_at(int row, int ch) {
    if constexpr (sizeof(T) == 2) return row * HD * 2 + ((ch ^ swz<HD>(row)) << 4);
    // a ds_read_b128 phase reads one chunk of 16 consecutive rows: 16 different bank groups
    else return row * HD * 4 + ((ch ^ (HD == 32 ? (row >> 1) & 7 : row & 15)) << 4);
}

template <typename CT> __device__ __forceinline__ bool any_non_finite(uint4 x);
template <> __device__ __forceinline__ bool any_non_finite<bf16>(uint4 x) {
    bool bad = false;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f800000u) == 0x7f800000u || (w[i] & 0x7f80u) == 0x7f80u;
    return bad;
}
template <> __device__ __forceinline__ bool any_non_finite<float>(uint4 x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
    return bad;
}

// The four V values at columns d0 .. d0+3 of a tile's row.
template <typename T, int HD>
__device__ __forceinline__ float4 v4_at(const char* tile, int row, int d0) {
    if constexpr (sizeof(T) == 2) {
        const bf16x4 x = *reinterpret_cast<const bf16x4*>(tile + chunk_at<T, HD>(row, d0 >> 3) + (d0 & 7) * 2);
        return make_float4(bf2f(x[0]), bf2f(x[1]), bf2f(x[2]), bf2f(x[3]));
    } else {
        return *reinterpret_cast<const float4*>(tile + chunk_at<T, HD>(row, d0 >> 2));
    }
}

// The running state of 32 query rows: lane owns row lane % 32.
template <int OB>
struct Rows {
    f32x16 o[OB];
    float m = -INFINITY, l = 0.0f;
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int i = 0; i < OB; ++i) zero(o[i]);
    }
    // A tile's row maximum joins the reference maximum, which moves only by more than 2^8.
    __device__ __forceinline__ void absorb(float mx, float c) {
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const bool grow = (mx - m) * c > kLazyRescale;
        if (__any(grow)) {
            const float m_new = grow ? mx : m;
            const float alpha = m == -INFINITY ? 0.0f : grow ? __builtin_amdgcn_exp2f((m - m_new) * c) : 1.0f;
            l *= alpha;
#pragma unroll
            for (int ob = 0; ob < OB; ++ob)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[ob][e] *= alpha;
            m = m_new;
        }
    }
    // -m in log2 units; a row that has seen only scores of -infinity counts from zero
    __device__ __forceinline__ float offset(float c) const { return m == -INFINITY ? 0.0f : -m * c; }
};

// o += sum over the tile's keys of p v, key by key and only where the row sees the key: a hidden key has
// weight zero in the matrix product, and zero times an infinity or NaN in its v is NaN.  For tiles
// that hold both a hidden key and a non-finite v.  p[jb][e] is key 32 jb + 8 (e >> 2) + 4 h + (e & 3).
template <typename T, int HD, int JB, typename Seen>
__device__ __forceinline__ void add_seen_rows(f32x16 (&o)[HD / 32], const f32x16 (&p)[JB], const char* vt, Seen seen) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll 1
        for (int e = 0; e < 16; ++e) {
            const float mine = p[jb][e], other = __shfl_xor(mine, 32, 64);
#pragma unroll 1
            for (int hh = 0; hh < 2; ++hh) {
                const int key = 32 * jb + 8 * (e >> 2) + 4 * hh + (e & 3);
                const float w = hh == h ? mine : other;
                const bool s = seen(key);
#pragma unroll
                for (int ob = 0; ob < HD / 32; ++ob)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 x = v4_at<T, HD>(vt, key, 32 * ob + 8 * g + 4 * h);
                        const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            o[ob][4 * g + u] = s ? fmaf(w, y[u], o[ob][4 * g + u]) : o[ob][4 * g + u];
                    }
            }
        }
}

// Output of one query row: the lane's half of the head dimension.
template <typename T, int HD>
__device__ __forceinline__ void store_row(const PagedArgs& a, const Rows<HD / 32>& r, int64_t t, int head, bool empty,
                                          int split) {
    constexpr int OB = HD / 32;
    const int h = (threadIdx.x & 63) >> 5;
    if (a.nsplit > 1) {
        const int64_t i = (static_cast<int64_t>(split) * a.T + t) * a.H + head;
        if (h == 0) a.part_ml[i] = make_float2(r.m, empty ? 0.0f : r.l == 0.0f ? -1.0f : r.l);
        if (empty) return;
        float* p = a.part_o + i * HD;
#pragma unroll
        for (int ob = 0; ob < OB; ++ob)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(p + ob * 32 + 8 * g + 4 * h) =
                    make_float4(r.o[ob][4 * g], r.o[ob][4 * g + 1], r.o[ob][4 * g + 2], r.o[ob][4 * g + 3]);
        return;
    }
    const float inv = empty ? 0.0f : 1.0f / r.l;  // l == 0: only scores of -infinity, 0 / 0 = NaN below
    T* op = static_cast<T*>(a.o) + t * a.ldo + static_cast<int64_t>(head) * HD;
#pragma unroll
    for (int ob = 0; ob < OB; ++ob) {
        if constexpr (sizeof(T) == 2) {
            if (a.vec_o) {
                store_t(op, r.o[ob], ob, inv);
                continue;
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d0 = ob * 32 + 8 * g + 4 * h;
            if (sizeof(T) == 4 && a.vec_o) {
                *reinterpret_cast<float4*>(op + d0) = make_float4(r.o[ob][4 * g] * inv, r.o[ob][4 * g + 1] * inv,
                                                                  r.o[ob][4 * g + 2] * inv, r.o[ob][4 * g + 3] * inv);
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) st(op, d0 + u, r.o[ob][4 * g + u] * inv);
            }
        }
    }
    if (a.lse && h == 0) a.lse[t * a.H + head] = empty ? -INFINITY : log_sum(r.m, r.l, a.c);
}

// ------------------------------------------------------------------- the general kernel
// One block: 128 query rows (4 waves x 32) of one key/value head, over tiles of KT keys staged through
// registers (the next tile's loads are in flight during this one's products).
template <typename T, typename CT, int HD>
__global__ __launch_bounds__(256) void attn_paged_k(PagedArgs a) {
    constexpr int KT = sizeof(T) == 2 ? 64 : 32, JB = KT / 32, OB = HD / 32;
    constexpr int UPR = HD * sizeof(CT) / 16;        // 16-byte units of a cached row
    constexpr int NU = (KT * UPR + 255) / 256;       // units of a tile per thread
    constexpr bool E4 = sizeof(CT) == 1;
    __shared__ __attribute__((aligned(16))) char ks[KT * HD * sizeof(T)];
    __shared__ __attribute__((aligned(16))) char vs[KT * HD * sizeof(T)];

    const int Hkv = a.kv.Hkv;
    const int kvh = static_cast<int>(blockIdx.x) % Hkv;
    const int rest = static_cast<int>(blockIdx.x) / Hkv;
    const int split = rest % a.nsplit;
    int b, local;
    if (!find_tile<128>(a, rest / a.nsplit, b, local)) return;
    const Seq sq = sequence(a, b);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane >> 5;
    const int rows = sq.n * a.G, r0 = local * 128, r = r0 + wave * 32 + (lane & 31);
    const bool real = r < rows;
    const int tok = real ? r / a.G : 0, head = kvh * a.G + (real ? r % a.G : 0);
    const int64_t t = sq.row0 + tok;
    const int hi = real ? sq.len - sq.n + tok : -1;                    // last key this row sees
    const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;  // first

    // keys of the block: what its first row sees first .. what its last row sees last, of this split
    const int first_pos = sq.len - sq.n + r0 / a.G, last_pos = sq.len - sq.n + (min(r0 + 128, rows) - 1) / a.G;
    int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0, k_hi = last_pos + 1;
    if (a.chunk > 0) {
        k_lo = max(k_lo, split * a.chunk);
        if (split + 1 < a.nsplit) k_hi = min(k_hi, (split + 1) * a.chunk);
    }
    k_lo &= ~(KT - 1);
    const uint32_t span = static_cast<uint32_t>(max(min(hi, k_hi - 1) - lo + 1, 0));  // keys from lo on that it sees here
    const bool empty = span == 0 || min(hi, k_hi - 1) < k_lo;                          // of this split

    Rows<OB> st_;
    st_.init();
    if (k_lo < k_hi) {
        // Q fragments: bf16 8 values at 16 kk + 8 h; fp32 4 values at 8 c + 4 h
        constexpr int KS = HD / 16, KF = HD / 8;
        [[maybe_unused]] bf16x8 qb[KS];
        [[maybe_unused]] float4 qf[KF];
        const T* qp = static_cast<const T*>(a.q) + t * a.ldq + static_cast<int64_t>(head) * HD;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                if (a.vec_q) qb[kk] = __builtin_bit_cast(bf16x8, ldg16(qp + 16 * kk + 8 * hl, real));
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) qb[kk][j] = real ? qp[16 * kk + 8 * hl + j] : f2bf(0.0f);
            }
        } else {
#pragma unroll
            for (int cc = 0; cc < KF; ++cc) {
                const T* p = qp + 8 * cc + 4 * hl;
                qf[cc] = !real ? make_float4(0, 0, 0, 0) : a.vec_q ? *reinterpret_cast<const float4*>(p)
                                                                   : make_float4(p[0], p[1], p[2], p[3]);
            }
        }
        [[maybe_unused]] Frags<sizeof(T) == 2 ? HD : 32> F;
        if constexpr (sizeof(T) == 2) F.init();

        uint4 rk[NU], rv[NU];
        [[maybe_unused]] uint32_t xk[NU], xv[NU];  // exponent bytes
        const int32_t* tr = a.kv.table + b * a.kv.ld_table;
        auto load = [&](int k0) {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int u = i * 256 + static_cast<int>(threadIdx.x);
                // keys past the last are read as the last one: hidden below
                const int key = min(k0 + min(u / UPR, KT - 1), k_hi - 1);
                const int64_t row = a.kv.row(tr, key, kvh);
                const int64_t at = row * (UPR * 16) + (u % UPR) * 16;
                const char* none = reinterpret_cast<const char*>(&kNoPage);
                rk[i] = *reinterpret_cast<const uint4*>(row >= 0 ? a.kv.kp + at : none);
                rv[i] = *reinterpret_cast<const uint4*>(row >= 0 ? a.kv.vp + at : none);
                if constexpr (E4) {
                    xk[i] = row >= 0 ? a.kv.ke[row] : 127;
                    xv[i] = row >= 0 ? a.kv.ve[row] : 127;
                }
            }
        };
        auto put = [&](char* tile, int row, int c, uint4 x, [[maybe_unused]] uint32_t xe) {
            if constexpr (!E4) {
                *reinterpret_cast<uint4*>(tile + chunk_at<T, HD>(row, c)) = x;
            } else {
                const float s = exp_scale(xe);
                const uint2 w[2] = {make_uint2(x.x, x.y), make_uint2(x.z, x.w)};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (sizeof(T) == 2) {
                        *reinterpret_cast<uint4*>(tile + chunk_at<T, HD>(row, 2 * c + j)) = e4m3_bf16(w[j], s);
                    } else {
                        float y[8];
                        e4m3_floats(w[j], s, y);
                        *reinterpret_cast<float4*>(tile + chunk_at<T, HD>(row, 4 * c + 2 * j)) =
                            make_float4(y[0], y[1], y[2], y[3]);
                        *reinterpret_cast<float4*>(tile + chunk_at<T, HD>(row, 4 * c + 2 * j + 1)) =
                            make_float4(y[4], y[5], y[6], y[7]);
                    }
                }
            }
        };
        // this thread's part of the V tile in registers holds an infinity or NaN
        auto bad_v = [&] {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                if constexpr (E4) {
                    const uint32_t w[4] = {rv[i].x, rv[i].y, rv[i].z, rv[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int by = 0; by < 4; ++by) bad |= ((w[j] >> (8 * by)) & 0x7fu) == 0x7fu;
                } else {
                    bad |= any_non_finite<CT>(rv[i]);
                }
            }
            return bad;
        };

        load(k_lo);
        for (int k0 = k_lo; k0 < k_hi; k0 += KT) {
            // every row of the block sees every key of the tile?
            const bool open = k0 + KT - 1 <= first_pos && k0 + KT <= k_hi && r0 + 128 <= rows &&
                              (a.window <= 0 || k0 > last_pos - a.window);
            const int poison = __syncthreads_or(!open && bad_v());  // also: everyone is done with the last tile
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int u = i * 256 + static_cast<int>(threadIdx.x);
                if (u < KT * UPR) {
                    put(ks, u / UPR, u % UPR, rk[i], E4 ? xk[i] : 0);
                    put(vs, u / UPR, u % UPR, rv[i], E4 ? xv[i] : 0);
                }
            }
            __syncthreads();
            if (k0 + KT < k_hi) load(k0 + KT);

            f32x16 sc[JB];
#pragma unroll
            for (int jb = 0; jb < JB; ++jb) {
                zero(sc[jb]);
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk)
                        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.row(ks, 32 * jb, kk), qb[kk], sc[jb], 0, 0, 0);
                } else {
#pragma unroll
                    for (int cc = 0; cc < KF; ++cc) {
                        const float4 x = *reinterpret_cast<const float4*>(
                            ks + chunk_at<T, HD>(32 * jb + (lane & 31), 2 * cc + hl));
                        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, qf[cc].x, sc[jb], 0, 0, 0);
                        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, qf[cc].y, sc[jb], 0, 0, 0);
                        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, qf[cc].z, sc[jb], 0, 0, 0);
                        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, qf[cc].w, sc[jb], 0, 0, 0);
                    }
                }
            }
            auto seen = [&](int j) { return static_cast<uint32_t>(k0 + j - lo) < span; };
            if (!open)
#pragma unroll
                for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sc[jb][e] = seen(32 * jb + 8 * (e >> 2) + 4 * hl + (e & 3)) ? sc[jb][e] : -INFINITY;
            float mx = -INFINITY;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[jb][e]);
            st_.absorb(mx, a.c);
            const float off = st_.offset(a.c);
            float sum = 0.0f;
#pragma unroll
            for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[jb][e] = weight<T>(sc[jb][e], a.c, off);
                    sum += sc[jb][e];
                }
            st_.l += sum + __shfl_xor(sum, 32, 64);
            if (poison) {
                add_seen_rows<T, HD, JB>(st_.o, sc, vs, seen);
            } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int s = 0; s < KT / 16; ++s) {
                    const bf16x8 p = pack_bf16x8(sc[s >> 1], 8 * (s & 1));
#pragma unroll
                    for (int ob = 0; ob < OB; ++ob)
                        st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.tr(vs, ob, s), p, st_.o[ob], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int jb = 0; jb < JB; ++jb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
#pragma unroll
                        for (int ob = 0; ob < OB; ++ob) {
                            const int d = 32 * ob + (lane & 31), row = 32 * jb + 8 * (e >> 2) + 4 * hl + (e & 3);
                            const float x = *reinterpret_cast<const float*>(vs + chunk_at<T, HD>(row, d >> 2) + (d & 3) * 4);
                            st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, sc[jb][e], st_.o[ob], 0, 0, 0);
                        }
            }
        }
    }
    if (real) store_row<T, HD>(a, st_, t, head, empty, split);
}

// ------------------------------------------------------------------------- joining splits
// One wave per (token, head): M = max m_s, o = sum_s 2^((m_s - M) c) o_s / sum_s 2^((m_s - M) c) l_s.
template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_paged_join_k(PagedArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (i >= a.T * a.H) return;
    const int64_t t = i / a.H;
    if (t < a.offsets[0] || t >= a.offsets[a.B]) return;  // rows of no sequence stay as they are
    const int lane = threadIdx.x & 63;
    const int64_t step = a.T * a.H;
    float M = -INFINITY;
    bool any = false;
    for (int s = 0; s < a.nsplit; ++s) {
        const float2 ml = a.part_ml[s * step + i];
        if (ml.y != 0.0f) {
            any = true;
            M = fmaxf(M, ml.x);
        }
    }
    const float base = M == -INFINITY ? 0.0f : M;
    constexpr int PL = HD >= 64 ? HD / 64 : 1;
    float o[PL] = {}, l = 0.0f;
    for (int s = 0; s < a.nsplit; ++s) {
        const float2 ml = a.part_ml[s * step + i];
        if (ml.y == 0.0f || ml.y == -1.0f) continue;
        const float w = __builtin_amdgcn_exp2f((ml.x - base) * a.c);
        l = fmaf(w, ml.y, l);
#pragma unroll
        for (int u = 0; u < PL; ++u)
            if (lane * PL < HD) o[u] = fmaf(w, a.part_o[(s * step + i) * HD + lane * PL + u], o[u]);
    }
    const float inv = any ? 1.0f / l : 0.0f;
    T* op = static_cast<T*>(a.o) + t * a.ldo + (i % a.H) * HD;
#pragma unroll
    for (int u = 0; u < PL; ++u)
        if (lane * PL < HD) st(op, lane * PL + u, o[u] * inv);
    if (a.lse && lane == 0) a.lse[i] = any ? log_sum(base, l, a.c) : -INFINITY;
}

// --------------------------------------------------------------------------- the launch
int64_t tile_bound(int64_t T, int64_t G, int64_t B, int64_t R) { return T * G / R + std::min(B, T); }

constexpr int64_t kFill = 512;     // blocks that fill the card twice over
constexpr int64_t kMinChunk = 256;  // keys of a split, at least

struct Plan {
    int64_t tiles, nsplit, chunk;
};
// Splits over the keys where the query tiles alone do not fill the card: equal chunks of a multiple of 64
// keys that give about kFill blocks.
Plan plan(int64_t B, int64_t T, int64_t max_len, int64_t H, int64_t Hkv, int64_t) {
    Plan p{tile_bound(T, H / Hkv, B, 128), 1, 0};
    const int64_t blocks = p.tiles * Hkv;
    const int64_t want = std::min(kFill / std::max<int64_t>(blocks, 1), max_len / kMinChunk);
    if (want > 1) {
        p.chunk = ((max_len + want - 1) / want + 63) / 64 * 64;
        p.nsplit = (max_len + p.chunk - 1) / p.chunk;
        if (p.nsplit <= 1) p = {p.tiles, 1, 0};
    }
    return p;
}
int64_t plan_bytes(const Plan& p, int64_t T, int64_t H, int64_t hd) {
    return p.nsplit <= 1 ? 0 : p.nsplit * T * H * (hd + 2) * 4;
}

void check_sizes(const KVPages& c, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H) {
    AIC_CHECK(B >= 0 && T >= 0 && B <= INT32_MAX && T <= INT32_MAX, InvalidArgument, "attn_paged: B and T must be 0 .. 2^31 - 1");
    AIC_CHECK(max_q >= 0 && max_len >= 0 && max_len <= kMaxLen, InvalidArgument,
              "attn_paged: max_q must not be negative and max_len must be 0 .. ", kMaxLen);
    AIC_CHECK(c.kv_heads >= 1 && H >= 1 && H % c.kv_heads == 0, ShapeMismatch, "attn_paged: ", H, " query heads over ", c.kv_heads,
              " key/value heads");
    AIC_CHECK(T * (H / c.kv_heads) <= kMaxLen, OutOfRange, "attn_paged: more than ", kMaxLen, " query rows per key/value head");
}

}  // namespace

int64_t attn_paged_workspace(const KVPages& c, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H) {
    check_sizes(c, B, T, max_q, max_len, H);
    if (B == 0 || T == 0) return 0;
    return plan_bytes(plan(B, T, max_len, H, c.kv_heads, max_q), T, H, c.head_dim);
}

void attn_paged(const KVPages& c, const void* q, int64_t ld_q, void* o, int64_t ld_o, float* lse, const int64_t* offsets,
                const int64_t* lens, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H, int64_t window,
                float scale, void* workspace, int64_t workspace_bytes, DType dt, hipStream_t s) {
    check_sizes(c, B, T, max_q, max_len, H);
    AIC_CHECK(dt == DType::Float32 || dt == DType::BFloat16, DTypeMismatch, "attn_paged: queries are float32 or bfloat16");
    AIC_CHECK(c.type == dt || c.type == DType::UInt8, DTypeMismatch, "attn_paged: queries of ", dtype_name(dt),
              " with a cache of ", dtype_name(c.type));
    const PageView pv = page_view(c, "attn_paged");
    AIC_CHECK(ld_q >= H * c.head_dim && ld_o >= H * c.head_dim, InvalidArgument,
              "attn_paged: leading dimension below heads * head_dim");
    AIC_CHECK(std::isfinite(scale) && scale > 0.0f, InvalidArgument, "attn_paged: scale must be positive and finite, got ", scale);
    AIC_CHECK(window >= 0, InvalidArgument, "attn_paged: window must not be negative, got ", window);
    AIC_CHECK(workspace_bytes >= 0, InvalidArgument, "attn_paged: negative workspace size");
    if (B == 0 || T == 0) return;
    AIC_CHECK(q && o && offsets && lens, InvalidArgument, "attn_paged: null pointer");

    const int64_t size = static_cast<int64_t>(dtype_size(dt));
    PagedArgs a{};
    a.kv = pv;
    a.q = q, a.o = o, a.lse = lse;
    a.ldq = ld_q, a.ldo = ld_o, a.T = T;
    a.offsets = offsets, a.lens = lens;
    a.B = static_cast<int>(B), a.H = static_cast<int>(H), a.G = static_cast<int>(H / c.kv_heads);
    a.window = static_cast<int>(std::min<int64_t>(window, INT32_MAX));
    a.c = scale * kLog2e;
    a.vec_q = reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld_q * size % 16 == 0;
    a.vec_o = reinterpret_cast<uintptr_t>(o) % 16 == 0 && ld_o * size % 16 == 0;

    Plan p = plan(B, T, max_len, H, c.kv_heads, max_q);
    const int64_t need = plan_bytes(p, T, H, c.head_dim);
    const StreamScratchUse use(s);
    if (need > 0) {
        if (workspace) {
            AIC_CHECK(workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, InvalidArgument,
                      "attn_paged: the workspace must be 16-byte aligned and hold ", need, " bytes, got ", workspace_bytes);
        } else if (stream_scratch_ready(s)) {
            workspace = stream_scratch(static_cast<size_t>(need), s);
        } else {
            p = {p.tiles, 1, 0};  // captured without a workspace of its own
        }
    }
    a.nsplit = static_cast<int>(p.nsplit);
    a.chunk = static_cast<int>(p.chunk);
    if (p.nsplit > 1) {
        a.part_o = static_cast<float*>(workspace);
        a.part_ml = reinterpret_cast<float2*>(a.part_o + p.nsplit * T * H * c.head_dim);
    }
    const int64_t blocks = p.tiles * c.kv_heads * p.nsplit;
    AIC_CHECK(blocks <= INT32_MAX, OutOfRange, "attn_paged: too many rows in one call");
    auto run = [&](auto t, auto ct, auto hd) {
        using X = decltype(t);
        constexpr int D = decltype(hd)::value;
        attn_paged_k<X, decltype(ct), D><<<static_cast<unsigned>(blocks), 256, 0, s>>>(a);
        AIC_LAUNCH_CHECK("attn_paged");
        if (a.nsplit > 1) {
            const int64_t joins = (T * H + 3) / 4;
            AIC_CHECK(joins <= INT32_MAX, OutOfRange, "attn_paged: too many rows in one call");
            attn_paged_join_k<X, D><<<static_cast<unsigned>(joins), 256, 0, s>>>(a);
            AIC_LAUNCH_CHECK("attn_paged join");
        }
    };
    auto types = [&](auto hd) {
        if (dt == DType::Float32 && c.type == DType::Float32) run(float{}, float{}, hd);
        else if (dt == DType::Float32) run(float{}, uint8_t{}, hd);
        else if (c.type == DType::BFloat16) run(bf16{}, bf16{}, hd);
        else run(bf16{}, uint8_t{}, hd);
    };
    if (c.head_dim == 32) types(std::integral_constant<int, 32>{});
    else if (c.head_dim == 64) types(std::integral_constant<int, 64>{});
    else types(std::integral_constant<int, 128>{});
}

}  // namespace aic::hip
