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
//
// bf16 queries: attention_paged_tiles.hip, or attention_paged_few.hip for few rows per key/value head.  fp32
// queries: here, or attention_paged_f32_few.hip for up to 4.  Also here: the plan, the join and the launch.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_paged.hpp"
#include "../runtime/memory_pool.hpp"

namespace aic::hip {

namespace {

// ----------------------------------------------------------------------- the fp32 kernel
// Blocks of four waves: 4 / SH sets of 32 query rows, over tiles of 32 SH keys that the SH waves of a set
// share, 32 each, their states joined at the end.  SH = 1 where the batch fills the card with blocks of
// 128 rows; otherwise more and smaller blocks with fewer steps (f32_rows).
//
// One tile of K and one of V are in LDS: the next K is on its way while this V is multiplied, the next V while that K
// is, so nothing is staged twice and no copy is waited for.  The copies go straight to LDS (codes through registers)
// from page ids in LDS, and fragments are read a group of four products ahead from addresses made anew for each
// tile, so that two blocks of head_dim 128 keep their registers on one CU.  Bound by the fp32 matrix pipe (64 cycles
// per v_mfma_f32_32x32x2_f32) and by how evenly one round of blocks fills the card: 4000 rows of 16 heads of 128, 809 us,
// 81 TFLOP/s of 154, the pipe busy 51% of the time; behind 16000 cached tokens, where tiles are even, 117 TFLOP/s; 1000 on
// 2000 keys, 16 heads over 2, 158 us, 78 TFLOP/s (through registers, one block per CU: 210 us; from page ids in memory:
// 326 us); 856 of 16 heads of 64, 43 us, whose longest block takes most of it.
constexpr int kIds = 512;  // page ids in LDS at a time

template <typename CT, int HD, int SH, typename A>
__device__ __forceinline__ bool f32_pass(const A& a, int tid, int block, float down) {
    constexpr int SETS = 4 / SH, R = 32 * SETS, KT = 32 * SH, OB = HD / 32;
    constexpr int UPR = HD / kPer16<CT>;        // 16-byte units of a cached row
    constexpr int NU = (KT * UPR + 255) / 256;  // units of a tile per thread
    constexpr bool E4 = kE4<CT> || kE2<CT>;     // codes
    constexpr int TILE = KT * HD * 4;
    __shared__ __attribute__((aligned(16))) char tiles[2 * TILE];
    __shared__ int ids[kIds];
    char *ks = tiles, *vs = tiles + TILE;

    const int Hkv = a.kv.Hkv;
    const int rest = block / grid_heads(a);
    const int split = rest % a.nsplit, tile = static_cast<int>(gridDim.x) / (grid_heads(a) * a.nsplit) - 1 - rest / a.nsplit;  // long ones first
    int b, local;
    if (!find_tile<R>(a, tile, b, local)) return false;
    const int kvh = kv_head(a, b, block % grid_heads(a));
    const Seq sq = wave_sequence(a, b);
    if (std::is_same_v<A, PickedArgs> && sq.n == 0) return false;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hl = lane >> 5;
    const int set = wave % SETS, share = wave / SETS, sub = 32 * share;  // this wave's rows of the block and keys of a tile
    const int rows = sq.n * a.G, r0 = local * R, r = r0 + set * 32 + (lane & 31);
    const bool real = r < rows;
    const int tok = real ? r / a.G : 0, head = kvh * a.G + (real ? r % a.G : 0);
    const int64_t t = sq.row0 + tok;
    const int hi = real ? sq.len - sq.n + tok : -1;                       // last key this row sees
    const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;  // first

    // keys of the block: what its first row sees first .. what its last row sees last, of this split
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int first_pos = same(sq.len - sq.n + r0 / a.G), last_pos = same(sq.len - sq.n + (min(r0 + R, rows) - 1) / a.G);
    int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0, k_hi = last_pos + 1;
    k_lo &= ~63;
    part_of_keys(k_lo, k_hi, split, a.nsplit);
    // keys of this wave's rows: those of the set, none behind the sequence's last row
    const int set_r0 = r0 + set * 32, set_first = sq.len - sq.n + set_r0 / a.G, set_last = sq.len - sq.n + (min(set_r0 + 32, rows) - 1) / a.G;
    const int set_hi = set_r0 < rows ? min(k_hi, set_last + 1) : 0;
    const int set_lo = a.window > 0 ? max(set_first, 0) - a.window + 1 : 0;
    const uint32_t span = static_cast<uint32_t>(max(min(hi, k_hi - 1) - lo + 1, 0));  // keys from lo on that it sees here
    const bool empty = span == 0 || min(hi, k_hi - 1) < k_lo;                          // of this split

    Rows<OB> st_;
    st_.init();
    if (k_lo < k_hi) {
        constexpr int KF = HD / 8;
        float4 qf[KF];  // 4 values at 8 c + 4 h
        const float* qp = static_cast<const float*>(a.q) + t * a.ldq + static_cast<int64_t>(head) * HD;
#pragma unroll
        for (int cc = 0; cc < KF; ++cc) {
            const float* p = qp + 8 * cc + 4 * hl;
            qf[cc] = !real ? make_float4(0, 0, 0, 0) : a.vec_q ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
        }

        // Where this lane's fragments lie, in bytes: K row sub + lane % 32, chunk 2 c + h; V row sub + 8 (e >> 2) + 4 h + (e & 3),
        // column 32 ob + lane % 32.  The swizzles are exclusive-ors of a lane's part and constants.
        const int lr = lane & 31;
        const int k_lane = (sub + lr) * HD * 4 + ((hl ^ (HD == 32 ? (lr >> 1) & 7 : lr & 15)) << 4);
        const int v_lane = (sub + 4 * hl) * HD * 4 + (((lr >> 2) ^ (HD == 32 ? 2 * hl : 4 * hl)) << 4) + (lr & 3) * 4;
        auto k_at = [&](int lane_part, int c) { return (lane_part ^ ((2 * c & 15) << 4)) + ((2 * c & 16) << 4); };
        auto v_at = [&](int lane_part, int e, int ob) {
            const int g = (e >> 2) & 1, row = (8 * (e >> 2) + (e & 3)) * HD * 4;
            if constexpr (HD == 32) return (lane_part ^ (((e & 3) >> 1 | g << 2) << 4)) + row;
            else return (lane_part ^ ((e & 3) << 4)) + row + (ob ^ g) * 128;
        };
        // Copies of K and V of a tile: in fp32 straight to LDS, 1 KB per wave's instruction; codes through registers.
        struct Codes {
            uint4 w[NU];
            uint32_t e[NU];
        };
        [[maybe_unused]] Codes codes;
        const int32_t* tr = a.kv.table + b * a.kv.ld_table;
        const int window_keys = min((kIds - 1) * a.kv.ps, 1 << 20) & ~127;  // keys whose page ids fit: at least 384
        for (int w0 = k_lo, w1; w0 < k_hi; w0 = w1) {
            w1 = w0 + min(k_hi - w0, window_keys);
            const int p0 = a.kv.page_index(w0), nt = (w1 - w0 + KT - 1) / KT;
            __syncthreads();
            for (int i = tid; i <= a.kv.page_index(w1 - 1) - p0; i += 256) {
                const int page = p0 + i < a.kv.ld_table ? tr[p0 + i] : -1;
                ids[i] = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.n_pages) ? page : -1;
            }
            __syncthreads();
            auto row_at = [&](int key) -> int64_t {  // row in the pools, negative without a page; past the last key: the last
                key = min(key, w1 - 1);
                const int pi = a.kv.page_index(key), page = ids[pi - p0];
                const int64_t row = (static_cast<int64_t>(page) * Hkv + kvh) * a.kv.ps + (key - pi * a.kv.ps);
                return page < 0 ? -1 : row;
            };
            const char* none = reinterpret_cast<const char*>(&kNoPage);
            auto fetch = [&](const char* pool, [[maybe_unused]] const uint8_t* exps, int t, [[maybe_unused]] char* dst) {
                if constexpr (E4) {
#pragma unroll
                    for (int i = 0; i < NU; ++i) {
                        const int u = i * 256 + tid;
                        const int64_t row = row_at(w0 + t * KT + min(u / UPR, KT - 1));
                        codes.w[i] = *reinterpret_cast<const uint4*>(row >= 0 ? pool + row * kRowBytes<CT, HD> + (u % UPR) * 16 : none);
                        if constexpr (kE2<CT>) codes.e[i] = row >= 0 ? exps[row * UPR + u % UPR] : kNanGroup;
                        else codes.e[i] = row >= 0 ? exps[row] : 127;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < TILE / 4096; ++i) {
                        const int at = (4 * i + wave) * 1024, rr = (at + lane * 16) / (HD * 4), ch = lane % (HD / 4);
                        const int64_t row = row_at(w0 + t * KT + rr);
                        dma16(row >= 0 ? pool + row * (HD * 4) + ((ch ^ (HD == 32 ? (rr >> 1) & 7 : rr & 15)) << 4) : none, dst + at);
                    }
                }
            };
            auto put = [&]([[maybe_unused]] char* dst) {  // codes to LDS
                if constexpr (E4) {
#pragma unroll
                    for (int i = 0; i < NU; ++i) {
                        const int u = i * 256 + tid, row = u / UPR, c = u % UPR;
                        if (KT * UPR % 256 != 0 && u >= KT * UPR) continue;
                        const float s = exp_scale(codes.e[i]);
                        if constexpr (kE2<CT>) {
                            const uint32_t w[4] = {codes.w[i].x, codes.w[i].y, codes.w[i].z, codes.w[i].w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                float y[8];
                                e2m1_floats(w[j], s, y);
                                if (__builtin_expect(codes.e[i] == kNanGroup, 0))
#pragma unroll
                                    for (int x = 0; x < 8; ++x) y[x] = NAN;
                                *reinterpret_cast<float4*>(dst + chunk_at<float, HD>(row, 8 * c + 2 * j)) = make_float4(y[0], y[1], y[2], y[3]);
                                *reinterpret_cast<float4*>(dst + chunk_at<float, HD>(row, 8 * c + 2 * j + 1)) = make_float4(y[4], y[5], y[6], y[7]);
                            }
                            continue;
                        }
                        if (__builtin_expect(codes.e[i] >= kTopByte, 0)) codes.w[i] = e4m3_in_range(codes.w[i], codes.e[i]);
                        const uint2 w[2] = {make_uint2(codes.w[i].x, codes.w[i].y), make_uint2(codes.w[i].z, codes.w[i].w)};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float y[8];
                            e4m3_floats(w[j], s, y);
                            *reinterpret_cast<float4*>(dst + chunk_at<float, HD>(row, 4 * c + 2 * j)) = make_float4(y[0], y[1], y[2], y[3]);
                            *reinterpret_cast<float4*>(dst + chunk_at<float, HD>(row, 4 * c + 2 * j + 1)) = make_float4(y[4], y[5], y[6], y[7]);
                        }
                    }
                }
            };
            auto meet = [&] {  // what this wave brought is there and what it read is read; then everyone's
                wait_lds();
                if constexpr (!E4) wait_vmcnt<0>();
                __builtin_amdgcn_s_barrier();
            };
            fetch(a.kv.kp, a.kv.ke, 0, ks);
            put(ks);
            meet();
            fetch(a.kv.vp, a.kv.ve, 0, vs);
            put(vs);
            for (int t = 0; t < nt; ++t) {
                const int k0 = w0 + t * KT;
                const bool next = t + 1 < nt, mine = k0 + sub < set_hi && k0 + sub + 31 >= set_lo;  // else no row of this wave sees a key of its
                // made anew for each tile: dozens of addresses kept through the loop would take the registers of a second block
                int kl = k_lane, vl = v_lane;
                asm volatile("" : "+v"(kl), "+v"(vl));
                f32x16 sc[1];
                if (E4 && next) fetch(a.kv.kp, a.kv.ke, t + 1, ks);
                if (mine) {
                    zero(sc[0]);
                    // fragments are read one group of four products ahead, no further
                    float4 kx[2];
                    kx[0] = *reinterpret_cast<const float4*>(ks + k_at(kl, 0));
#pragma unroll
                    for (int cc = 0; cc < KF; ++cc) {
                        if (cc + 1 < KF) kx[(cc + 1) & 1] = *reinterpret_cast<const float4*>(ks + k_at(kl, cc + 1));
                        const float4 x = kx[cc & 1];
                        sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, qf[cc].x, sc[0], 0, 0, 0);
                        sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, qf[cc].y, sc[0], 0, 0, 0);
                        sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, qf[cc].z, sc[0], 0, 0, 0);
                        sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, qf[cc].w, sc[0], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                meet();  // V is there, K has been read
                if (next) {
                    if constexpr (E4) {
                        put(ks);
                        fetch(a.kv.vp, a.kv.ve, t + 1, vs);
                    } else {
                        fetch(a.kv.kp, a.kv.ke, t + 1, ks);
                    }
                }
                if (mine) {
                    const int kw = k0 + sub;  // this wave's first key of the tile
                    // every row of the set sees every one of them?
                    const bool open = kw + 31 <= set_first && kw + 32 <= k_hi && (a.window <= 0 || kw > set_last - a.window);
                    auto seen = [&](int j) { return static_cast<uint32_t>(kw + j - lo) < span; };
                    bool poison = false;  // a hidden key beside a non-finite v
                    if (!open) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) sc[0][e] = seen(8 * (e >> 2) + 4 * hl + (e & 3)) ? sc[0][e] : -INFINITY;
                        uint32_t bits = 0;
#pragma unroll 4
                        for (int i = 0; i < HD / 8; ++i)
                            bits |= non_finite_bits<float>(*reinterpret_cast<const uint4*>(vs + sub * HD * 4 + i * 1024 + lane * 16));
                        poison = __any(bits != 0);
                    }
                    float mx = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[0][e]);
                    st_.absorb(mx, a.c);
                    const float off = st_.offset(a.c, down);
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        sc[0][e] = weight(sc[0][e], a.c, off);
                        sum += sc[0][e];
                    }
                    st_.add(sum);
                    if (poison) {
                        add_seen_rows<HD, 1>(st_.o, sc, [&](int key, int d) { return v4_at<float, HD>(vs, sub + key, d); }, seen);
                    } else {
                        float vx[2][4];
                        auto read = [&](int g, float (&x)[4]) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const float*>(vs + v_at(vl, (4 * g + j) / OB, (4 * g + j) % OB));
                        };
                        read(0, vx[0]);
#pragma unroll
                        for (int g = 0; g < 4 * OB; ++g) {
                            if (g + 1 < 4 * OB) read(g + 1, vx[(g + 1) & 1]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int e = (4 * g + j) / OB, ob = (4 * g + j) % OB;
                                st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x2f32(vx[g & 1][j], sc[0][e], st_.o[ob], 0, 0, 0);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
                meet();  // K of the next tile is there, V has been read
                if (next) {
                    if constexpr (E4) put(vs);
                    else fetch(a.kv.vp, a.kv.ve, t + 1, vs);
                }
            }
        }
    }
    if constexpr (SH > 1) {
        // each set's first wave takes the others' states: M = max m_w, o = sum 2^((m_w - M) c) o_w, l alike
        float* os = reinterpret_cast<float*>(tiles);  // [SETS][SH - 1][OB * 16][64]
        __shared__ float2 mls[4][32];
        __syncthreads();  // the tiles have been read
        if (hl == 0) mls[wave][lane] = make_float2(st_.m, st_.l);
        __syncthreads();
        float M = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < SH; ++w) M = fmaxf(M, mls[set + w * SETS][lane & 31].x);
        const float base = M == -INFINITY ? 0.0f : M;
        const float factor = __builtin_amdgcn_exp2f((st_.m - base) * a.c);
#pragma unroll
        for (int w = 0; w < SH; ++w) {
            const float2 ml = mls[set + w * SETS][lane & 31];
            l = fmaf(__builtin_amdgcn_exp2f((ml.x - base) * a.c), ml.y, l);
        }
        auto at = [&](int w, int i) { return ((set * (SH - 1) + w - 1) * OB * 16 + i) * 64 + lane; };
#pragma unroll
        for (int ob = 0; ob < OB; ++ob)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                st_.o[ob][e] *= factor;
                if (share > 0) os[at(share, ob * 16 + e)] = st_.o[ob][e];
            }
        __syncthreads();
        if (share > 0) return false;
#pragma unroll
        for (int ob = 0; ob < OB; ++ob)
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int w = 1; w < SH; ++w) st_.o[ob][e] += os[at(w, ob * 16 + e)];
        st_.m = M;
        st_.l = l;
    }
    return real && store_row<float, HD>(a, st_, t, head, empty, split, down > 0.0f);
}

template <typename CT, int HD, int SH, typename A>
__global__ __launch_bounds__(256, 2) void attn_paged_f32_k(A a) {
    one_or_two_passes(a, [](const A& args, int tid, int block, float down) { return f32_pass<CT, HD, SH>(args, tid, block, down); });
}

// ------------------------------------------------------------------------- joining splits
// One wave per (token, head): M = max m_s, w_s = 2^((m_s - M) c) l_s, o = sum_s w_s o_s / sum_s w_s; o_s is divided by l_s.
// Bound by reading the parts: 12 us for two of 2048 rows of 16 heads of 128 (34 MB read, 8 MB written: 3.5 TB/s).
template <typename T, int HD, typename A>
__global__ __launch_bounds__(256) void attn_paged_join_k(A a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (i >= a.T * a.H) return;
    const int64_t t = i / a.H;
    // rows of no sequence stay as they are
    if constexpr (std::is_same_v<A, PickedArgs>) {
        if (a.lens[t * a.kv.Hkv + i % a.H / a.G] < 0) return;
    } else {
        if (t < a.offsets[0] || t >= a.offsets[a.B]) return;
    }
    const int lane = threadIdx.x & 63;
    const int64_t step = a.T * a.H;
    // a lane per split: the splits of one launch are at most kMaxSplits
    const float2 ml = lane < a.nsplit ? a.part_ml[lane * step + i] : make_float2(-INFINITY, 0.0f);
    const bool any = __any(ml.y != 0.0f);
    const float M = wave_all(ml.y != 0.0f ? ml.x : -INFINITY, [](float x, float y) { return fmaxf(x, y); });
    const float base = M == -INFINITY ? 0.0f : M;
    const bool some = ml.y != 0.0f && ml.y != -1.0f;
    const float own = some ? __builtin_amdgcn_exp2f((ml.x - base) * a.c) * ml.y : 0.0f;
    const float l = wave_all(own, [](float x, float y) { return x + y; });
    const float w = own * (1.0f / l);  // of a part's row, which is divided by its own sum
    constexpr int PL = HD >= 64 ? HD / 64 : 1;
    float o[PL] = {};
    uint64_t left = __ballot(some);  // their partial rows, four at a time
    while (left) {
        int at[4];
        float x[4][PL], ws[4];
        bool live[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            live[j] = left != 0;
            at[j] = live[j] ? __builtin_ctzll(left) : at[j > 0 ? j - 1 : 0];
            ws[j] = __shfl(w, at[j], 64);
            left &= left - 1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int u = 0; u < PL; ++u)
                if (lane * PL < HD) x[j][u] = a.part_o[(at[j] * step + i) * HD + lane * PL + u];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int u = 0; u < PL; ++u) o[u] = live[j] ? fmaf(ws[j], x[j][u], o[u]) : o[u];
    }
    T* op = static_cast<T*>(a.o) + t * a.ldo + (i % a.H) * HD;
#pragma unroll
    for (int u = 0; u < PL; ++u)
        if (lane * PL < HD) st(op, lane * PL + u, any && l == 0.0f ? NAN : o[u]);  // only scores of -infinity: NaN
    if (a.lse && lane == 0) a.lse[i] = any ? log_sum(base, l, a.c) : -INFINITY;
}

// --------------------------------------------------------------------------- the launch
int64_t tile_bound(int64_t T, int64_t G, int64_t B, int64_t R) { return T * G / R + std::min(B, T); }

constexpr int64_t kMaxSplits = 64;  // a wave joins them, a lane each
struct Plan {
    int64_t tiles, nsplit;
};
// Parts of the keys where the query tiles alone do not fill the card: as many as make one round of about 512 blocks (two
// per CU; 2048 rows of 16 heads twice: 52.6 us in 464 blocks, 73.6 us in 928), of at least 448 keys where
// there are more than four (256 rows on 4096 keys: 26.2 us in 8 parts, 30.5 us in 16, 33.0 us in 4).  Where the parts'
// rows are little to join (4 MB), of 128 keys from 512 on: 8 rows of 16 heads of 128 over 2 on 2000 keys, 19.6 us in 4
// parts and 15.5 us in 15; but 40 rows of 12 heads of 64 on 300, 10.7 us in one and 12.2 us in 2.  R: query rows of a block.
Plan plan(int64_t B, int64_t T, int64_t max_len, int64_t H, const KVPages& c, int64_t R) {
    const int64_t Hkv = c.kv_heads;
    Plan p{tile_bound(T, H / Hkv, B, R), 1};
    // two times the blocks there probably are; tiles of up to 4 rows hold a sequence each
    const int64_t twice = (R <= 4 ? 2 * std::min(B, T) : 2 * T * (H / Hkv) / R + std::min(B, T)) * Hkv;
    int64_t most = std::max<int64_t>(std::min<int64_t>(4, max_len / 256), max_len / 448);
    if (max_len >= 512) most = std::max(most, std::min(max_len / 128, (int64_t{4} << 20) / (T * H * (c.head_dim + 2) * 4)));
    p.nsplit = std::clamp<int64_t>((1024 + twice / 2) / std::max<int64_t>(twice, 1), 1, std::clamp<int64_t>(most, 1, kMaxSplits));
    return p;
}
// fp32: query rows of a block: 32 where rows have pages of their own, a group each; otherwise fewer than 128 where such blocks are fewer than two per CU; at head_dim 128 then 64, two
// blocks to a CU, or 32 where a block is alone there and the keys are not divided: 300 rows of 16 heads on 300 keys,
// 33.9 us in 32 and 39.7 us in 64; on 452 rows and 554 keys, in two parts, 59.0 and 48.4 us.
int64_t f32_rows(int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H, int64_t Hkv, int64_t hd, bool picked) {
    if (const int few = f32_few_rows(max_q, H / Hkv)) return few;
    if (picked) return 32;
    if (tile_bound(T, H / Hkv, B, 128) * Hkv >= 512) return 128;
    return hd == 128 && (max_len >= 512 || tile_bound(T, H / Hkv, B, 32) * Hkv > 256) ? 64 : 32;
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
    AIC_CHECK(H <= INT32_MAX, InvalidArgument, "attn_paged: more than 2^31 - 1 query heads");  // the products below stay in 64 bits
    AIC_CHECK(T * (H / c.kv_heads) <= kMaxLen, OutOfRange, "attn_paged: more than ", kMaxLen, " query rows per key/value head");
}

}  // namespace

namespace {

// Bytes of the parts of a call's sizes; picked: of rows with pages of their own, a sequence each (bf16 queries then always go to the
// few rows' kernel).
int64_t parts_bytes(const KVPages& c, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H, bool picked) {
    check_sizes(c, B, T, max_q, max_len, H);
    check_cache_shape(c, "attn_paged");
    if (B == 0 || T == 0) return 0;
    max_q = std::min(max_q, T);
    // the cache's type does not tell the queries' (codes serve both): room for either
    int64_t n = 0;
    const int64_t G = H / c.kv_heads;
    const bool few = picked || few_rows(B * c.kv_heads, max_q, max_len, G, c.head_dim, c.type);
    if (c.type != DType::Float32 && few)
        n = few_workspace(B, c.kv_heads, max_q, max_len, G, c.head_dim, c.type, picked);
    if (c.type != DType::Float32 && !few)
        n = plan_bytes(plan(B, T, max_len, H, c, 128), T, H, c.head_dim);
    if (c.type != DType::BFloat16)
        n = std::max(n, plan_bytes(plan(B, T, max_len, H, c, f32_rows(B, T, max_q, max_len, H, c.kv_heads, c.head_dim, picked)), T, H, c.head_dim));
    return n;
}

struct Workspace {
    void* at;
    int64_t bytes;
};

// a: pointers, strides, T, H, G and the batch; the rest follows from the sizes, which are those of the sequences that the blocks see.
template <typename A>
void attend(A& a, const KVPages& c, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H, float scale, Workspace w,
            DType dt, hipStream_t s) {
    constexpr bool picked = std::is_same_v<A, PickedArgs>;
    max_q = std::min(max_q, T);
    const int64_t size = static_cast<int64_t>(dtype_size(dt));
    a.c = scale * kLog2e;
    a.vec_q = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.ldq * size % 16 == 0;
    a.vec_o = reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && a.ldo * size % 16 == 0;

    const bool few = dt == DType::BFloat16 && (picked || few_rows(B * c.kv_heads, max_q, max_len, a.G, c.head_dim, c.type));
    const int64_t R = dt == DType::BFloat16 ? 128 : f32_rows(B, T, max_q, max_len, H, c.kv_heads, c.head_dim, picked);
    Plan p = plan(B, T, max_len, H, c, R);
    const int64_t need = parts_bytes(c, B, T, max_q, max_len, H, picked);
    const StreamScratchUse use(s);
    void* workspace = w.at;
    if (workspace)
        AIC_CHECK(w.bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, InvalidArgument,
                  "attn_paged: the workspace must be 16-byte aligned and hold ", need, " bytes, got ", w.bytes);
    else if (need > 0 && stream_scratch_ready(s))
        workspace = stream_scratch(static_cast<size_t>(need), s);
    AIC_CHECK(a.q != a.o, InvalidArgument, "attn_paged: q and o must not overlap");  // a second pass reads q anew
    if (need == 0) workspace = nullptr;
    if (few) {
        // need may be the other kernel's alone
        const bool shares = few_workspace(B, c.kv_heads, max_q, max_len, a.G, c.head_dim, c.type, picked) > 0;
        attn_paged_few(a, max_q, c.type, static_cast<int>(c.head_dim), shares ? workspace : nullptr, s);
        return;
    }
    if (!workspace) p.nsplit = 1;  // nothing to split, or captured without a workspace of its own
    a.nsplit = static_cast<int>(p.nsplit);
    if (p.nsplit > 1) {
        a.part_o = static_cast<float*>(workspace);
        a.part_ml = reinterpret_cast<float2*>(a.part_o + p.nsplit * T * H * c.head_dim);
    }
    const int64_t blocks = p.tiles * c.kv_heads * p.nsplit;
    AIC_CHECK(blocks <= INT32_MAX, OutOfRange, "attn_paged: too many rows in one call");
    auto run = [&](auto t, auto hd) {
        using X = decltype(t);
        constexpr int D = decltype(hd)::value;
        const auto grid = static_cast<unsigned>(blocks);
        if constexpr (sizeof(X) == 2) {
            attn_paged_tiles(a, c.type, D, grid, s);
        } else if (R <= 4) {
            attn_paged_f32_few(a, static_cast<int>(R), c.type, D, grid, s);
        } else {
            by_cache_type<float>(c.type, [&](auto ct) {
                using CT = decltype(ct);
                if constexpr (!picked) {
                    if (R == 128) return attn_paged_f32_k<CT, D, 1><<<grid, 256, 0, s>>>(a);
                    if (R == 64) return attn_paged_f32_k<CT, D, 2><<<grid, 256, 0, s>>>(a);
                }
                attn_paged_f32_k<CT, D, 4><<<grid, 256, 0, s>>>(a);
            });
            AIC_LAUNCH_CHECK("attn_paged");
        }
        if (a.nsplit > 1) {
            const int64_t joins = (T * H + 3) / 4;
            AIC_CHECK(joins <= INT32_MAX, OutOfRange, "attn_paged: too many rows in one call");
            attn_paged_join_k<X, D><<<static_cast<unsigned>(joins), 256, 0, s>>>(a);
            AIC_LAUNCH_CHECK("attn_paged join");
        }
    };
    auto types = [&](auto hd) {
        if (dt == DType::Float32) run(float{}, hd);
        else if constexpr (!picked) run(bf16{}, hd);  // picked: the few rows' kernel, always
    };
    if (c.head_dim == 32) types(std::integral_constant<int, 32>{});
    else if (c.head_dim == 64) types(std::integral_constant<int, 64>{});
    else types(std::integral_constant<int, 128>{});
}

void check_call(const KVPages& c, int64_t ld_q, int64_t ld_o, int64_t H, float scale, int64_t workspace_bytes, DType dt) {
    AIC_CHECK(ld_q >= H * c.head_dim && ld_o >= H * c.head_dim, InvalidArgument,
              "attn_paged: leading dimension below heads * head_dim");
    AIC_CHECK(std::isfinite(scale * kLog2e) && scale > 0.0f, InvalidArgument, "attn_paged: scale must be positive and below 2.3e38, got ", scale);
    AIC_CHECK(workspace_bytes >= 0, InvalidArgument, "attn_paged: negative workspace size");
}

void check_types(const KVPages& c, DType dt) {
    AIC_CHECK(dt == DType::Float32 || dt == DType::BFloat16, DTypeMismatch, "attn_paged: queries are float32 or bfloat16");
    AIC_CHECK(c.type == dt || holds_codes(c.type), DTypeMismatch, "attn_paged: queries of ", dtype_name(dt),
              " with a cache of ", dtype_name(c.type));
}

// The cache as its (row, key/value head) pairs see it: sequences of one head.
KVPages one_head(const KVPages& c) {
    AIC_CHECK(c.kv_heads >= 1 && c.kv_heads <= 4096, InvalidArgument, "attn_paged: kv_heads must be 1 .. 4096, got ", c.kv_heads);
    KVPages x = c;
    x.kv_heads = 1;
    return x;
}

// Sizes of attn_paged_selected: keys of a row.
int64_t check_picked(const KVPages& c, int64_t T, int64_t n_sel, int64_t H) {
    check_cache_shape(c, "attn_paged");
    AIC_CHECK(T >= 0 && T <= INT32_MAX, InvalidArgument, "attn_paged: T must be 0 .. 2^31 - 1");
    AIC_CHECK(H >= 1 && H % c.kv_heads == 0, ShapeMismatch, "attn_paged: ", H, " query heads over ", c.kv_heads, " key/value heads");
    AIC_CHECK(T * c.kv_heads <= INT32_MAX, OutOfRange, "attn_paged: more than 2^31 - 1 pairs of rows and key/value heads");
    AIC_CHECK(c.page_size >= 1 && c.page_size <= 65536, InvalidArgument, "attn_paged: page_size must be 1 .. 65536, got ", c.page_size);
    AIC_CHECK(n_sel >= 1 && n_sel <= kMaxLen / c.page_size, InvalidArgument, "attn_paged: n_sel must be 1 .. ", kMaxLen / c.page_size, ", got ",
              n_sel);
    return n_sel * c.page_size;
}

}  // namespace

int64_t attn_paged_workspace(const KVPages& c, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H) {
    return parts_bytes(c, B, T, max_q, max_len, H, false);
}

void attn_paged(const KVPages& c, const void* q, int64_t ld_q, void* o, int64_t ld_o, float* lse, const int64_t* offsets,
                const int64_t* lens, int64_t B, int64_t T, int64_t max_q, int64_t max_len, int64_t H, int64_t window,
                float scale, void* workspace, int64_t workspace_bytes, DType dt, hipStream_t s) {
    check_sizes(c, B, T, max_q, max_len, H);
    check_types(c, dt);
    const PageView pv = page_view(c, "attn_paged");
    check_call(c, ld_q, ld_o, H, scale, workspace_bytes, dt);
    AIC_CHECK(window >= 0, InvalidArgument, "attn_paged: window must not be negative, got ", window);
    if (B == 0 || T == 0) return;
    AIC_CHECK(q && o && offsets && lens, InvalidArgument, "attn_paged: null pointer");
    PagedArgs a{};
    a.kv = pv;
    a.q = q, a.o = o, a.lse = lse;
    a.ldq = ld_q, a.ldo = ld_o, a.T = T;
    a.offsets = offsets, a.lens = lens;
    a.B = static_cast<int>(B), a.H = static_cast<int>(H), a.G = static_cast<int>(H / c.kv_heads);
    a.window = static_cast<int>(std::min<int64_t>(window, INT32_MAX));
    attend(a, c, B, T, max_q, max_len, H, scale, {workspace, workspace_bytes}, dt, s);
}

int64_t attn_paged_selected_workspace(const KVPages& c, int64_t T, int64_t n_sel, int64_t H) {
    const int64_t len = check_picked(c, T, n_sel, H), rows = T * c.kv_heads;
    return parts_bytes(one_head(c), rows, rows, 1, len, H / c.kv_heads, true);
}

void attn_paged_selected(const KVPages& c, const void* q, int64_t ld_q, void* o, int64_t ld_o, float* lse, const int32_t* picked,
                         const int64_t* picked_lens, int64_t T, int64_t n_sel, int64_t H, float scale, void* workspace,
                         int64_t workspace_bytes, DType dt, hipStream_t s) {
    const int64_t len = check_picked(c, T, n_sel, H), rows = T * c.kv_heads, G = H / c.kv_heads;
    const KVPages one = one_head(c);
    check_sizes(one, rows, rows, 1, len, G);
    check_types(c, dt);
    KVPages view = c;
    view.page_table = picked;
    view.ld_table = n_sel;
    if (T > 0) AIC_CHECK(picked && picked_lens, InvalidArgument, "attn_paged: null pointer");
    else view.page_table = reinterpret_cast<const int32_t*>(c.k_pages);  // nothing is read
    const PageView pv = page_view(view, "attn_paged");
    check_call(c, ld_q, ld_o, H, scale, workspace_bytes, dt);
    if (T == 0) return;
    AIC_CHECK(q && o, InvalidArgument, "attn_paged: null pointer");
    PickedArgs a{};
    a.kv = pv;
    a.q = q, a.o = o, a.lse = lse;
    a.ldq = ld_q, a.ldo = ld_o, a.T = T;
    a.lens = picked_lens;
    a.B = static_cast<int>(rows), a.H = static_cast<int>(H), a.G = static_cast<int>(G);
    attend(a, one, rows, rows, 1, len, G, scale, {workspace, workspace_bytes}, dt, s);
}

}  // namespace aic::hip
