// Attention over the paged cache for many query rows per key/value head (chunks of prompts), bf16: bound by the matrix
// cores, the softmax between their products and the waits of two blocks for each other.
//
// One block: 128 query rows (4 waves x 32) of one sequence and key/value head, over tiles of 64 keys that the four waves
// share.  Software-pipelined as the causal kernel of whole batches: stage unit t holds K of tile t + 1 and V of
// tile t, so that while a wave multiplies P(t) V(t) it already holds the scores of tile t + 1.  An iteration is
// two groups of MFMAs, each with the work that overlaps it:
//   A  S(t+1) = K(t+1) Q^T with the exponentials, sum and packing of tile t
//   B  O^T += V(t)^T P(t)^T with the row maximum of tile t + 1
// then one barrier, after which unit t + 2 goes where unit t was.  A wave copies 16 consecutive keys of each tile,
// which lie in one page where page_size is a multiple of 16: one page id from LDS, uniform bases.  bf16
// pools travel by direct global -> LDS copies; e4m3 pools through registers, a unit ahead, and are
// converted once per block as they are stored (converted by each wave as it reads them, the
// conversions would be four times as many, about as much as the softmax).
//
// 2048 rows of 16 heads of 128 over 2, behind 6144 cached tokens: 136 us, 883 TFLOP/s with the join of its two parts
// per tile (124 us and 12 us); two blocks per CU, for their products fill each other's softmax: matrix pipe busy
// about 40% of the cycles, vector units 36%.  Behind 30720 tokens, where tiles are even, 1070 TFLOP/s.
//
// Tiles that some row does not see whole (the chunk's own keys, a window's edge: two or three per block) run first, in a
// plain loop that masks and looks for non-finite v: the order of the keys is free, and the pipelined loop keeps
// its registers (with masks in it, it spilled, and a reload waits for the copies in flight).
#include <type_traits>

#include "attention_paged.hpp"

namespace aic::hip {

namespace {

constexpr int kIds = 512;  // page ids in LDS at a time

// What a pass has found.  kTop: a row whose codes can be past the range (e4m3_in_range): looked for in the first pass only, and kept
// in the range by the other one, for a branch between the products costs 4% at head_dim 128.
constexpr int kPast = 1, kTop = 2;

template <int HD>
struct TilesLds {
    __attribute__((aligned(16))) bf16 sm[2][2 * 64 * HD];
    int ids[kIds];
    int past, top;
};

template <int HD, bool E4, bool SECOND>
__device__ __forceinline__ int tiles_pass(TilesLds<HD>& lds, const PagedArgs& a, int tid, int block, float down) {
    constexpr int KS = HD / 16, OB = HD / 32, TILE = 64 * HD;  // elements of a tile
    constexpr int NA = 2 * KS, NB = 4 * OB;                   // MFMAs of groups A and B
    constexpr int EA = 32 / NA, EB = 32 / NB;                 // elements per slot
    constexpr int NR = OB + 1, KR = 3;                        // fragment rings
    constexpr int RB = HD * 2, NC = RB / 16, RPS = 1024 / RB, PW = 16 / RPS;  // bf16 copies: of a wave's 16 rows
    constexpr int UPR = HD / 16, UNITS = 64 * UPR, NU = (UNITS + 255) / 256;  // e4m3: 16-byte units of a tile
    auto& sm = lds.sm;
    auto& ids = lds.ids;

    const int Hkv = a.kv.Hkv, ps = a.kv.ps;
    const int kvh = block % Hkv, rest = block / Hkv;
    const int split = rest % a.nsplit, tile = static_cast<int>(gridDim.x) / (Hkv * a.nsplit) - 1 - rest / a.nsplit;  // long ones first
    int b, local;
    if (!find_tile<128>(a, tile, b, local)) return 0;
    const Seq sq = wave_sequence(a, b);
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hl = lane >> 5;
    const int rows = sq.n * a.G, r0 = local * 128, r = r0 + wave * 32 + (lane & 31);
    const bool real = r < rows;
    const int tok = real ? r / a.G : 0, head = kvh * a.G + (real ? r % a.G : 0);
    const int64_t trow = sq.row0 + tok;
    const int hi = real ? sq.len - sq.n + tok : -1;
    const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // divisions leave uniform values in vector registers
    const int first_pos = same(sq.len - sq.n + r0 / a.G), last_pos = same(sq.len - sq.n + (min(r0 + 128, rows) - 1) / a.G);
    int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0, k_hi = last_pos + 1;
    k_lo &= ~63;
    part_of_keys(k_lo, k_hi, split, a.nsplit);
    const uint32_t span = static_cast<uint32_t>(max(min(hi, k_hi - 1) - lo + 1, 0));
    const bool empty = span == 0 || min(hi, k_hi - 1) < k_lo;

    [[maybe_unused]] uint64_t top = 0;  // lanes, in scalar registers
    Rows<OB> st_;
    st_.init();
    if (k_lo < k_hi) {
        bf16x8 qf[KS];
        const bf16* qp = static_cast<const bf16*>(a.q) + trow * a.ldq + static_cast<int64_t>(head) * HD + 8 * hl;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            if (a.vec_q) qf[kk] = __builtin_bit_cast(bf16x8, ldg16(qp + 16 * kk, real));
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) qf[kk][j] = real ? qp[16 * kk + j] : f2bf(0.0f);
        }
        Frags<HD> F;
        F.init(lane);
        [[maybe_unused]] uint32_t voff[PW];
        if constexpr (!E4) {
#pragma unroll
            for (int i = 0; i < PW; ++i) {
                const int rr = i * RPS + lane / NC;
                voff[i] = static_cast<uint32_t>(rr * RB + (((lane % NC) ^ swz<HD>(rr)) << 4));
            }
        }
        const int32_t* tr = a.kv.table + b * a.kv.ld_table;
        const char* none = reinterpret_cast<const char*>(&kNoPage);

        const int window_keys = min((kIds - 1) * ps, 1 << 20) & ~63;  // keys whose page ids fit: at least 448
        for (int w0 = k_lo, w1; w0 < k_hi; w0 = w1) {
            w1 = w0 + min(k_hi - w0, window_keys);
            const int p0 = a.kv.page_index(w0), np = a.kv.page_index(w1 - 1) - p0 + 1;
            __syncthreads();
            for (int i = tid; i < np; i += 256) {
                const int page = p0 + i < a.kv.ld_table ? tr[p0 + i] : -1;
                ids[i] = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.n_pages) ? page : -1;
            }
            __syncthreads();
            const int nt = (w1 - w0 + 63) / 64;
            auto row_at = [&](int key) -> int64_t {  // row in the pools, negative without a page; past the last key: the last
                key = min(key, w1 - 1);
                const int pi = a.kv.page_index(key), page = ids[pi - p0];
                const int64_t row = (static_cast<int64_t>(page) * Hkv + kvh) * ps + (key - pi * ps);
                return page < 0 ? -1 : row;
            };
            // bf16: this wave's 16 rows of tile t of a pool into dst
            auto copy = [&](const char* pool, int t, bf16* dst) {
                const int key = w0 + 64 * t + 16 * wave;
                dst += wave * 16 * HD;
                if (ps % 16 == 0 && key + 16 <= w1) {
                    const int pi = a.kv.page_index(key), page = __builtin_amdgcn_readfirstlane(ids[pi - p0]);
                    if (page >= 0) {
                        const char* base = pool + ((static_cast<int64_t>(page) * Hkv + kvh) * ps + (key - pi * ps)) * RB;
#pragma unroll
                        for (int i = 0; i < PW; ++i) dma16s(base, voff[i], dst + i * 512);
                        return;
                    }
                }
                int l = lane;
                asm volatile("" : "+v"(l));  // kept out of the loop's registers: the path of odd page sizes and last tiles
#pragma unroll
                for (int i = 0; i < PW; ++i) {
                    const int rr = i * RPS + l / NC;
                    const int64_t row = row_at(key + rr);
                    dma16(row >= 0 ? pool + row * RB + (((l % NC) ^ swz<HD>(rr)) << 4) : none, dst + i * 512);
                }
            };
            // e4m3: units of tile t of a pool in registers, and into dst
            struct Codes {
                uint4 w[NU];
                uint32_t e[NU];
            };
            auto fetch = [&](const char* pool, const uint8_t* exps, int t, Codes& c) {
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    const int u = i * 256 + tid;
                    const int64_t row = row_at(w0 + 64 * t + min(u / UPR, 63));
                    c.w[i] = *reinterpret_cast<const uint4*>(row >= 0 ? pool + row * HD + (u % UPR) * 16 : none);
                    c.e[i] = row >= 0 ? exps[row] : 127;
                }
            };
            auto put_unit = [&](const Codes& c, int i, bf16* dst) {
                const int u = i * 256 + tid;
                if (UNITS % 256 != 0 && u >= UNITS) return;
                uint4 w = c.w[i];
                if constexpr (SECOND) {
                    if (c.e[i] >= kTopByte) w = e4m3_in_range(w, c.e[i]);
                } else {
                    top |= __ballot(c.e[i] >= kTopByte);
                }
                const float s = exp_scale(c.e[i]);
                char* tile = reinterpret_cast<char*>(dst);
                const int rr = u / UPR, ch = 2 * (u % UPR);
                *reinterpret_cast<uint4*>(tile + chunk_at<bf16, HD>(rr, ch)) = e4m3_bf16(make_uint2(w.x, w.y), s);
                *reinterpret_cast<uint4*>(tile + chunk_at<bf16, HD>(rr, ch + 1)) = e4m3_bf16(make_uint2(w.z, w.w), s);
            };
            auto put = [&](const Codes& c, bf16* dst) {
#pragma unroll
                for (int i = 0; i < NU; ++i) put_unit(c, i, dst);
            };
            [[maybe_unused]] Codes ck, cv;  // the next unit's
            // tiles [t_a, t_b): every row sees every key
            int t_b = min(nt, max(0, min(first_pos + 1, k_hi) - w0) / 64), t_a = 0;
            if (a.window > 0 && last_pos - a.window >= w0) t_a = (last_pos - a.window - w0) / 64 + 1;
            if (t_a >= t_b) t_a = t_b = 0;

            // The others, two stages of K and V.
            const int n_plain = nt - (t_b - t_a);
            auto plain_tile = [&](int i) { return i < t_a ? i : t_b + (i - t_a); };
            auto plain_copy = [&](int i) {
                bf16* dst = sm[i & 1];
                if constexpr (E4) {
                    fetch(a.kv.kp, a.kv.ke, plain_tile(i), ck);
                    fetch(a.kv.vp, a.kv.ve, plain_tile(i), cv);
                    put(ck, dst);
                    put(cv, dst + TILE);
                } else {
                    copy(a.kv.kp, plain_tile(i), dst);
                    copy(a.kv.vp, plain_tile(i), dst + TILE);
                }
            };
            if (n_plain > 0) plain_copy(0);
            for (int i = 0; i < n_plain; ++i) {
                wait_lds();
                wait_vmcnt<0>();
                __builtin_amdgcn_s_barrier();
                if (i + 1 < n_plain) plain_copy(i + 1);
                const char* Kb = reinterpret_cast<const char*>(sm[i & 1]);
                const char* Vb = reinterpret_cast<const char*>(sm[i & 1] + TILE);
                const int k0 = w0 + 64 * plain_tile(i);
                auto seen = [&](int k) { return static_cast<uint32_t>(k0 + k - lo) < span; };
                f32x16 sc[2];
                uint32_t bits = 0;
#pragma unroll 4
                for (int j = 0; j < TILE * 2 / 1024; ++j)
                    bits |= non_finite_bits<bf16>(*reinterpret_cast<const uint4*>(Vb + j * 1024 + lane * 16));
                const bool bad = __any(bits != 0);  // a non-finite v beside a hidden key
                float mx = -INFINITY;
#pragma unroll
                for (int jb = 0; jb < 2; ++jb) {
                    zero(sc[jb]);
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk)
                        sc[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.row(Kb, jb * 32, kk), qf[kk], sc[jb], 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        sc[jb][e] = seen(jb * 32 + 8 * (e >> 2) + 4 * hl + (e & 3)) ? sc[jb][e] : -INFINITY;
                        mx = fmaxf(mx, sc[jb][e]);
                    }
                }
                st_.absorb(mx, a.c);
                const float off = st_.offset(a.c, down);
                float sum = 0.0f;
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        sc[jb][e] = weight(sc[jb][e], a.c, off);
                        sum += sc[jb][e];
                    }
                st_.add(sum);
                if (bad) {
                    add_seen_rows<HD, 2>(st_.o, sc, [&](int key, int d) { return v4_at<bf16, HD>(Vb, key, d); }, seen);
                } else {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const bf16x8 p = pack_bf16x8(sc[ks >> 1], 8 * (ks & 1));
#pragma unroll
                        for (int ob = 0; ob < OB; ++ob)
                            st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.tr(Vb, ob, ks), p, st_.o[ob], 0, 0, 0);
                    }
                }
            }
            if (t_a == t_b) continue;
            wait_lds();
            __builtin_amdgcn_s_barrier();  // the stages are free

            // The pipelined loop over tiles t_a .. t_b - 1; stage of unit t: (t - t_a + 1) & 1
            // unit t on its way (bf16: into stage st; e4m3: to registers, into the stage by iteration t - 1)
            auto begin = [&](int t, [[maybe_unused]] int st) {
                if constexpr (E4) {
                    if (t + 1 < t_b) fetch(a.kv.kp, a.kv.ke, t + 1, ck);
                    fetch(a.kv.vp, a.kv.ve, t, cv);
                } else {
                    if (t + 1 < t_b) copy(a.kv.kp, t + 1, sm[st]);
                    copy(a.kv.vp, t, sm[st] + TILE);
                }
            };
            f32x16 s0[2], s1[2];  // scores of tile t, then its weights, and scores of tile t + 1: in turn
            if constexpr (E4) {
                fetch(a.kv.kp, a.kv.ke, t_a, ck);
                put(ck, sm[0]);
                begin(t_a, 1);
                put(ck, sm[1]);
                put(cv, sm[1] + TILE);
                if (t_a + 1 < t_b) begin(t_a + 1, 0);
            } else {
                copy(a.kv.kp, t_a, sm[0]);
                begin(t_a, 1);
                wait_vmcnt<0>();
            }
            wait_lds();
            __builtin_amdgcn_s_barrier();
            {
                const char* Kb = reinterpret_cast<const char*>(sm[0]);
                zero(s0[0]);
                zero(s0[1]);
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                    for (int jb = 0; jb < 2; ++jb)
                        s0[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.row(Kb, jb * 32, kk), qf[kk], s0[jb], 0, 0, 0);
                float mx = -INFINITY;
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s0[jb][e]);
                st_.absorb(mx, a.c);
            }
            wait_lds();
            __builtin_amdgcn_s_barrier();  // K(t_a)'s stage is free
            if (!E4 && t_a + 1 < t_b) begin(t_a + 1, 0);

            // One iteration.  HN: tile t + 1 exists.
            auto iter = [&](int t, auto hn, f32x16 (&sc)[2], f32x16 (&sn)[2]) {
                constexpr bool HN = decltype(hn)::value;
                const int st = (t - t_a + 1) & 1;
                const char* Kb = reinterpret_cast<const char*>(sm[st]);
                const char* Vb = reinterpret_cast<const char*>(sm[st] + TILE);
                const float off = st_.offset(a.c, down);
                bf16x8 rk[KR], tv[NR], pf[4];
                auto rd_k = [&](int g) { rk[g % KR] = F.row(Kb, 32 * (g / KS), g % KS); };
                auto rd_v = [&](int f) { tv[f % NR] = F.tr(Vb, f % OB, f / OB); };
                float sum = 0.0f;
                if constexpr (HN) {
                    zero(sn[0]);
                    zero(sn[1]);
#pragma unroll
                    for (int g = 0; g < KR - 1; ++g) rd_k(g);
                }
                // A
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    if constexpr (HN) {
                        const int jb = i / KS, kk = i % KS;
                        sn[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rk[i % KR], qf[kk], sn[jb], 0, 0, 0);
                        if (i + KR - 1 < NA) rd_k(i + KR - 1);
                    }
#pragma unroll
                    for (int x = i * EA; x < (i + 1) * EA; ++x) {
                        const int jb = x >> 4, e = x & 15;
                        const float p = weight(sc[jb][e], a.c, off);
                        sc[jb][e] = p;
                        sum += p;
                        if ((e & 7) == 7) pf[2 * jb + (e >> 3)] = pack_bf16x8(sc[jb], e - 7);
                    }
                    if (i >= NA - OB) rd_v(i - (NA - OB));
                    if constexpr (HN) __builtin_amdgcn_sched_barrier(0);
                }
                st_.add(sum);
                // B, ahead of the other block's waves: their exponentials fill the slots between its MFMAs (3% at head_dim 128)
                float mx = -INFINITY;
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int f = 0; f < NB; ++f) {
                    const int ks = f / OB, ob = f % OB;
                    st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tv[f % NR], pf[ks], st_.o[ob], 0, 0, 0);
                    if (f + OB < NB) rd_v(f + OB);
                    if constexpr (HN) {
#pragma unroll
                        for (int x = f * EB; x < (f + 1) * EB; ++x) mx = fmaxf(mx, sn[x >> 4][x & 15]);
                        if constexpr (E4) {
                            // unit t + 1 from registers (past the last tile stale codes, which nobody reads)
                            constexpr int EVERY = NB / (2 * NU);
                            if (f % EVERY == EVERY - 1) {
                                const int j = f / EVERY;
                                if (j < NU) put_unit(ck, j, sm[st ^ 1]);
                                else put_unit(cv, j - NU, sm[st ^ 1] + TILE);
                            }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
                if constexpr (HN) st_.absorb(mx, a.c);
                wait_lds();
                if constexpr (!E4) wait_vmcnt<0>();  // unit t + 1
                __builtin_amdgcn_s_barrier();        // everyone is done with unit t's stage; unit t + 1 is visible
                if (t + 2 < t_b) begin(t + 2, st);
            };
            using T1 = std::true_type;
            using F0 = std::false_type;
            int t = t_a;
            for (; t + 2 < t_b; t += 2) {
                iter(t, T1{}, s0, s1);
                iter(t + 1, T1{}, s1, s0);
            }
            if (t + 1 < t_b) {
                iter(t, T1{}, s0, s1);
                iter(t + 1, F0{}, s1, s0);
            } else {
                iter(t, F0{}, s0, s1);
            }
        }
    }
    const int past = real && store_row<bf16, HD>(a, st_, trow, head, empty, split, down > 0.0f) ? kPast : 0;
    return past | (top ? kTop : 0);
}

template <int HD, bool E4>
__global__ __launch_bounds__(256, 2) void attn_paged_tiles_k(PagedArgs a) {
    // as one_or_two_passes; where a row of the largest powers was found, the second pass is anew from the start, and there
    // may be a third
    __shared__ TilesLds<HD> lds;
    const int tid = threadIdx.x;
    if (tid == 0) lds.past = 0, lds.top = 0;
    const int found = tiles_pass<HD, E4, false>(lds, a, tid, static_cast<int>(blockIdx.x), 0.0f);
    if (found & kPast) lds.past = 1;
    if (E4 && found & kTop) lds.top = 1;
    lds_barrier();
    if (__builtin_expect(lds.past || (E4 && lds.top), 0)) {
#pragma unroll 1
        for (float down = E4 && lds.top ? 0.0f : kDown;; down = kDown) {
            lds_barrier();
            if (threadIdx.x == 0) lds.past = 0;
            const int again = tiles_pass<HD, E4, true>(lds, fresh_argument<PagedArgs>(), fresh(tid), fresh_uniform(static_cast<int>(blockIdx.x)), down);
            lds_barrier();  // (a tile without keys has none)
            if (again & kPast) lds.past = 1;
            lds_barrier();
            if (down > 0.0f || !lds.past) return;
        }
    }
}

template <int HD, bool E4>
void launch(const PagedArgs& a, unsigned blocks, hipStream_t s) {
    attn_paged_tiles_k<HD, E4><<<blocks, 256, 0, s>>>(a);
    AIC_LAUNCH_CHECK("attn_paged");
}

}  // namespace

void attn_paged_tiles(const PagedArgs& a, bool e4m3, int head_dim, unsigned blocks, hipStream_t s) {
    if (head_dim == 32) e4m3 ? launch<32, true>(a, blocks, s) : launch<32, false>(a, blocks, s);
    else if (head_dim == 64) e4m3 ? launch<64, true>(a, blocks, s) : launch<64, false>(a, blocks, s);
    else e4m3 ? launch<128, true>(a, blocks, s) : launch<128, false>(a, blocks, s);
}

}  // namespace aic::hip
