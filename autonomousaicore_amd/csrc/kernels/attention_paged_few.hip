// Attention over the paged cache for few query rows per key/value head (single tokens, drafted tokens): bound by
// reading the cache, once for every 32 rows.
//
// A group of up to 32 query rows of one sequence and key/value head is worked on by a block at a time.  The
// four waves take tiles of 32 keys in turn, each into LDS of its own, so no barrier stands between a
// tile's arrival and its use, and each wave keeps its own copies in flight; their (m, l, O) are joined
// once at the end.  The page ids of the keys are in LDS before the first tile, so a tile's addresses
// cost no memory latency.
//
// Shares: the keys of all groups, in steps of 128, form one list that is cut into as many equal parts as blocks
// are resident at once, so that batches of uneven lengths end together; a group that a cut divides leaves
// its parts' states in the workspace and attn_paged_few_join_k adds them.  (Equal splits per
// sequence ran in one and a half rounds of blocks: 28.7 us at best and 40 us at worst for 32 e4m3 caches of up to
// 8000 tokens, by the number of splits.)  Where the groups are few, each is cut by itself into parts of nearly
// a share: a block that ends one group and begins another waits twice for its first tile, which is then
// most of its time.  Every block finds its part from offsets and lens by itself.
//
// 32 single tokens on e4m3 caches of up to 8000 tokens, 16 heads of 128 over 2: 29.7 us, 84 MB at 2.8 TB/s (the kernel
// 24 us, of which 7 before the first tile, and 5 for the join); on bf16 caches of up to 16384, 16 over 8: 242 us,
// 5.7 TB/s of the 6.5 that reading alone reaches; one token of 12 heads of 64 on 513: 8.6 us, a chain of latencies.
//
// Tiles arrive by direct global -> LDS copies, two stages per wave: 32 KB per wave at head_dim 128 in bf16 (one
// block and up to 128 KB in flight per CU), 16 KB in e4m3 (two blocks).
//
// e4m3 tiles stay codes in LDS.  K fragments are converted as they are read, a lane holding codes of one key
// and so one power of two; V fragments (transposed reads) hold eight keys, so they are converted with
// the tile's largest power 2^E, and the weights take 2^(e - E).  That loses what is below 2^-86 of
// the tile's largest: where the tile's powers differ by more than 2^40, its keys are added one by one instead,
// so that a hidden key's large v costs a visible one nothing; and
// from power kTopByte on, where other rows' codes with that power would be past the range.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attention_paged_shares.hpp"

namespace aic::hip {

namespace {

template <int HD, bool E4, int NW>
struct FewLds {
    static constexpr int TILE = 32 * HD * (E4 ? 1 : 2);          // bytes of a tile of K or V
    static constexpr int STAGE = 2 * TILE + (E4 ? 256 : 0);      // and the exponents of 32 keys of K, then of V, a word each
    static constexpr int WAVE = 2 * STAGE;
    static constexpr int BYTES = NW * WAVE > NW * 32 * HD * 4 ? NW * WAVE : NW * 32 * HD * 4;  // also the waves' O at the end
    static constexpr int COPIES = 2 * (TILE / 1024) + (E4 ? 1 : 0);  // of a stage
};

// A byte per lane to LDS, zero-extended to words: lane i's at lds + 4 i.  As dma16.
__device__ __forceinline__ void dma_byte(const void* g, const void* lds) {
    const uint32_t l = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_ubyte %1, off"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(l)), "v"(g)
                 : "memory", "m0");
}
__device__ const uint8_t kNoExponent = 1;  // of keys without a page: their codes are NaN, their power the least

// [32][HD] tiles of codes, 16-byte chunks swizzled by row: 16 consecutive rows of one chunk (ds_read_b128) and the
// rows {0-3, 8-11} + 4h of two neighbouring chunks (transposed reads) lie in different banks (the latter two-way at
// head_dim 32).
template <int HD>
__device__ __forceinline__ int swz8(int row) {
    if constexpr (HD == 128) return ((row >> 1) & 1) << 1 | ((row >> 3) & 1) << 2 | ((row >> 2) & 1);
    else if constexpr (HD == 64) return ((row >> 3) & 1) << 1 | ((row >> 2) & 1);
    else return (row >> 3) & 1;
}
typedef int v2i_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i_t lds_v2i_t;

//   k(t, j):     lane = key lane % 32, its 16 codes of chunk 2 j + h: two k steps of S = K Q^T, whose Q fragments
//                hold the columns 32 j + 16 h + 0..7 and + 8..15
//   v(t, ob, s): lane = column 32 ob + lane % 32, 8 codes along the keys of step s in the order of Frags::tr, by
//                one ds_read_b64_tr_b8: within 16 lanes, output lane i slot j takes byte i % 8 of the 8 at source
//                lane 2 j + i / 8, so source lane 2 j + p addresses row j, columns 8 p .. +7
template <int HD>
struct Frags8 {
    int k_off[HD / 32], v_off[HD / 32];
    __device__ __forceinline__ void init(int lane) {
        const int h = lane >> 5, r = lane & 31;
        const int g = lane >> 4, j = (lane & 15) >> 1, p = lane & 1, row = (j & 3) + 8 * (j >> 2) + 4 * h;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            k_off[i] = r * HD + (((2 * i + h) ^ swz8<HD>(r)) << 4);
            v_off[i] = row * HD + (((2 * i + (g & 1)) ^ swz8<HD>(row)) << 4) + 8 * p;
        }
    }
    __device__ __forceinline__ uint4 k(const char* t, int j) const { return *reinterpret_cast<const uint4*>(t + k_off[j]); }
    __device__ __forceinline__ uint2 v(const char* t, int ob, int s) const {
        const v2i_t x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_t*)(t + 16 * s * HD + v_off[ob]));
        return make_uint2(static_cast<uint32_t>(x[0]), static_cast<uint32_t>(x[1]));
    }
};

// What a thread knows of the tiles: where its copies and fragments lie.
template <int HD, bool E4>
struct FewLane {
    static constexpr int TILE = FewLds<HD, E4, 1>::TILE;
    static constexpr int RB = HD * (E4 ? 1 : 2), NC = RB / 16, RPS = 1024 / RB;  // bytes and chunks of a row, rows of a 1 KB copy
    uint32_t voff[TILE / 1024];
    std::conditional_t<E4, Frags8<HD>, Frags<HD>> F;
    __device__ __forceinline__ void init(int lane) {
#pragma unroll
        for (int i = 0; i < TILE / 1024; ++i) {
            const int rr = i * RPS + lane / NC;
            const int ch = (lane % NC) ^ (E4 ? swz8<HD>(rr) : swz<HD>(rr));
            voff[i] = static_cast<uint32_t>((rr - (i * RPS >= 16 ? 16 : 0)) * RB + ch * 16);
        }
        F.init(lane);
    }
};
// The work on one part: true where a sum of this thread's has left fp32's range.
template <int HD, bool E4, int NW, typename A>
__device__ __forceinline__ bool few_part(const FewArgs<A>& f, const Part& pt, const FewLane<HD, E4>& me, float down) {
    using L = FewLds<HD, E4, NW>;
    const PagedArgs& a = f.a;
    constexpr int KS = HD / 16, OB = HD / 32;
    constexpr int RB = FewLane<HD, E4>::RB, NC = FewLane<HD, E4>::NC, RPS = FewLane<HD, E4>::RPS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int ids[kIds];
    __shared__ float2 mls[NW][32];

    const Seq sq = pt.sq;
    const int Hkv = a.kv.Hkv, ps = a.kv.ps, kvh = pt.kvh, r0 = pt.r0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hl = lane >> 5;
    char* mine = lds + wave * L::WAVE;
    const bool paged = ps % (RPS > 16 ? RPS : 16) == 0;  // halves of tiles (whole ones where one copy spans both) do not leave a page

    const int32_t* tr = a.kv.table + pt.b * a.kv.ld_table;
    const int rows = min(sq.n * a.G, r0 + f.group);
    const int r = r0 + (lane & 31);
    const bool real = r < rows;
    const int tok = real ? r / a.G : 0, head = kvh * a.G + (real ? r % a.G : 0);
    const int hi = real ? sq.len - sq.n + tok : -1;
    const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;
    const int first_pos = sq.len - sq.n + r0 / a.G, last_pos = sq.len - sq.n + (rows - 1) / a.G;
    // keys of this part that the group sees
    int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0;
    k_lo = max(k_lo & ~31, pt.first);
    const int k_hi = min(last_pos + 1, pt.end);
    const uint32_t span = static_cast<uint32_t>(max(min(hi, k_hi - 1) - lo + 1, 0));

    Rows<OB> st_;
    st_.init();
    if (k_lo < k_hi) {
        bf16x8 qb[KS];
        const bf16* qp = static_cast<const bf16*>(a.q) + (sq.row0 + tok) * a.ldq + static_cast<int64_t>(head) * HD;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            const int col = E4 ? 32 * (kk >> 1) + 16 * hl + 8 * (kk & 1) : 16 * kk + 8 * hl;
            if (a.vec_q) qb[kk] = __builtin_bit_cast(bf16x8, ldg16(qp + col, real));
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) qb[kk][j] = real ? qp[col + j] : f2bf(0.0f);
        }

        // one tile's products, from the stage it arrived in
        auto compute = [&](char* kt, int k0) {
            const char* vt = kt + L::TILE;
            [[maybe_unused]] const uint32_t* ex = reinterpret_cast<const uint32_t*>(vt + L::TILE);
            f32x16 sc[1];
            zero(sc[0]);
            [[maybe_unused]] int e_max = 0;
            bool one_by_one = false;
            if constexpr (E4) {
                const uint32_t ek = ex[lane & 31];
                const float sk = exp_scale(ek);
                if (__builtin_expect(__any(ek >= kTopByte), 0)) {  // each lane what it reads
#pragma unroll
                    for (int j = 0; j < HD / 32; ++j) {
                        uint4* x = reinterpret_cast<uint4*>(kt + me.F.k_off[j]);
                        if (ek >= kTopByte) *x = e4m3_in_range(*x, ek);
                    }
                }
                const int ev = static_cast<int>(ex[32 + (lane & 31)]);
                e_max = wave_all(ev, [](int x, int y) { return max(x, y); });
                one_by_one = __any(e_max - ev > 40) || e_max >= static_cast<int>(kTopByte);
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    const uint4 x = me.F.k(kt, j);
                    sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, e4m3_bf16(make_uint2(x.x, x.y), sk)),
                                                                    qb[2 * j], sc[0], 0, 0, 0);
                    sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, e4m3_bf16(make_uint2(x.z, x.w), sk)),
                                                                    qb[2 * j + 1], sc[0], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
                    sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(me.F.row(kt, 0, kk), qb[kk], sc[0], 0, 0, 0);
            }
            // every row sees every key of the tile?
            const bool open = k0 + 31 <= first_pos && k0 + 32 <= k_hi && (a.window <= 0 || k0 > last_pos - a.window);
            auto seen = [&](int j) { return static_cast<uint32_t>(k0 + j - lo) < span; };
            if (!open) {
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[0][e] = seen(8 * (e >> 2) + 4 * hl + (e & 3)) ? sc[0][e] : -INFINITY;
                uint32_t bits = 0;  // a hidden key and a non-finite v
#pragma unroll
                for (int i = 0; i < L::TILE / 1024; ++i)
                    bits |= non_finite_bits<std::conditional_t<E4, uint8_t, bf16>>(*reinterpret_cast<const uint4*>(vt + i * 1024 + lane * 16));
                one_by_one |= __any(bits != 0) != 0;
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
            if (one_by_one) {
                if constexpr (E4)
                    add_seen_rows<HD, 1>(st_.o, sc, [&](int key, int d) {
                        uint32_t w = *reinterpret_cast<const uint32_t*>(vt + key * HD + (((d >> 4) ^ swz8<HD>(key)) << 4) + (d & 15));
                        if (ex[32 + key] >= kTopByte) w = e4m3_in_range(w, ex[32 + key]);
                        const float s = exp_scale(ex[32 + key]);
                        const auto x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, false), y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, true);
                        return make_float4(x[0], x[1], y[0], y[1]);
                    }, seen);
                else add_seen_rows<HD, 1>(st_.o, sc, [&](int key, int d) { return v4_at<bf16, HD>(vt, key, d); }, seen);
                return;
            }
            if constexpr (E4) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint4 x = *reinterpret_cast<const uint4*>(ex + 32 + 8 * g + 4 * hl);
                    const uint32_t ev[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) sc[0][4 * g + u] = __builtin_amdgcn_ldexpf(sc[0][4 * g + u], static_cast<int>(ev[u]) - e_max);
                }
            }
            [[maybe_unused]] const float sv = exp_scale(static_cast<uint32_t>(e_max));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 p = pack_bf16x8(sc[0], 8 * s);
#pragma unroll
                for (int ob = 0; ob < OB; ++ob) {
                    bf16x8 v;
                    if constexpr (E4) v = __builtin_bit_cast(bf16x8, e4m3_bf16(me.F.v(vt, ob, s), sv));
                    else v = me.F.tr(vt, ob, s);
                    st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p, st_.o[ob], 0, 0, 0);
                }
            }
        };

        const int window_keys = min((kIds - 1) * ps, 1 << 20) & ~31;  // keys whose page ids fit
        for (int w0 = k_lo, w1; w0 < k_hi; w0 = w1) {
            w1 = w0 + min(k_hi - w0, window_keys);
            const int p0 = a.kv.page_index(w0), np = a.kv.page_index(w1 - 1) - p0 + 1;
            __syncthreads();
            for (int i = tid; i < np; i += NW * 64) {
                const int page = p0 + i < a.kv.ld_table ? tr[p0 + i] : -1;
                ids[i] = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.n_pages) ? page : -1;
            }
            __syncthreads();
            const int first = w0 + 32 * wave, nt = first < w1 ? (w1 - first + 32 * NW - 1) / (32 * NW) : 0;  // this wave's tiles
            // byte offset of key's row in the pools, negative without a page; keys past the last as the last
            auto row_at = [&](int key) -> int64_t {
                key = min(key, w1 - 1);
                const int pi = a.kv.page_index(key), page = ids[pi - p0];
                const int64_t row = (static_cast<int64_t>(page) * Hkv + kvh) * ps + (key - pi * ps);
                return page < 0 ? -1 : row;
            };
            auto issue = [&](int t) {
                char* dst = mine + (t & 1) * L::STAGE;
                const int k0 = first + 32 * NW * t;
                if (paged && k0 + 32 <= w1) {
                    // each half of the tile lies in one page: uniform bases, offsets per lane made once
                    const int pi = a.kv.page_index(k0), pj = a.kv.page_index(k0 + 16);
                    const int page0 = __builtin_amdgcn_readfirstlane(ids[pi - p0]), page1 = __builtin_amdgcn_readfirstlane(ids[pj - p0]);
                    if (page0 >= 0 && page1 >= 0) {
                        const int64_t row[2] = {(static_cast<int64_t>(page0) * Hkv + kvh) * ps + (k0 - pi * ps),
                                                (static_cast<int64_t>(page1) * Hkv + kvh) * ps + (k0 + 16 - pj * ps)};
#pragma unroll
                        for (int i = 0; i < L::TILE / 1024; ++i) {
                            const int64_t at = row[i * RPS >= 16 ? 1 : 0] * RB;
                            dma16s(a.kv.kp + at, me.voff[i], dst + i * 1024);
                            dma16s(a.kv.vp + at, me.voff[i], dst + L::TILE + i * 1024);
                        }
                        if constexpr (E4)
                            dma_byte((hl ? a.kv.ve : a.kv.ke) + (lane & 16 ? row[1] : row[0]) + (lane & 15), dst + 2 * L::TILE);
                        return;
                    }
                }
                const char* none = reinterpret_cast<const char*>(&kNoPage);
#pragma unroll
                for (int i = 0; i < L::TILE / 1024; ++i) {
                    const int rr = i * RPS + lane / NC;
                    int ch = lane % NC;
                    if constexpr (E4) ch ^= swz8<HD>(rr);
                    else ch ^= swz<HD>(rr);
                    const int64_t row = row_at(k0 + rr), at = row * RB + ch * 16;
                    dma16(row >= 0 ? a.kv.kp + at : none, dst + i * 1024);
                    dma16(row >= 0 ? a.kv.vp + at : none, dst + L::TILE + i * 1024);
                }
                if constexpr (E4) {
                    const int64_t row = row_at(k0 + (lane & 31));
                    dma_byte(row >= 0 ? (hl ? a.kv.ve : a.kv.ke) + row : &kNoExponent, dst + 2 * L::TILE);
                }
            };
            wait_vmcnt<0>();  // Q is there: left to the compiler, which does not count the copies, it would be waited for with all of them, at every tile
            if (nt > 0) issue(0);
            if (nt > 1) issue(1);
            for (int t = 0; t < nt; ++t) {
                if (t + 1 < nt) wait_vmcnt<L::COPIES>();  // tile t has landed; t + 1 may be in flight
                else wait_vmcnt<0>();
                compute(mine + (t & 1) * L::STAGE, first + 32 * NW * t);
                wait_lds();  // the tile has been read
                if (t + 2 < nt) issue(t + 2);
            }
        }
    }

    // The waves' states joined: everyone's factor against the common maximum, then the sums over the waves.
    bool over = false;
    if (hl == 0) mls[wave][lane] = make_float2(st_.m, st_.l);
    __syncthreads();  // also: the tiles have been read
    const int q = lane & 31;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, mls[w][q].x);
    const float base = M == -INFINITY ? 0.0f : M;
    const float factor = __builtin_amdgcn_exp2f((st_.m - base) * a.c);
    float* os = reinterpret_cast<float*>(lds);  // [NW][32][HD], 16-byte groups swizzled by row
#pragma unroll
    for (int ob = 0; ob < OB; ++ob)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c4 = (ob * 32 + 8 * g + 4 * hl) / 4;
            *reinterpret_cast<float4*>(os + (wave * 32 + q) * HD + ((c4 ^ (q & 7)) << 2)) =
                make_float4(st_.o[ob][4 * g] * factor, st_.o[ob][4 * g + 1] * factor, st_.o[ob][4 * g + 2] * factor,
                            st_.o[ob][4 * g + 3] * factor);
        }
    __syncthreads();
    for (int i = tid; i < 32 * (HD / 4); i += NW * 64) {
        const int qr = i / (HD / 4), c4 = i % (HD / 4), rr = r0 + qr;
        if (rr >= rows) break;
        const int tk = rr / a.G, hd_ = kvh * a.G + rr % a.G, h2 = sq.len - sq.n + tk;
        const int l2 = a.window > 0 ? max(0, max(h2, 0) - a.window + 1) : 0;
        const bool empty = h2 < 0 || max(l2, k_lo) > min(h2, k_hi - 1);
        float mm = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, mls[w][qr].x);
        const float bs = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 ml = mls[w][qr];
            l = fmaf(__builtin_amdgcn_exp2f((ml.x - bs) * a.c), ml.y, l);
        }
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(os + (w * 32 + qr) * HD + ((c4 ^ (qr & 7)) << 2));
            v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
        }
        Range range;
        range.look(v.x), range.look(v.y), range.look(v.z), range.look(v.w);
        over |= !empty && range.left(l);
        const float inv = empty ? 0.0f : 1.0f / l;
        const float4 y = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        const int64_t t = sq.row0 + tk;
        if (!pt.whole) {
            const int64_t at = static_cast<int64_t>(pt.slot) * f.group + qr;
            if (c4 == 0 && !(down > 0.0f)) f.part_ml[at] = make_float2(mm, empty ? 0.0f : l == 0.0f ? -1.0f : l);
            if (!empty) store4(f.part_o + at * HD + c4 * 4, y, true, down > 0.0f);
            continue;
        }
        bf16* op = static_cast<bf16*>(a.o) + t * a.ldo + static_cast<int64_t>(hd_) * HD + c4 * 4;
        store4(op, y, a.vec_o, down > 0.0f);
        if (a.lse && c4 == 0 && !(down > 0.0f)) a.lse[t * a.H + hd_] = empty ? -INFINITY : log_sum(bs, l, a.c);
    }
    return over;
}

// NW waves: four, and two blocks per CU (bf16 at head_dim 128: one); or eight that divide a group among them where nothing
// else is divided and a block is alone on its CU.
template <int HD, bool E4, int NW, typename A>
__global__ __launch_bounds__(NW * 64, NW == 8 || (HD == 128 && !E4) ? 1 : 2) void attn_paged_few_k(FewArgs<A> f) {
    FewLane<HD, E4> me;
    me.init(threadIdx.x & 63);
    work_on_parts<NW == 4>(f, [&](const Part& pt, float down) { return few_part<HD, E4, NW>(f, pt, me, down); });
}

// Blocks that are resident at once on 256 CUs: LDS holds one of bf16 at head_dim 128, two of the others.
int64_t resident(int64_t head_dim, DType type) { return head_dim == 128 && !holds_codes(type) ? 256 : 512; }

template <int HD, bool E4, int NW, typename A>
void launch(const FewArgs<A>& f, int64_t blocks, hipStream_t s) {
    constexpr int bytes = FewLds<HD, E4, NW>::BYTES;
    static std::atomic<bool> allowed[64];  // by device
    int dev = 0;
    AIC_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !allowed[dev].load()) {
        AIC_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_few_k<HD, E4, NW, A>),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) allowed[dev].store(true);
    }
    attn_paged_few_k<HD, E4, NW><<<static_cast<unsigned>(blocks), NW * 64, bytes, s>>>(f);
    AIC_LAUNCH_CHECK("attn_paged");
}

template <int HD, bool E4, typename A>
void launch(const FewArgs<A>& f, hipStream_t s) {
    const int64_t pairs = (std::is_same_v<A, PickedArgs> ? int64_t{1} : f.a.kv.Hkv) * f.a.B;
    AIC_CHECK(pairs <= INT32_MAX, OutOfRange, "attn_paged: too many sequences in one call");
    if (f.shares == 0) {
        // eight waves' stages are beyond the LDS for bf16 at head_dim 128; with more blocks than CUs four waves keep two of them there
        if constexpr (HD < 128 || E4) {
            if (pairs <= 256) return launch<HD, E4, 8>(f, pairs, s);
        }
        return launch<HD, E4, 4>(f, pairs, s);
    }
    launch<HD, E4, 4>(f, f.shares, s);
    attn_paged_few_join_k<HD><<<dim3(static_cast<unsigned>(pairs), static_cast<unsigned>((f.group + 3) / 4)), 256, 0, s>>>(f);
    AIC_LAUNCH_CHECK("attn_paged join");
}

int64_t group_of(int64_t max_q, int64_t G) { return std::clamp<int64_t>(max_q * G, 1, 32); }

// Longest cache whose groups are not divided: finding shares and joining them cost about 7 us, and 128 keys of an
// undivided group 0.3 us (head_dim 64) to 0.7 us (128).  One sequence of 1600 tokens, shares and whole: 13.3 and
// 11.9 us with 12 heads of 64, 15.9 and 20.8 us with 8 of 128; of 2048: 13.3 and 13.9, 16.1 and 23.9 us.  With a group
// for most CUs nothing is won by dividing up to 2048: 32 sequences with 8 heads of 128, 47.6 and 42.8 us.
// e2m1, whose tiles take less time to come: 32 sequences of 4096, 37.1 in shares and 32.8 us whole, of a quarter of that and more 31.2 and
// 31.8, 24 sequences 34.4 and 32.0, 29.8 and 31.8 (one of 4096 among others of 512, 20 and 31); 64 of them 54.3 and 55.7.
// Rows with pages of their own, heads of 128, shares and whole.  Rows of one length, as those of long caches mostly are, end together where
// their blocks fill a round of the card: 256 of 8192 tokens, bf16 191 and 188 us, e2m1 69 and 62; 128 of 4096, bf16 50.3 and 46.9, e2m1
// 30.1 and 31.7; of 8192, 102.1 and 102.3, 46.1 and 55.0; but 288 of 4096, a round and a little, 118 and 140, 48 and 57; 384 of
// 8192 280 and 283; 512, 364 and 361, e2m1 124 and 114.  A caller's lengths may differ: 8 long rows among 216 of 1024 tokens are left alone at
// the end, of 4096 30 and 48 us, of 8192 35 and 83, of 32768 54 and 296; with 504, 59 and 60, 58 and 94, 76 and 307.  So whole up to 8192.
// From 2048 on at any length: these are a chunk's rows, which choose the same pages and take them from each other's cache while their blocks
// run in step: 2600 of 4096, 808 and 486 us, of 16384, 3242 and 1653, of a quarter of that and more, 1886 and 1134 (pages chosen at random:
// 3316 and 3388, 2029 and 2075); 8 of 32768 among 2592 of 1024, 267 and 380.
int64_t whole_len(int64_t pairs, int64_t head_dim, DType type, bool picked) {
    const bool one_round = pairs <= 256;
    if (picked && pairs >= 2048) return kMaxLen;
    if (picked && (pairs >= 512 || (pairs >= 224 && one_round))) return 8192;
    if (picked ? pairs >= 128 && one_round : type == DType::UInt4 && head_dim == 128 && pairs >= 192 && one_round) return 4096;
    return pairs >= 192 && !picked ? 2048 : head_dim < 128 ? 1536 : 1024;
}

}  // namespace

// One group; or two where the cache is e4m3 and head_dim 128, whose tiles of 128 rows go through registers: 30 sequences of
// up to 8000 tokens, 16 heads over 2, 64 rows: 41.6 us so, 66.6 us there; one sequence: 22.5 and 26.7 us; 96 rows on
// up to 4000: 41.1 and 39.1 us.  bf16, 64 rows: 61.6 and 55.5 us; head_dim 64 25.0 and 22.7 us in e4m3.
// e2m1: two where there are 200000 keys to read.  64 rows over 8 heads of 128 of 8 sequences of 3000 tokens: 29.2 us so and 28.9 there; of 8000,
// 41.1 and 48.3; 30 of 1000, 31.2 and 38.0; 16 of 1000, 30.7 and 24.0.  64 rows, 12 heads of 64: 4 of 8000, 27.7 and 33.0;
// 16 of 1000, 20.3 and 24.3; 8 of 1000, 20.3 and 18.1.
bool few_rows(int64_t pairs, int64_t max_q, int64_t max_len, int64_t G, int64_t head_dim, DType type) {
    const bool two = type == DType::UInt4 ? pairs > 200000 / std::max<int64_t>(max_len, 1) : type == DType::UInt8 && head_dim == 128;
    return max_q * G <= (two ? 64 : 32);
}

int64_t few_workspace(int64_t B, int64_t Hkv, int64_t max_q, int64_t max_len, int64_t G, int64_t head_dim, DType type, bool picked) {
    if (max_len <= whole_len(B * Hkv, head_dim, type, picked)) return 0;
    return (2 * resident(head_dim, type) * group_of(max_q, G) * (head_dim + 2) * 4 + (B + 1) * 8 + 15) / 16 * 16;
}

template <typename A>
void attn_paged_few(const A& a, int64_t max_q, DType type, int head_dim, void* workspace, hipStream_t s) {
    // e2m1 and picked pages: shares of two steps where there are few.  One token, 2 heads of 128, 64 pages of 64: 13.6 us so and 15.1 in fours (bf16 14.4 and
    // 16.2), 256 pages, 18.0 and 17.5; of 2000 tokens, 13.4 and 15.5; of 16000, 250 steps, 18.3 and 17.6; of 32000, 24.9 and 20.7; 8 heads, 64
    // pages, 14.0 and 15.7.  (Other calls keep their parts, and so their sums' last bits.)
    const int least = std::is_same_v<A, PickedArgs> || type == DType::UInt4 ? 2 : kLeast;
    FewArgs<A> f{a, static_cast<int>(group_of(max_q, a.G)), 0, least, nullptr, nullptr, nullptr};
    if (workspace) {
        f.shares = static_cast<int>(resident(head_dim, type));
        f.part_o = static_cast<float*>(workspace);
        f.part_ml = reinterpret_cast<float2*>(f.part_o + 2LL * f.shares * f.group * head_dim);
        f.plan = reinterpret_cast<int64_t*>(f.part_ml + 2LL * f.shares * f.group);
    }
    if (type == DType::UInt4) return attn_paged_e2m1_few(f, head_dim, s);
    const bool e4m3 = type == DType::UInt8;
    if (head_dim == 32) e4m3 ? launch<32, true>(f, s) : launch<32, false>(f, s);
    else if (head_dim == 64) e4m3 ? launch<64, true>(f, s) : launch<64, false>(f, s);
    else e4m3 ? launch<128, true>(f, s) : launch<128, false>(f, s);
}

template void attn_paged_few(const PagedArgs&, int64_t, DType, int, void*, hipStream_t);
template void attn_paged_few(const PickedArgs&, int64_t, DType, int, void*, hipStream_t);

}  // namespace aic::hip
