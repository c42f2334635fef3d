// Attention over an e2m1 cache for few query rows per key/value head, bf16 queries: bound by reading the cache, 68 bytes for
// a key or value of 128, and by what the vector units have to do for them.
//
// Blocks, shares and joins are attention_paged_shares.hpp's; four (or eight) waves take tiles of 32 keys in turn, each through LDS of its
// own.  A tile's codes arrive by direct global -> LDS copies, two tiles ahead.  K's become fragments as they are read: a lane
// holds one key's columns in runs of 32 (the order of the columns is free, as long as Q's is the same), so that a fragment has
// one power.  V's become a bf16 tile in LDS for the products' transposed reads; code times power is exact in bf16.
//
// R: query rows of a tile.  Groups of up to 16 rows, nearly all of single tokens, run on 16-row matrix instructions: with 32
// rows, of which most are none, the softmax's instructions and the accumulators would be twice as many (8 heads of 128, one token: of
// 1000, 13.3 us and 15.3 on 32 rows; 32 sequences of up to 8000, 50.8 and 63.9; 12 heads of 64, 45.7 and 55.7).
//
// 32 tokens over 8 heads of 128 on caches of up to 16384: 82 us, 4.5 TB/s of codes and exponents, 90% of a large copy's rate; 16 x 5 drafted
// tokens over 16 heads on up to 3000, pages of 24: 26.7 us, 2.5 TB/s, where a block has 12 tiles for each wave at most and
// a launch, the look-ups and the joining of its waves are a third; one token, 12 heads of 64 on 513: 7.9 us, latency.
#include <algorithm>
#include <atomic>

#include "attention_paged_shares.hpp"

namespace aic::hip {

namespace {

// The bytes of a key's head to LDS, zero-extended to words: a word (head_dim 128), two bytes or one.  As dma16.
template <int HD>
__device__ __forceinline__ void dma_exps(const void* g, const void* lds) {
    const uint32_t l = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
    if constexpr (HD == 128)
        dma4(g, lds);
    else if constexpr (HD == 64)
        asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_ushort %1, off"
                     :
                     : "s"(__builtin_amdgcn_readfirstlane(l)), "v"(g)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_ubyte %1, off"
                     :
                     : "s"(__builtin_amdgcn_readfirstlane(l)), "v"(g)
                     : "memory", "m0");
}
// Whether one of four bytes is 255.
__device__ __forceinline__ bool any_nan_group(uint32_t w) { return ((~w - 0x01010101u) & w & 0x80808080u) != 0; }

template <int HD, int NW, int R>
struct Lds4 {
    static constexpr int CODES = 16 * HD;              // bytes of a tile's codes of K or V
    static constexpr int STAGE = 2 * CODES + 256;      // and a word of exponents for each of 32 keys of K, then of V
    static constexpr int V = 2 * STAGE;                // V's tile as bf16 behind the stages
    static constexpr int WAVE = 2 * STAGE + 64 * HD;
    static constexpr int BYTES = std::max(NW * WAVE, NW * R * HD * 4);    // also the waves' O at the end
    static constexpr int COPIES = (2 * CODES + 1023) / 1024 + 1;          // of a stage
};

// A lane's places in a tile, as bytes.  Codes: rows of HD / 32 chunks of 16 bytes, swizzled so that a chunk of 16 neighbouring rows
// lies in different banks.  V as bf16: 16-byte chunks swizzled so that the same holds, and that the transposed reads, which take
// 4 rows per 16 lanes, spread over the banks as well.  Swizzles go by a row's place among 16, so that what lies 16 rows on is an
// instruction's offset, and chunks of a row are exclusive-ors of constants.
template <int HD, int R>
struct Lane4 {
    static constexpr int RB = HD / 2, NC = RB / 16, NV = HD / 64 > 0 ? HD / 64 : 1;  // bytes and chunks of a row of codes, units of V of a lane
    static constexpr int KL = R == 16 ? 4 : 2, KH = 32 / (64 / KL);  // lanes of a key; keys of a lane
    static constexpr int KW = HD / 8 / KL;                           // words of a key in a lane: 8 columns each
    static constexpr int KC = 64 / KL;                               // lanes of a column of keys
    int k, ke, ke_shift, v, ve, put, frag;
    uint32_t voff;  // 16 bytes of 16 rows of a pool (head_dim 128)
    __device__ static __forceinline__ int swz4(int r) { return NC == 4 ? (r >> 2) & 3 : NC == 2 ? (r >> 3) & 1 : 0; }
    // row of V's bf16 tile, chunk of 8 columns
    __device__ static __forceinline__ int v_swz(int r) {
        if constexpr (R == 32) return swz<HD>(r);
        else if constexpr (HD == 128) return 4 * (r & 3) | 2 * ((r >> 2) & 1) | ((r >> 3) & 1);
        else if constexpr (HD == 64) return 2 * ((r >> 1) & 3) | ((r >> 3) & 1);
        else return 2 * ((r >> 2) & 1) | ((r >> 3) & 1);
    }
    __device__ static __forceinline__ int v_chunk(int r, int ch) { return r * HD * 2 + ((ch ^ v_swz(r)) << 4); }
    __device__ __forceinline__ explicit Lane4(int lane) {
        const int r = lane & (KC - 1), q = lane / KC, at = q * (RB / KL);  // key, its part, the part's byte of a row
        k = r * RB + ((at >> 4 ^ swz4(r)) << 4) + (at & 15);
        ke = r * 4;
        ke_shift = NC == 1 ? 0 : 8 * (q * (HD / KL) / kGroup);
        // 16 lanes hold a chunk of 16 rows of V each
        const int vr = NC == 4 ? lane & 15 : lane & 31, g = NC == 4 ? lane >> 4 : NC == 2 ? lane >> 5 : 0;
        v = vr * RB + ((g ^ swz4(vr)) << 4);
        ve = vr * 4 + g;
        put = v_chunk(vr, 4 * g);
        const int s = lane & 15, fr = 4 * (lane >> 4) + (s >> 2), c = s & 3;
        frag = v_chunk(fr, c >> 1) + (c & 1) * 8;
        voff = static_cast<uint32_t>(lane / NC * RB + ((lane % NC ^ swz4(lane / NC)) << 4));
    }
    // Words of the lane's u-th key; the lane's columns are HD / KL neighbouring ones.
    __device__ __forceinline__ void k_words(const char* t, int u, uint32_t (&w)[KW]) const {
        const char* p = t + u * KC * RB;
        if constexpr (KW >= 4) {
#pragma unroll
            for (int i = 0; i < KW / 4; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(p + (k ^ (i << 4)));
                w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
            }
        } else if constexpr (KW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(p + k);
            w[0] = x.x, w[1] = x.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p + k);
        }
    }
    __device__ __forceinline__ uint32_t k_exps(const char* exps, int u) const { return *reinterpret_cast<const uint32_t*>(exps + ke + u * KC * 4); }
    // Byte of word i's group, from the key's word of them.
    __device__ __forceinline__ uint32_t k_byte(uint32_t e, int i) const { return e >> (ke_shift + (HD / KL > kGroup ? 8 * (8 * i / kGroup) : 0)) & 255u; }
    __device__ static __forceinline__ bool k_nan(uint32_t e) { return NC == 1 ? e == kNanGroup : any_nan_group(NC == 2 ? e & 0xffffu : e); }
    // V's bf16 tile from codes and words of exponents; the largest byte of the lane's groups.
    __device__ __forceinline__ uint32_t put_v(const char* codes, const char* exps, char* tile, bool mine) const {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(codes + v + i * 16 * RB);
            const uint32_t e = *reinterpret_cast<const uint8_t*>(exps + ve + i * 64);
            most = max(most, e);
            if (NC == 1 && !mine) break;  // half of the lanes hold all
            const float s = scale_of(e);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(tile + (put ^ (c << 4)) + i * 32 * HD) = e2m1_bf16(w[c], s);
        }
        return most;
    }
    __device__ __forceinline__ void put_nan(const char* exps, char* tile) const {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (*reinterpret_cast<const uint8_t*>(exps + ve + i * 64) == kNanGroup)
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(tile + (put ^ (c << 4)) + i * 32 * HD) = make_uint4(~0u, ~0u, ~0u, ~0u);
    }
    // A byte's power; of kNanGroup no number, for what it makes is overwritten.
    __device__ static __forceinline__ float scale_of(uint32_t e) { return __uint_as_float(e << 23); }
    // Operand of O^T += V^T P^T, 8 keys of one column: R 16: column 16 ob + lane % 16, keys 4 q + 0..3 and 16 more, q = lane / 16.
    __device__ __forceinline__ bf16x8 v_frag16(const char* tile, int ob) const {
        const char* p = tile + (frag ^ (ob << 5));
        const v4i16_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)p);
        const v4i16_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(p + 16 * HD * 2));
        const uint2 a = __builtin_bit_cast(uint2, x), b = __builtin_bit_cast(uint2, y);
        return __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
    }
};

// The running state of R query rows: lane owns row lane % R, the sum of its keys' weights, and HD / KL columns of O.
template <int HD, int R>
struct State {
    static constexpr int KL = R == 16 ? 4 : 2, NS = 32 / KL, NO = HD / R;  // scores of a tile in a lane; accumulators
    using acc_t = std::conditional_t<R == 16, f32x4, f32x16>;
    acc_t o[NO];
    float m, l;
    // Key of the tile that score e stands for, column of element e of accumulator ob.
    __device__ static __forceinline__ int key(int e, int lane) { return R == 16 ? 16 * (e >> 2) + 4 * (lane >> 4) + (e & 3) : 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }
    __device__ static __forceinline__ int column(int ob, int e, int lane) {
        return R == 16 ? 16 * ob + 4 * (lane >> 4) + e : 32 * ob + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    }
    template <typename F>
    __device__ static __forceinline__ float across(float x, F f) {  // over a row's lanes
        if constexpr (R == 16) x = facing_op<16>(x, f);
        return facing_op<32>(x, f);
    }
    __device__ __forceinline__ void init() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int e = 0; e < NS; ++e)
                if (e < (R == 16 ? 4 : 16)) o[i][e] = 0.0f;
    }
    // Whether a row maximum (over all of its lanes) moves the reference by more than 2^8, of any row.
    __device__ __forceinline__ bool moves(float mx, float c) const { return __ballot((mx - m) * c > kLazyRescale) != 0; }
    __device__ __forceinline__ void absorb(float mx, float c) {
        const bool grow = (mx - m) * c > kLazyRescale;
        const float m_new = grow ? mx : m;
        const float alpha = m == -INFINITY ? 0.0f : grow ? __builtin_amdgcn_exp2f((m - m_new) * c) : 1.0f;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < NO; ++i) o[i] *= alpha;
        m = m_new;
    }
    __device__ __forceinline__ float offset(float c, float down) const { return m == -INFINITY ? -down : fmaf(-m, c, -down); }
};

// As add_seen_rows (attention_paged.hpp): o += p v key by key, only where the row sees the key.
template <int HD, int R, typename Seen>
__device__ __forceinline__ void add_seen(State<HD, R>& st_, const float (&p)[State<HD, R>::NS], const char* tile, int lane, Seen seen) {
    using S = State<HD, R>;
#pragma unroll
    for (int e = 0; e < S::NS; ++e)
#pragma unroll 1
        for (int q = 0; q < S::KL; ++q) {
            const float w = __shfl(p[e], lane % R + R * q, 64);
            const int key = S::key(e, R * q);
            const bool s = seen(key);
#pragma unroll
            for (int ob = 0; ob < S::NO; ++ob)
#pragma unroll
                for (int g = 0; g < (R == 16 ? 1 : 4); ++g) {
                    const int d = S::column(ob, 4 * g, lane);
                    const bf16x4 x = *reinterpret_cast<const bf16x4*>(tile + Lane4<HD, R>::v_chunk(key, d >> 3) + (d & 7) * 2);
#pragma unroll
                    for (int u = 0; u < 4; ++u) st_.o[ob][4 * g + u] = s ? fmaf(w, bf2f(x[u]), st_.o[ob][4 * g + u]) : st_.o[ob][4 * g + u];
                }
        }
}

// The work on one part: true where a sum of this thread's has left fp32's range.
template <int HD, int NW, int R, typename A>
__device__ __forceinline__ bool few4_part(const FewArgs<A>& f, const Part& pt, float down) {
    using L = Lds4<HD, NW, R>;
    using P = Lane4<HD, R>;
    using S = State<HD, R>;
    const PagedArgs& a = f.a;
    constexpr int KS = P::KW, KH = P::KH, RB = P::RB, NC = P::NC;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int ids[kIds];
    __shared__ float2 mls[NW][R];

    // one for the whole block, which the compiler does not see where parts follow one another: in scalar registers
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const uint64_t row0 = static_cast<uint64_t>(pt.sq.row0);
    const Seq sq{static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(same(static_cast<int>(row0 >> 32)))) << 32 |
                                      static_cast<uint32_t>(same(static_cast<int>(row0)))),
                 same(pt.sq.n), same(pt.sq.len)};
    const int Hkv = a.kv.Hkv, ps = a.kv.ps, kvh = same(pt.kvh), r0 = same(pt.r0), seq = same(pt.b);
    const int part_first = same(pt.first), part_end = same(pt.end);
    const int tid = threadIdx.x, lane = tid & 63, wave = same(tid >> 6);
    char* mine = lds + wave * L::WAVE;

    const int32_t* tr = a.kv.table + seq * a.kv.ld_table;
    const int rows = min(sq.n * a.G, r0 + f.group);
    const int r = r0 + lane % R;
    const bool real = r < rows;
    const int tok = real ? r / a.G : 0, head = kvh * a.G + (real ? r % a.G : 0);
    const int hi = real ? sq.len - sq.n + tok : -1;
    const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;
    const int first_pos = same(sq.len - sq.n + r0 / a.G), last_pos = same(sq.len - sq.n + (rows - 1) / a.G);
    // keys of this part that the group sees
    int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0;
    k_lo = max(k_lo & ~31, part_first);
    const int k_hi = min(last_pos + 1, part_end);
    const uint32_t span = static_cast<uint32_t>(max(min(hi, k_hi - 1) - lo + 1, 0));

    S st_;
    st_.init();
    if (k_lo < k_hi) {
        bf16x8 qb[KS];
        const bf16* qp = static_cast<const bf16*>(a.q) + (sq.row0 + tok) * a.ldq + static_cast<int64_t>(head) * HD + lane / R * (HD / P::KL);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            if (a.vec_q) qb[kk] = __builtin_bit_cast(bf16x8, ldg16(qp + 8 * kk, real));
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) qb[kk][j] = real ? qp[8 * kk + j] : f2bf(0.0f);
        }
        std::conditional_t<R == 32, Frags<HD>, char> F;
        if constexpr (R == 32) F.init(lane);

        // R 32: made anew for each tile, for kept through the loop they would take registers that it does not have
        [[maybe_unused]] const P own(lane);
        auto places = [&] {
            if constexpr (R == 16) return own;
            else return P(fresh(lane));
        };
        // A tile's scores and the maximum of the lane's row; one_by_one: where its keys have to be added so.  read() where the stage has
        // been read.
        auto scores = [&](const char* kt, int k0, float (&sc)[S::NS], int& one_by_one, auto read) {
            const P at = places();
            char* vt = mine + L::V;
            const char* exps = kt + 2 * L::CODES;
            uint32_t ek[KH];
            typename S::acc_t acc[KH];
            uint32_t most = at.put_v(kt + L::CODES, exps + 128, vt, lane < 32);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < KH; ++u) {
                ek[u] = at.k_exps(exps, u);
                uint32_t w[KS];
                at.k_words(kt, u, w);
#pragma unroll
                for (int e = 0; e < S::NS / KH; ++e) acc[u][e] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    const uint32_t byte = at.k_byte(ek[u], kk);
                    most = max(most, byte);
                    const bf16x8 x = __builtin_bit_cast(bf16x8, e2m1_bf16(w[kk], P::scale_of(byte)));
                    if constexpr (R == 16) acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qb[kk], acc[u], 0, 0, 0);
                    else acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, qb[kk], acc[u], 0, 0, 0);
                }
            }
#pragma unroll
            for (int e = 0; e < S::NS; ++e) sc[e] = acc[e / (S::NS / KH)][e % (S::NS / KH)];
            if (__builtin_expect(__ballot(most == kNanGroup) != 0, 0)) {
                at.put_nan(exps + 128, vt);
                uint32_t bad = 0;  // by key
#pragma unroll
                for (int u = 0; u < KH; ++u) bad |= (static_cast<uint32_t>(__ballot(P::k_nan(ek[u]))) & (R == 16 ? 0xffffu : ~0u)) << (16 * u);
                bad >>= 4 * (fresh(lane) / R);
#pragma unroll
                for (int e = 0; e < S::NS; ++e) sc[e] = bad & (1u << S::key(e, 0)) ? NAN : sc[e];
            }
            wave_lds_fence();
            wait_lds();
            read();
            // every row sees every key of the tile?
            const bool open = k0 + 31 <= first_pos && k0 + 32 <= k_hi && (a.window <= 0 || k0 > last_pos - a.window);
            one_by_one = 0;
            if (!open) {
#pragma unroll
                for (int e = 0; e < S::NS; ++e) sc[e] = static_cast<uint32_t>(k0 + S::key(e, lane) - lo) < span ? sc[e] : -INFINITY;
                uint32_t bits = 0;  // a hidden key and a non-finite v
#pragma unroll
                for (int i = 0; i < 64 * HD / 1024; ++i)
                    bits |= non_finite_bits<bf16>(*reinterpret_cast<const uint4*>(vt + i * 1024 + lane * 16));
                one_by_one = __ballot(bits != 0) != 0 ? 1 : 0;
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < S::NS; ++e) mx = fmaxf(mx, sc[e]);
            mx = fmaxf(mx, -INFINITY);  // a NaN does not stay alone
            return S::across(mx, [](float x, float y) { return fmaxf(x, y); });
        };
        // The weights, and the tile's values into the sums.
        auto add = [&](int k0, float (&sc)[S::NS], bool one_by_one) {
            const char* vt = mine + L::V;
            const float off = st_.offset(a.c, down);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < S::NS; ++e) {
                sc[e] = weight(sc[e], a.c, off);
                sum += sc[e];
            }
            st_.l += sum;
            if (one_by_one) {
                add_seen<HD, R>(st_, sc, vt, lane, [&](int j) { return static_cast<uint32_t>(k0 + j - lo) < span; });
                return;
            }
            if constexpr (R == 16) {
                const P at = places();
                const bf16x8 p = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16x2(sc[0], sc[1]), pack_bf16x2(sc[2], sc[3]), pack_bf16x2(sc[4], sc[5]),
                                                                       pack_bf16x2(sc[6], sc[7])));
#pragma unroll
                for (int ob = 0; ob < S::NO; ++ob)
                    st_.o[ob] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at.v_frag16(vt, ob), p, st_.o[ob], 0, 0, 0);
            } else {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 p = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16x2(sc[8 * s], sc[8 * s + 1]), pack_bf16x2(sc[8 * s + 2], sc[8 * s + 3]),
                                                                           pack_bf16x2(sc[8 * s + 4], sc[8 * s + 5]), pack_bf16x2(sc[8 * s + 6], sc[8 * s + 7])));
#pragma unroll
                    for (int ob = 0; ob < S::NO; ++ob)
                        st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.tr(vt, ob, s), p, st_.o[ob], 0, 0, 0);
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
            // a key's row in the pools, negative without a page; keys past the last as the last
            auto row_at = [&](int key) -> int64_t {
                key = min(key, w1 - 1);
                const int pi = a.kv.page_index(key), page = ids[pi - p0];
                const int64_t row = (static_cast<int64_t>(page) * Hkv + kvh) * ps + (key - pi * ps);
                return page < 0 ? -1 : row;
            };
            auto issue = [&](int t) {
                char* dst = mine + (t & 1) * L::STAGE;
                const int k0 = first + 32 * NW * t, fl = R == 16 ? lane : fresh(lane);
                const P at = places();
                if (HD == 128 && ps % 16 == 0 && k0 + 32 <= w1) {
                    // each half of the tile lies in one page: uniform bases
                    const int pi = a.kv.page_index(k0), pj = a.kv.page_index(k0 + 16);
                    const int page0 = same(ids[pi - p0]), page1 = same(ids[pj - p0]);
                    if (page0 >= 0 && page1 >= 0) {
                        const int64_t row[2] = {(static_cast<int64_t>(page0) * Hkv + kvh) * ps + (k0 - pi * ps),
                                                (static_cast<int64_t>(page1) * Hkv + kvh) * ps + (k0 + 16 - pj * ps)};
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            dma16s(a.kv.kp + row[i] * RB, at.voff, dst + i * 1024);
                            dma16s(a.kv.vp + row[i] * RB, at.voff, dst + L::CODES + i * 1024);
                        }
                        dma_exps<HD>((fl >> 5 ? a.kv.ve : a.kv.ke) + ((fl & 16 ? row[1] : row[0]) + (fl & 15)) * NC, dst + 2 * L::CODES);
                        return;
                    }
                }
                const char* none = reinterpret_cast<const char*>(&kNoPage);
                const int64_t row = row_at(k0 + (fl & 31));
                if constexpr (NC == 1) {  // one copy, K's by half of the lanes
                    dma16(row >= 0 ? (fl < 32 ? a.kv.kp : a.kv.vp) + row * RB : none, dst);
                } else {
#pragma unroll(R == 16 ? 2 : 1)
                    for (int i = 0; i < L::CODES / 1024; ++i) {
                        const int rr = (i * 64 + fl) / NC;
                        const int64_t at_row = row_at(k0 + rr), off = at_row * RB + ((fl % NC ^ P::swz4(rr)) << 4);
                        dma16(at_row >= 0 ? a.kv.kp + off : none, dst + i * 1024);
                        dma16(at_row >= 0 ? a.kv.vp + off : none, dst + L::CODES + i * 1024);
                    }
                }
                dma_exps<HD>(row >= 0 ? reinterpret_cast<const char*>(fl >> 5 ? a.kv.ve : a.kv.ke) + row * NC : none, dst + 2 * L::CODES);
            };
            wait_vmcnt<0>();  // Q is there: left to the compiler, which does not count the copies, it would be waited for with all of them, at every tile
            if (nt > 0) issue(0);
            if (nt > 1) issue(1);
            float sc[S::NS], mx;
            int one_by_one;
            // The tiles whose row maxima stand, which are nearly all, in a loop of their own: with the rescaling in it the sums would be
            // copied from one set of registers to another for every tile.
            for (int t = 0; t < nt; ++t) {
                int turn;  // one for the whole wave, in a scalar register
                do {
                    if (t + 1 < nt) wait_vmcnt<L::COPIES>();  // tile t has landed; t + 1 may be in flight
                    else wait_vmcnt<0>();
                    mx = scores(mine + (t & 1) * L::STAGE, first + 32 * NW * t, sc, one_by_one, [&] {
                        if (t + 2 < nt) issue(t + 2);
                    });
                    turn = same(one_by_one | (st_.moves(mx, a.c) ? 2 : 0));
                    if (turn) break;
                    add(first + 32 * NW * t, sc, false);
                    wave_lds_fence();
                } while (++t < nt);
                if (!turn) break;
                st_.absorb(mx, a.c);
                add(first + 32 * NW * t, sc, turn & 1);
                wave_lds_fence();
            }
        }
    }

    // The waves' states joined: everyone's factor against the common maximum, then the sums over the waves.
    bool over = false;
    st_.l = S::across(st_.l, [](float x, float y) { return x + y; });
    if (lane < R) mls[wave][lane] = make_float2(st_.m, st_.l);
    __syncthreads();  // also: the tiles have been read
    const int q = lane % R;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, mls[w][q].x);
    const float base = M == -INFINITY ? 0.0f : M;
    const float factor = __builtin_amdgcn_exp2f((st_.m - base) * a.c);
    float* os = reinterpret_cast<float*>(lds);  // [NW][R][HD], 16-byte groups swizzled by row
#pragma unroll
    for (int ob = 0; ob < S::NO; ++ob)
#pragma unroll
        for (int g = 0; g < (R == 16 ? 1 : 4); ++g) {
            const int c4 = S::column(ob, 4 * g, lane) / 4;
            *reinterpret_cast<float4*>(os + (wave * R + q) * HD + ((c4 ^ (q & 7)) << 2)) =
                make_float4(st_.o[ob][4 * g] * factor, st_.o[ob][4 * g + 1] * factor, st_.o[ob][4 * g + 2] * factor,
                            st_.o[ob][4 * g + 3] * factor);
        }
    __syncthreads();
    for (int i = tid; i < R * (HD / 4); i += NW * 64) {
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
            const float4 y = *reinterpret_cast<const float4*>(os + (w * R + qr) * HD + ((c4 ^ (qr & 7)) << 2));
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

template <int HD, int NW, int R, typename A>
__global__ __launch_bounds__(NW * 64, NW == 8 ? 1 : 2) void attn_paged_e2m1_k(FewArgs<A> f) {
    work_on_parts<NW == 4>(f, [&](const Part& pt, float down) { return few4_part<HD, NW, R>(f, pt, down); });
}

template <int HD, int NW, int R, typename A>
void launch(const FewArgs<A>& f, int64_t blocks, hipStream_t s) {
    constexpr int bytes = Lds4<HD, NW, R>::BYTES;
    static std::atomic<bool> allowed[64];  // by device
    int dev = 0;
    AIC_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !allowed[dev].load()) {
        AIC_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_e2m1_k<HD, NW, R, A>),
                                          hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) allowed[dev].store(true);
    }
    attn_paged_e2m1_k<HD, NW, R><<<static_cast<unsigned>(blocks), NW * 64, bytes, s>>>(f);
    AIC_LAUNCH_CHECK("attn_paged");
}

template <int HD, int R, typename A>
void launch(const FewArgs<A>& f, hipStream_t s) {
    const int64_t pairs = (std::is_same_v<A, PickedArgs> ? int64_t{1} : f.a.kv.Hkv) * f.a.B;
    AIC_CHECK(pairs <= INT32_MAX, OutOfRange, "attn_paged: too many sequences in one call");
    // a CU's one block of eight waves, or blocks of four where there are more: 8 sequences of up to 1000 with 8 heads of 128, 13.1 us and 15.3 in
    // fours; 32 of 3000, 26.7 and 34.3; 40 of 1000, 20.9 and 18.3; 64 of 2000, 36.6 and 32.3
    if (f.shares == 0) return pairs <= 256 ? launch<HD, 8, R>(f, pairs, s) : launch<HD, 4, R>(f, pairs, s);
    launch<HD, 4, R>(f, f.shares, s);
    attn_paged_few_join_k<HD><<<dim3(static_cast<unsigned>(pairs), static_cast<unsigned>((f.group + 3) / 4)), 256, 0, s>>>(f);
    AIC_LAUNCH_CHECK("attn_paged join");
}

}  // namespace

template <typename A>
void attn_paged_e2m1_few(const FewArgs<A>& f, int head_dim, hipStream_t s) {
    auto rows = [&](auto hd) {
        constexpr int D = decltype(hd)::value;
        f.group <= 16 ? launch<D, 16>(f, s) : launch<D, 32>(f, s);
    };
    if (head_dim == 32) rows(std::integral_constant<int, 32>{});
    else if (head_dim == 64) rows(std::integral_constant<int, 64>{});
    else rows(std::integral_constant<int, 128>{});
}

template void attn_paged_e2m1_few(const FewArgs<PagedArgs>&, int, hipStream_t);
template void attn_paged_e2m1_few(const FewArgs<PickedArgs>&, int, hipStream_t);

}  // namespace aic::hip
