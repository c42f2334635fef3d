// Attention over the paged cache for few query rows per key/value head (single tokens, drafted tokens): bound by
// reading the cache once.
//
// One block: up to 32 query rows of one sequence and key/value head, over one split of its keys.  The
// four waves take tiles of 32 keys in turn, each into LDS of its own, so no barrier stands between a
// tile's arrival and its use, and each wave keeps its own copies in flight; their (m, l, O) are joined
// once at the end.  The page ids of the split are in LDS before the first tile, so a tile's
// addresses cost no memory latency.
//   bf16  two stages per wave, filled by direct global -> LDS copies two tiles ahead (32 KB per wave at
//         head_dim 128: one block and up to 128 KB in flight per CU)
//   e4m3  one stage of bf16: the next tile's codes travel to registers (8 KB per wave at head_dim 128, two
//         blocks per CU) while this one is multiplied, and are converted as they are stored
#include "attention_paged.hpp"

namespace aic::hip {

namespace {

constexpr int kIds = 512;  // page ids in LDS at a time

template <int HD, bool E4>
struct FewLds {
    static constexpr int TILE = 32 * HD * 2;  // bytes of a tile of K or V
    static constexpr int STAGES = E4 ? 1 : 2;
    static constexpr int WAVE = STAGES * 2 * TILE;
    static constexpr int BYTES = 4 * WAVE > 4 * 32 * HD * 4 ? 4 * WAVE : 4 * 32 * HD * 4;  // also the waves' O at the end
};

template <int HD, bool E4>
__global__ __launch_bounds__(256, HD == 128 ? 1 : 2) void attn_paged_few_k(PagedArgs a) {
    using L = FewLds<HD, E4>;
    constexpr int KS = HD / 16, OB = HD / 32;
    constexpr int SEG = HD / 16, RPS = 512 / HD, NC = HD / 8;  // bf16: 1 KB copies of a tile, rows of one, chunks of a row
    constexpr int UPR = HD / 16, NU = 32 * UPR / 64;           // e4m3: units of a row, units of a tile per lane
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int ids[kIds];
    __shared__ float2 mls[4][32];

    const int Hkv = a.kv.Hkv, ps = a.kv.ps;
    const int kvh = static_cast<int>(blockIdx.x) % Hkv, rest = static_cast<int>(blockIdx.x) / Hkv;
    const int b = rest % a.B, split = rest / a.B;
    const Seq sq = sequence(a, b);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hl = lane >> 5;
    char* mine = lds + wave * L::WAVE;
    const int32_t* tr = a.kv.table + b * a.kv.ld_table;
    const int rows = sq.n * a.G;
    Frags<HD> F;
    F.init();

    for (int r0 = 0; r0 < rows; r0 += 32) {
        const int r = r0 + (lane & 31);
        const bool real = r < rows;
        const int tok = real ? r / a.G : 0, head = kvh * a.G + (real ? r % a.G : 0);
        const int hi = real ? sq.len - sq.n + tok : -1;
        const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;
        const int first_pos = sq.len - sq.n + r0 / a.G, last_pos = sq.len - sq.n + (min(r0 + 32, rows) - 1) / a.G;
        int k_lo = a.window > 0 ? max(0, max(first_pos, 0) - a.window + 1) : 0, k_hi = last_pos + 1;
        if (a.chunk > 0) {
            k_lo = max(k_lo, split * a.chunk);
            if (split + 1 < a.nsplit) k_hi = min(k_hi, (split + 1) * a.chunk);
        }
        k_lo &= ~31;
        const uint32_t span = static_cast<uint32_t>(max(min(hi, k_hi - 1) - lo + 1, 0));

        Rows<OB> st_;
        st_.init();
        if (k_lo < k_hi) {
            bf16x8 qb[KS];
            const bf16* qp = static_cast<const bf16*>(a.q) + (sq.row0 + tok) * a.ldq + static_cast<int64_t>(head) * HD;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                if (a.vec_q) qb[kk] = __builtin_bit_cast(bf16x8, ldg16(qp + 16 * kk + 8 * hl, real));
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) qb[kk][j] = real ? qp[16 * kk + 8 * hl + j] : f2bf(0.0f);
            }

            // one tile's products, from bf16 K and V tiles in LDS
            auto compute = [&](const char* kt, const char* vt, int k0) {
                f32x16 sc[1];
                zero(sc[0]);
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
                    sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.row(kt, 0, kk), qb[kk], sc[0], 0, 0, 0);
                // every row sees every key of the tile?
                const bool open = k0 + 31 <= first_pos && k0 + 32 <= k_hi && (a.window <= 0 || k0 > last_pos - a.window);
                auto seen = [&](int j) { return static_cast<uint32_t>(k0 + j - lo) < span; };
                bool poison = false;  // a hidden key and a non-finite v
                if (!open) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) sc[0][e] = seen(8 * (e >> 2) + 4 * hl + (e & 3)) ? sc[0][e] : -INFINITY;
#pragma unroll
                    for (int i = 0; i < L::TILE / 1024; ++i)
                        poison |= any_non_finite<bf16>(*reinterpret_cast<const uint4*>(vt + i * 1024 + lane * 16));
                    poison = __any(poison);
                }
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[0][e]);
                st_.absorb(mx, a.c);
                const float off = st_.offset(a.c);
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[0][e] = weight<bf16>(sc[0][e], a.c, off);
                    sum += sc[0][e];
                }
                st_.add(sum);
                if (poison) {
                    add_seen_rows<bf16, HD, 1>(st_.o, sc, vt, seen);
                    return;
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 p = pack_bf16x8(sc[0], 8 * s);
#pragma unroll
                    for (int ob = 0; ob < OB; ++ob)
                        st_.o[ob] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(F.tr(vt, ob, s), p, st_.o[ob], 0, 0, 0);
                }
            };

            const int window_keys = min((kIds - 1) * ps, 1 << 20) & ~31;  // keys whose page ids fit
            for (int w0 = k_lo; w0 < k_hi; w0 += window_keys) {
                const int w1 = min(k_hi, w0 + window_keys), p0 = a.kv.page_index(w0), np = a.kv.page_index(w1 - 1) - p0 + 1;
                __syncthreads();
                for (int i = threadIdx.x; i < np; i += 256) {
                    const int page = p0 + i < a.kv.ld_table ? tr[p0 + i] : -1;
                    ids[i] = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.n_pages) ? page : -1;
                }
                __syncthreads();
                const int first = w0 + 32 * wave, nt = first < w1 ? (w1 - first + 127) / 128 : 0;  // this wave's tiles
                // byte offset of key's row in the pools, negative without a page; keys past the last as the last
                auto row_at = [&](int key) -> int64_t {
                    key = min(key, w1 - 1);
                    const int pi = a.kv.page_index(key), page = ids[pi - p0];
                    const int64_t row = (static_cast<int64_t>(page) * Hkv + kvh) * ps + (key - pi * ps);
                    return page < 0 ? -1 : row;
                };
                if constexpr (!E4) {
                    auto issue = [&](int t) {
                        char* dst = mine + (t & 1) * 2 * L::TILE;
                        const int k0 = first + 128 * t;
                        const char* none = reinterpret_cast<const char*>(&kNoPage);
#pragma unroll
                        for (int i = 0; i < SEG; ++i) {
                            const int rr = i * RPS + lane / NC, ch = (lane % NC) ^ swz<HD>(rr);
                            const int64_t row = row_at(k0 + rr);
                            const int64_t at = row * (HD * 2) + ch * 16;
                            dma16(row >= 0 ? a.kv.kp + at : none, dst + i * 1024);
                            dma16(row >= 0 ? a.kv.vp + at : none, dst + L::TILE + i * 1024);
                        }
                    };
                    if (nt > 0) issue(0);
                    if (nt > 1) issue(1);
                    for (int t = 0; t < nt; ++t) {
                        if (t + 1 < nt) wait_vmcnt<2 * SEG>();  // tile t has landed; t + 1 may be in flight
                        else wait_vmcnt<0>();
                        const char* src = mine + (t & 1) * 2 * L::TILE;
                        compute(src, src + L::TILE, first + 128 * t);
                        wait_lds();  // the tile has been read
                        if (t + 2 < nt) issue(t + 2);
                    }
                } else {
                    uint4 rk[NU], rv[NU];
                    uint32_t xk[NU], xv[NU];
                    auto load = [&](int t) {
                        const char* none = reinterpret_cast<const char*>(&kNoPage);
#pragma unroll
                        for (int i = 0; i < NU; ++i) {
                            const int u = i * 64 + lane;
                            const int64_t row = row_at(first + 128 * t + u / UPR), at = row * HD + (u % UPR) * 16;
                            rk[i] = *reinterpret_cast<const uint4*>(row >= 0 ? a.kv.kp + at : none);
                            rv[i] = *reinterpret_cast<const uint4*>(row >= 0 ? a.kv.vp + at : none);
                            xk[i] = row >= 0 ? a.kv.ke[row] : 127;
                            xv[i] = row >= 0 ? a.kv.ve[row] : 127;
                        }
                    };
                    if (nt > 0) load(0);
                    for (int t = 0; t < nt; ++t) {
#pragma unroll
                        for (int i = 0; i < NU; ++i) {
                            const int u = i * 64 + lane, rr = u / UPR, ch = u % UPR;
                            const float sk = exp_scale(xk[i]), sv = exp_scale(xv[i]);
                            char *kt = mine, *vt = mine + L::TILE;
                            *reinterpret_cast<uint4*>(kt + chunk_at<bf16, HD>(rr, 2 * ch)) = e4m3_bf16(make_uint2(rk[i].x, rk[i].y), sk);
                            *reinterpret_cast<uint4*>(kt + chunk_at<bf16, HD>(rr, 2 * ch + 1)) = e4m3_bf16(make_uint2(rk[i].z, rk[i].w), sk);
                            *reinterpret_cast<uint4*>(vt + chunk_at<bf16, HD>(rr, 2 * ch)) = e4m3_bf16(make_uint2(rv[i].x, rv[i].y), sv);
                            *reinterpret_cast<uint4*>(vt + chunk_at<bf16, HD>(rr, 2 * ch + 1)) = e4m3_bf16(make_uint2(rv[i].z, rv[i].w), sv);
                        }
                        if (t + 1 < nt) load(t + 1);
                        __builtin_amdgcn_wave_barrier();
                        wait_lds();  // the wave's own stores are there
                        compute(mine, mine + L::TILE, first + 128 * t);
                        wait_lds();
                        __builtin_amdgcn_wave_barrier();
                    }
                }
            }
        }

        // The waves' states joined: everyone's factor against the common maximum, then the sums over the waves.
        if (hl == 0) mls[wave][lane] = make_float2(st_.m, st_.l);
        __syncthreads();  // also: the tiles have been read
        const int q = lane & 31;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, mls[w][q].x);
        const float base = M == -INFINITY ? 0.0f : M;
        const float f = __builtin_amdgcn_exp2f((st_.m - base) * a.c);
        float* os = reinterpret_cast<float*>(lds);  // [4][32][HD], 16-byte groups swizzled by row
#pragma unroll
        for (int ob = 0; ob < OB; ++ob)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c4 = (ob * 32 + 8 * g + 4 * hl) / 4;
                *reinterpret_cast<float4*>(os + (wave * 32 + q) * HD + ((c4 ^ (q & 7)) << 2)) =
                    make_float4(st_.o[ob][4 * g] * f, st_.o[ob][4 * g + 1] * f, st_.o[ob][4 * g + 2] * f, st_.o[ob][4 * g + 3] * f);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * (HD / 4); i += 256) {
            const int qr = i / (HD / 4), c4 = i % (HD / 4), rr = r0 + qr;
            if (rr >= rows) break;
            const int tk = rr / a.G, hd_ = kvh * a.G + rr % a.G, h2 = sq.len - sq.n + tk;
            const int l2 = a.window > 0 ? max(0, max(h2, 0) - a.window + 1) : 0;
            const bool empty = h2 < 0 || max(l2, k_lo) > min(h2, k_hi - 1);
            float mm = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) mm = fmaxf(mm, mls[w][qr].x);
            const float bs = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float2 ml = mls[w][qr];
                l = fmaf(__builtin_amdgcn_exp2f((ml.x - bs) * a.c), ml.y, l);
            }
            float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4 y = *reinterpret_cast<const float4*>(os + (w * 32 + qr) * HD + ((c4 ^ (qr & 7)) << 2));
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            const int64_t t = sq.row0 + tk;
            if (a.nsplit > 1) {
                const int64_t at = (static_cast<int64_t>(split) * a.T + t) * a.H + hd_;
                if (c4 == 0) a.part_ml[at] = make_float2(mm, empty ? 0.0f : l == 0.0f ? -1.0f : l);
                if (!empty) *reinterpret_cast<float4*>(a.part_o + at * HD + c4 * 4) = x;
                continue;
            }
            const float inv = empty ? 0.0f : 1.0f / l;
            bf16* op = static_cast<bf16*>(a.o) + t * a.ldo + static_cast<int64_t>(hd_) * HD + c4 * 4;
            if (a.vec_o) {
                *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
            } else {
                op[0] = f2bf(x.x * inv), op[1] = f2bf(x.y * inv), op[2] = f2bf(x.z * inv), op[3] = f2bf(x.w * inv);
            }
            if (a.lse && c4 == 0) a.lse[t * a.H + hd_] = empty ? -INFINITY : log_sum(bs, l, a.c);
        }
        __syncthreads();  // before the next rows' tiles
    }
}

template <int HD, bool E4>
void launch(const PagedArgs& a, hipStream_t s) {
    constexpr int bytes = FewLds<HD, E4>::BYTES;
    static const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_few_k<HD, E4>),
                                                          hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    AIC_HIP_CHECK(allowed);
    const int64_t blocks = static_cast<int64_t>(a.kv.Hkv) * a.B * a.nsplit;
    AIC_CHECK(blocks <= INT32_MAX, OutOfRange, "attn_paged: too many sequences in one call");
    attn_paged_few_k<HD, E4><<<static_cast<unsigned>(blocks), 256, bytes, s>>>(a);
    AIC_LAUNCH_CHECK("attn_paged");
}

}  // namespace

void attn_paged_few(const PagedArgs& a, bool e4m3, int head_dim, hipStream_t s) {
    if (head_dim == 32) e4m3 ? launch<32, true>(a, s) : launch<32, false>(a, s);
    else if (head_dim == 64) e4m3 ? launch<64, true>(a, s) : launch<64, false>(a, s);
    else e4m3 ? launch<128, true>(a, s) : launch<128, false>(a, s);
}

}  // namespace aic::hip
