// What the kernels of attention over the paged cache share (attention_paged*.hip): their arguments, a row's state
// and its output.
#pragma once

#include "attention_tiles.hpp"
#include "paged_kv.hpp"
#include "wave_dpp.hpp"

namespace aic::hip {

struct PagedArgs {
    PageView kv;
    const void* q;
    void* o;
    float* lse;
    int64_t ldq, ldo, T;
    const int64_t *offsets, *lens;
    int B, H, G, window;
    float c;         // scale in log2 units
    int nsplit;      // parts of a tile's keys, a block each
    float2* part_ml;  // [nsplit][T][H]: maximum, sum (-1: only scores of -infinity)
    float* part_o;    // [nsplit][T][H][hd]
    bool vec_q, vec_o;
};
// The same for rows that have pages picked for them: each (row, key/value head) is a sequence of its own, its pages the page table's row.
// A type, not a flag, which would cost the calls without it (one token of 12 heads on 513 keys 0.2 us).
struct PickedArgs : PagedArgs {};

namespace {

// All ones: a NaN in fp32, bf16 and e4m3.  Keys whose page id is out of range are read from here, so
// that exactly the queries that would see them become NaN.
__device__ const uint4 kNoPage = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};

constexpr int64_t kMaxLen = INT32_MAX - 4095;  // positions and a tile past them fit in 32 bits

// Weights are at most 2^8 of the maximum's, and sums of many of them times values near the largest number can leave fp32's
// range where the output does not.  A block that ends with such a sum goes over its keys again with the weights times 2^-40
// (2^31 of them stay below the largest v then) and replaces the elements that had left the range, only those: so small, weights
// cost values below 2^-86 their digits.  down: 0, then kDown.  An infinity or NaN in a v that is seen takes the second pass too.
constexpr float kDown = 40.0f;
__device__ __forceinline__ float weight(float s, float c, float off) { return __builtin_amdgcn_exp2f(fmaf(s, c, off)); }
__device__ __forceinline__ float log_sum(float m, float l, float c) { return (m * c + log2f(l)) * kLn2; }
// Whether some sums have left the range: are not finite, and not by the scores, whose weights' sum l shows theirs.
struct Range {
    float none = 0.0f;  // NaN once one of them is not finite
    __device__ __forceinline__ void look(float o) { none = fmaf(o, 0.0f, none); }
    __device__ __forceinline__ bool left(float l) const { return none != 0.0f && l > 0.0f && l < INFINITY; }
};

// x, with its origin hidden (fresh_uniform: one for the whole wave); and the kernel's only argument, loaded anew.  A second pass made
// of them alone shares nothing with the first that the first one's loops would have to carry in registers (both as one loop:
// 2048 rows behind 6144 tokens 143.6 us for 135.9, 256 rows on 4096 keys 32.6 for 30.3, fp32 1000 rows on 2000 keys 178 for 159).
template <typename T>
__device__ __forceinline__ T fresh(T x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ int fresh_uniform(int x) { return __builtin_amdgcn_readfirstlane(fresh(x)); }
template <typename A>
__device__ __forceinline__ A fresh_argument() {
    static_assert(sizeof(A) % 4 == 0);
    typedef const __attribute__((address_space(4))) uint32_t* words_t;
    struct Words {
        uint32_t w[sizeof(A) / 4];
    } x;
    words_t p = (words_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
#pragma unroll
    for (size_t i = 0; i < sizeof(A) / 4; ++i) x.w[i] = p[i];
    return __builtin_bit_cast(A, x);
}
// A barrier for what is in LDS: stores to memory are not waited for.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// A block's first pass and, where a sum has left the range, its second.  pass(argument, thread, block, down): all of a thread's work,
// true where a sum has left the range, with a barrier before its first true.
template <typename A, typename F>
__device__ __forceinline__ void one_or_two_passes(const A& a, F pass) {
    __shared__ int past;
    if (threadIdx.x == 0) past = 0;
    if (pass(a, static_cast<int>(threadIdx.x), static_cast<int>(blockIdx.x), 0.0f)) past = 1;
    lds_barrier();
    if (__builtin_expect(past, 0))
        pass(fresh_argument<A>(), fresh(static_cast<int>(threadIdx.x)), fresh_uniform(static_cast<int>(blockIdx.x)), kDown);
}

struct Seq {
    int64_t row0;  // first packed row
    int n, len;    // queries, cached keys
};
// A picked row stands behind its pages' positions; length -1: nobody's row, left as it is.  Past the pages: one position
// without a place tells as much as all of them.
__device__ __forceinline__ Seq sequence(const PickedArgs& a, int b) {
    const int64_t len = a.lens[b];
    return {static_cast<uint32_t>(b) / static_cast<uint32_t>(a.kv.Hkv), len >= 0, static_cast<int>(min(max(len, int64_t{0}), a.kv.ld_table * a.kv.ps + 1))};
}
__device__ __forceinline__ Seq sequence(const PagedArgs& a, int b) {
    const int64_t lo = min(max(a.offsets[b], int64_t{0}), a.T), hi = min(max(a.offsets[b + 1], lo), a.T);
    return {lo, static_cast<int>(hi - lo), static_cast<int>(min(max(a.lens[b], int64_t{0}), kMaxLen))};
}

// Key/value heads that a launch's blocks go over beside the sequences; the one of sequence b's blocks numbered h.
__device__ __forceinline__ int grid_heads(const PagedArgs& a) { return a.kv.Hkv; }
__device__ __forceinline__ int grid_heads(const PickedArgs&) { return 1; }
__device__ __forceinline__ int kv_head(const PagedArgs&, int, int h) { return h; }
__device__ __forceinline__ int kv_head(const PickedArgs& a, int b, int) {
    return static_cast<int>(static_cast<uint32_t>(b) % static_cast<uint32_t>(a.kv.Hkv));
}

// The same for a b that is one for the whole wave, in scalar registers.
template <typename A>
__device__ __forceinline__ Seq wave_sequence(const A& a, int b) {
    const Seq x = sequence(a, b);
    const uint64_t r = static_cast<uint64_t>(x.row0);
    const uint32_t r_lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(r)));
    const uint32_t r_hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(r >> 32)));
    return {static_cast<int64_t>(static_cast<uint64_t>(r_hi) << 32 | r_lo), __builtin_amdgcn_readfirstlane(x.n),
            __builtin_amdgcn_readfirstlane(x.len)};
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

template <int R>
__device__ __forceinline__ bool find_tile(const PickedArgs& a, int tile, int& b, int& local) {  // all have as many tiles
    const uint32_t per = static_cast<uint32_t>((a.G + R - 1) / R);
    b = static_cast<int>(static_cast<uint32_t>(tile) / per);
    local = tile - b * static_cast<int>(per);
    return b < a.B;
}

// The keys [k_lo, k_hi) of part `split` of a query tile's, k_lo a multiple of 64: equal parts of whole tiles of 64, by
// the tile's own range, so that the parts of one tile end together.
__device__ __forceinline__ void part_of_keys(int& k_lo, int& k_hi, int split, int nsplit) {
    if (nsplit == 1 || k_hi <= k_lo) return;
    const uint32_t n = static_cast<uint32_t>(k_hi - k_lo + 63) / 64;
    const int lo = k_lo;
    k_lo = lo + 64 * static_cast<int>(n * static_cast<uint32_t>(split) / static_cast<uint32_t>(nsplit));
    if (split + 1 < nsplit) k_hi = lo + 64 * static_cast<int>(n * static_cast<uint32_t>(split + 1) / static_cast<uint32_t>(nsplit));
}

// What lanes have stored to LDS, for other lanes of the wave: LDS works in order, so this is for the compiler alone.
__device__ __forceinline__ void wave_lds_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

// ------------------------------------------------------------------------------- tiles
// [KT][HD] tiles of T in LDS, 16-byte chunks swizzled per row.
template <typename T, int HD>
__device__ __forceinline__ int chunk_at(int row, int ch) {
    if constexpr (sizeof(T) == 2) return row * HD * 2 + ((ch ^ swz<HD>(row)) << 4);
    // a ds_read_b128 phase reads one chunk of 16 consecutive rows: 16 different bank groups
    else return row * HD * 4 + ((ch ^ (HD == 32 ? (row >> 1) & 7 : row & 15)) << 4);
}

// Non-zero where one of 16 bytes' elements is an infinity or NaN; a zero field of (x ^ pattern) borrows into its
// top bit.
template <typename CT> __device__ __forceinline__ uint32_t non_finite_bits(uint4 x);
template <> __device__ __forceinline__ uint32_t non_finite_bits<bf16>(uint4 x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = (w[i] & 0x7f807f80u) ^ 0x7f807f80u;
        bits |= (t - 0x00010001u) & ~t & 0x80008000u;
    }
    return bits;
}
template <> __device__ __forceinline__ uint32_t non_finite_bits<float>(uint4 x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = (w[i] & 0x7f800000u) ^ 0x7f800000u;
        bits |= (t - 1u) & ~t & 0x80000000u;
    }
    return bits;
}
template <> __device__ __forceinline__ uint32_t non_finite_bits<uint8_t>(uint4 x) {  // e4m3: NaN
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = (w[i] & 0x7f7f7f7fu) ^ 0x7f7f7f7fu;
        bits |= (t - 0x01010101u) & ~t & 0x80808080u;
    }
    return bits;
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
    float m, l;
    __device__ __forceinline__ void init() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < OB; ++i) zero(o[i]);
    }
    // A tile's row maximum joins the reference maximum, which moves only by more than 2^8.
    __device__ __forceinline__ void absorb(float mx, float c) {
        mx = facing_op<32>(mx, [](float x, float y) { return fmaxf(x, y); });
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
    // A tile's weights of this half of the wave join the sum.
    __device__ __forceinline__ void add(float sum) { l += facing_op<32>(sum, [](float x, float y) { return x + y; }); }
    // -m in log2 units, less down; a row that has seen only scores of -infinity counts from zero
    __device__ __forceinline__ float offset(float c, float down) const { return m == -INFINITY ? -down : fmaf(-m, c, -down); }
};

// o += sum over the tile's keys of p v, key by key and only where the row sees the key: a hidden key has
// weight zero in the matrix product, and zero times an infinity or NaN in its v is NaN.  For tiles
// that hold both a hidden key and a non-finite v.  p[jb][e] is key 32 jb + 8 (e >> 2) + 4 h + (e & 3);
// v4(key, d) gives v[key][d .. d+3].
template <int HD, int JB, typename V4, typename Seen>
__device__ __forceinline__ void add_seen_rows(f32x16 (&o)[HD / 32], const f32x16 (&p)[JB], V4 v4, Seen seen) {
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
                        const float4 x = v4(key, 32 * ob + 8 * g + 4 * h);
                        const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            o[ob][4 * g + u] = s ? fmaf(w, y[u], o[ob][4 * g + u]) : o[ob][4 * g + u];
                    }
            }
        }
}

// Four neighbouring elements of a row of outputs or parts.  again: those that stand there and are finite stay.
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 x, bool vec, bool again) {
    float y[4] = {x.x, x.y, x.z, x.w};
    if (__builtin_expect(again, 0)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float old = static_cast<float>(p[u]);
            y[u] = fabsf(old) < INFINITY ? old : y[u];
        }
    }
    if (__builtin_expect(!vec, 0)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) st(p, u, y[u]);
    } else if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    } else {
        *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
    }
}

// Output of one query row, the lane's half of the head dimension; or of its part, divided by the part's own sum of weights, so
// that parts join without leaving the range.  True where a sum has left it.  again: with the weights' down.
template <typename T, int HD>
__device__ __forceinline__ bool store_row(const PagedArgs& a, const Rows<HD / 32>& r, int64_t t, int head, bool empty,
                                          int split, bool again) {
    constexpr int OB = HD / 32;
    const int h = (threadIdx.x & 63) >> 5;
    const float inv = empty ? 0.0f : 1.0f / r.l;  // l == 0: only scores of -infinity, 0 / 0 = NaN below
    const int64_t part = (static_cast<int64_t>(split) * a.T + t) * a.H + head;
    if (h == 0 && !again) {
        if (a.nsplit > 1) a.part_ml[part] = make_float2(r.m, empty ? 0.0f : r.l == 0.0f ? -1.0f : r.l);
        else if (a.lse) a.lse[t * a.H + head] = empty ? -INFINITY : log_sum(r.m, r.l, a.c);
    }
    if (empty && a.nsplit > 1) return false;
    T* op = static_cast<T*>(a.o) + t * a.ldo + static_cast<int64_t>(head) * HD;
    Range range;
#pragma unroll
    for (int ob = 0; ob < OB; ++ob)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d0 = ob * 32 + 8 * g + 4 * h;
#pragma unroll
            for (int u = 0; u < 4; ++u) range.look(r.o[ob][4 * g + u]);
            const float4 x = make_float4(r.o[ob][4 * g] * inv, r.o[ob][4 * g + 1] * inv, r.o[ob][4 * g + 2] * inv, r.o[ob][4 * g + 3] * inv);
            if (a.nsplit > 1) store4(a.part_o + part * HD + d0, x, true, again);
            else store4(op + d0, x, a.vec_o, again);
        }
    return range.left(r.l) && !empty;
}

}  // namespace

// f(cache type) of a cache that bf16 or fp32 (T) queries read.
template <typename T, typename F>
void by_cache_type(DType type, F&& f) {
    if (type == DType::UInt8) f(uint8_t{});
    else if (type == DType::UInt4) f(e2m1x2{});
    else f(T{});
}

// Few query rows per key/value head, bf16 queries (attention_paged_few.hip): row groups of `group` rows; with a
// workspace the batch's keys are cut into equal shares, one per resident block.
bool few_rows(int64_t pairs, int64_t max_q, int64_t max_len, int64_t G, int64_t head_dim, DType type);
int64_t few_workspace(int64_t B, int64_t Hkv, int64_t max_q, int64_t max_len, int64_t G, int64_t head_dim, DType type, bool picked);
template <typename A>
void attn_paged_few(const A& a, int64_t max_q, DType type, int head_dim, void* workspace, hipStream_t s);

// Up to 4 query rows per key/value head, fp32 queries (attention_paged_f32_few.hip): tiles of so many rows, 0 for
// more of them; tiles x splits x key/value heads blocks.
int f32_few_rows(int64_t max_q, int64_t G);
template <typename A>
void attn_paged_f32_few(const A& a, int rows, DType type, int head_dim, unsigned blocks, hipStream_t s);

// Many query rows per key/value head, bf16 queries (attention_paged_tiles.hip): tiles x splits x key/value heads blocks.
void attn_paged_tiles(const PagedArgs& a, DType type, int head_dim, unsigned blocks, hipStream_t s);

}  // namespace aic::hip
