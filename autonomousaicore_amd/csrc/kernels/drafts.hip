// Verification of drafted tokens: speculative sampling on the target's logits, from given uniforms.
//
// Sequence b brings the packed rows offsets[b] .. offsets[b+1] (n of them): its newest token and n - 1
// drafted ones, in ids.  Row t's target logits z and draft logits y give the distributions
// p = softmax(z / temperature) and d = softmax(y / temperature) of the token after t; the drafted
// x = ids[t + 1] is kept where u[t] d(x) < p(x).  The first one that is not is replaced by a draw from
// max(0, p - d); if all are kept, one more token is drawn from the last row's p.  A draw is the first
// token whose running sum passes u_next[b] times the whole.  So every token is distributed as the
// target's, whatever the draft was.
//
// The running sum's steps are as close as 1e-5 of the whole at a vocabulary of 32000, and p - d
// cancels: sums, p and d are kept in 64 bits (a sum in 32 bits would move one draw in a few hundred
// to a neighbouring token).  exp in 64 bits is reduced to 2^f, |f| <= 1/2, and the Taylor polynomial
// of degree 10 (remainder (ln 2 / 2)^11 / 11! = 2e-13 of the value).
//
// Three launches: the rows' statistics by parts of kPart logits (one pass over all logits: the only
// work that grows with the batch's bytes), then per sequence the decision and the parts' residual
// sums, then the draw inside the one part it falls into.  Nothing is returned to the host.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"
#include "../runtime/memory_pool.hpp"

namespace aic::hip {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;                    // logits per thread
constexpr int kPart = kThreads * kPer;      // logits per block

struct Stat {
    double sum;   // of 2^((z - max) c) over the part
    float max;
    int32_t best;  // lowest index of the maximum, -1 if every logit is -infinity or NaN
};

struct DraftArgs {
    const void *z, *y;
    int64_t ldz, ldy;
    const int64_t* ids;
    const float *u, *u_next;
    const int64_t *offsets, *lens;
    int B, V, parts;
    int64_t T, max_q;
    double c;  // log2(e) / temperature; 0: greedy
    int64_t *tokens, *counts, *new_lens;
    Stat *sz, *sy;     // [T][parts]
    double* left;      // [B][parts]: residual sums
    bool vec_z, vec_y;
};

// 2^x for x <= 0, to 3e-13 of the value.
__device__ __forceinline__ double exp2_neg(double x) {
    x = fmax(x, -1100.0);  // below the smallest number: zero
    const double n = rint(x), f = x - n;
    double p = 7.054911620801123e-9;  // (ln 2)^k / k!, k = 10 .. 0
    p = fma(p, f, 1.0178086009239699e-7);
    p = fma(p, f, 1.3215486790144309e-6);
    p = fma(p, f, 1.5252733804059841e-5);
    p = fma(p, f, 1.5403530393381609e-4);
    p = fma(p, f, 1.3333558146428443e-3);
    p = fma(p, f, 9.6181291076284770e-3);
    p = fma(p, f, 5.5504108664821580e-2);
    p = fma(p, f, 2.4022650695910072e-1);
    p = fma(p, f, 6.9314718055994531e-1);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}
// Weight of a logit against its row's maximum; an infinite maximum shares the mass among the infinities.
__device__ __forceinline__ double weight(float z, float top, double c) {
    if (z == top) return 1.0;
    return exp2_neg((static_cast<double>(z) - static_cast<double>(top)) * c);
}

// kPer logits of a row from i0 on; -infinity past the row's end and in the place of a NaN.
template <typename T>
__device__ __forceinline__ void load_logits(const T* row, int i0, int V, bool vec, float (&z)[kPer]) {
    constexpr int W = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(W)));
#pragma unroll
    for (int j0 = 0; j0 < kPer; j0 += W) {
        // lane-contiguous vectors: element j of group j0 sits at i0 + j0 * kThreads + lane * W
        const int i = i0 + j0 * kThreads + static_cast<int>(threadIdx.x) * W;
        if (vec && i + W <= V) {
            const vec_t x = *reinterpret_cast<const vec_t*>(row + i);
#pragma unroll
            for (int j = 0; j < W; ++j) z[j0 + j] = static_cast<float>(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) z[j0 + j] = i + j < V ? static_cast<float>(row[i + j]) : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) z[j] = z[j] == z[j] ? z[j] : -INFINITY;
}
template <typename T>
__device__ __forceinline__ int logit_index(int i0, int j) {
    constexpr int W = 16 / sizeof(T);
    return i0 + (j / W) * W * kThreads + static_cast<int>(threadIdx.x) * W + j % W;
}

__device__ __forceinline__ double block_sum_d(double v, double* red) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void draft_stats_k(DraftArgs a) {
    __shared__ double red[4];
    __shared__ float redf[16];
    __shared__ int redi[4];
    const int part = static_cast<int>(blockIdx.x) % a.parts;
    int64_t row = static_cast<int64_t>(blockIdx.x) / a.parts;
    const bool draft = row >= a.T;
    if (draft) row -= a.T;
    const T* src = draft ? static_cast<const T*>(a.y) + row * a.ldy : static_cast<const T*>(a.z) + row * a.ldz;
    float z[kPer];
    load_logits(src, part * kPart, a.V, draft ? a.vec_y : a.vec_z, z);
    float mx = z[0];
#pragma unroll
    for (int j = 1; j < kPer; ++j) mx = fmaxf(mx, z[j]);
    mx = block_max(mx, redf);
    Stat st{0.0, mx, -1};
    if (mx > -INFINITY) {
        if (!draft) {
            int best = INT32_MAX;
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (z[j] == mx) best = min(best, logit_index<T>(part * kPart, j));
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, kWave));
            if ((threadIdx.x & 63) == 0) redi[threadIdx.x >> 6] = best;
            __syncthreads();
            st.best = min(min(redi[0], redi[1]), min(redi[2], redi[3]));
        }
        if (a.c > 0.0) {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) sum += weight(z[j], mx, a.c);
            st.sum = block_sum_d(sum, red);
        }
    }
    if (threadIdx.x == 0) (draft ? a.sy : a.sz)[row * a.parts + part] = st;
}

// A row's maximum and sum from its parts.
struct Whole {
    float max;
    double sum;
};
__device__ __forceinline__ Whole whole(const Stat* s, int parts, double c) {
    float m = -INFINITY;
    for (int i = 0; i < parts; ++i) m = fmaxf(m, s[i].max);
    double sum = 0.0;
    for (int i = 0; i < parts; ++i)
        if (s[i].max > -INFINITY) sum += s[i].sum * weight(s[i].max, m, c);
    return {m, sum};
}
template <typename T>
__device__ __forceinline__ double prob(const T* row, int64_t x, int V, const Whole& w, double c) {
    if (x < 0 || x >= V || w.max == -INFINITY) return 0.0;
    const float z = static_cast<float>(row[x]);
    return z == z ? weight(z, w.max, c) / w.sum : 0.0;
}

struct Decision {
    int64_t row;    // the packed row whose distribution the new token comes from
    int64_t off;    // the draft token taken out of it (one-hot drafts), -1: none
    int n, kept;
    bool short_;    // a draft was refused
};
// How many drafts of sequence b are kept.  Every thread of the block asks; drafts go by lanes of a wave.
template <typename T>
__device__ __forceinline__ Decision decide(const DraftArgs& a, int b, int* first_bad) {
    const int64_t lo = min(max(a.offsets[b], int64_t{0}), a.T);
    const int64_t hi = min(max(a.offsets[b + 1], lo), a.T);
    Decision d{lo, -1, static_cast<int>(min(hi - lo, a.max_q)), 0, false};
    if (threadIdx.x == 0) *first_bad = INT32_MAX;
    __syncthreads();
    for (int i0 = 0; i0 + 1 < d.n; i0 += kThreads) {
        const int i = i0 + static_cast<int>(threadIdx.x);
        if (i + 1 < d.n) {
            const int64_t t = lo + i, x = a.ids[t + 1];
            bool keep;
            if (a.c == 0.0) {
                float m = -INFINITY;
                int64_t best = -1;
                for (int s = 0; s < a.parts; ++s)
                    if (a.sz[t * a.parts + s].max > m) {
                        m = a.sz[t * a.parts + s].max;
                        best = a.sz[t * a.parts + s].best;
                    }
                keep = x == best && best >= 0;
            } else {
                const Whole p = whole(a.sz + t * a.parts, a.parts, a.c);
                const double px = prob(static_cast<const T*>(a.z) + t * a.ldz, x, a.V, p, a.c);
                double dx = 1.0;
                if (a.y) dx = prob(static_cast<const T*>(a.y) + t * a.ldy, x, a.V, whole(a.sy + t * a.parts, a.parts, a.c), a.c);
                keep = static_cast<double>(a.u[t]) * dx < px;
            }
            if (!keep) atomicMin(first_bad, i);
        }
    }
    __syncthreads();
    d.kept = min(*first_bad, max(d.n - 1, 0));
    d.short_ = d.kept < d.n - 1;
    d.row = lo + d.kept;
    if (d.short_ && !a.y) d.off = a.ids[d.row + 1];
    return d;
}

// The residual weights max(0, p - d) of this thread's logits of one part.
template <typename T>
__device__ __forceinline__ void residual(const DraftArgs& a, const Decision& d, int part, double (&r)[kPer]) {
    const Stat* sz = a.sz + d.row * a.parts;
    const Whole p = whole(sz, a.parts, a.c);
    float z[kPer];
    load_logits(static_cast<const T*>(a.z) + d.row * a.ldz, part * kPart, a.V, a.vec_z, z);
    const bool some = p.max > -INFINITY;
    const double ip = some ? 1.0 / p.sum : 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) r[j] = some && z[j] > -INFINITY ? weight(z[j], p.max, a.c) * ip : 0.0;
    if (!d.short_) return;
    if (!a.y) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (logit_index<T>(part * kPart, j) == d.off) r[j] = 0.0;
        return;
    }
    const Whole q = whole(a.sy + d.row * a.parts, a.parts, a.c);
    if (!(q.max > -INFINITY)) return;
    load_logits(static_cast<const T*>(a.y) + d.row * a.ldy, part * kPart, a.V, a.vec_y, z);
    const double iq = 1.0 / q.sum;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (z[j] > -INFINITY) r[j] = fmax(0.0, r[j] - weight(z[j], q.max, a.c) * iq);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void draft_residual_k(DraftArgs a) {
    __shared__ double red[4];
    __shared__ int first_bad;
    const int part = static_cast<int>(blockIdx.x) % a.parts, b = static_cast<int>(blockIdx.x) / a.parts;
    const Decision d = decide<T>(a, b, &first_bad);
    if (d.n == 0) return;
    double r[kPer], sum = 0.0;
    residual<T>(a, d, part, r);
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += r[j];
    sum = block_sum_d(sum, red);
    if (threadIdx.x == 0) a.left[static_cast<int64_t>(b) * a.parts + part] = sum;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void draft_pick_k(DraftArgs a) {
    constexpr int W = 16 / sizeof(T);
    __shared__ int first_bad, pick, last;
    __shared__ double wsum[4];
    const int b = static_cast<int>(blockIdx.x);
    const Decision d = decide<T>(a, b, &first_bad);
    int64_t token = -1;
    if (d.n > 0) {
        if (a.c == 0.0) {
            float m = -INFINITY;
            for (int s = 0; s < a.parts; ++s)
                if (a.sz[d.row * a.parts + s].max > m) {
                    m = a.sz[d.row * a.parts + s].max;
                    token = a.sz[d.row * a.parts + s].best;
                }
        } else {
            // the part that the target sum falls into; parts of weight zero hold no token
            const double* left = a.left + static_cast<int64_t>(b) * a.parts;
            double total = 0.0;
            for (int s = 0; s < a.parts; ++s) total += left[s];
            const double target = total * static_cast<double>(a.u_next[b]);
            int part = -1;
            double below = 0.0, run = 0.0;
            for (int s = 0; s < a.parts; ++s) {
                if (left[s] > 0.0) {
                    part = s;
                    below = run;
                    if (run + left[s] > target) break;
                }
                run += left[s];
            }
            if (part >= 0) {
                if (threadIdx.x == 0) pick = INT32_MAX, last = -1;
                double r[kPer];
                residual<T>(a, d, part, r);
                const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
                // index order: groups of W * kThreads logits, W of each thread
#pragma unroll
                for (int g = 0; g < kPer / W; ++g) {
                    double mine = 0.0;
#pragma unroll
                    for (int j = 0; j < W; ++j) mine += r[g * W + j];
                    double upto = mine;
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) {
                        const double x = __shfl_up(upto, o, 64);
                        if (lane >= o) upto += x;
                    }
                    __syncthreads();
                    if (lane == 63) wsum[wave] = upto;
                    __syncthreads();
                    double run2 = below;
                    for (int w = 0; w < wave; ++w) run2 += wsum[w];
                    run2 += upto - mine;
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        run2 += r[g * W + j];
                        const int i = logit_index<T>(part * kPart, g * W + j);
                        if (r[g * W + j] > 0.0) {
                            atomicMax(&last, i);
                            if (run2 > target) atomicMin(&pick, i);
                        }
                    }
                    below += wsum[0] + wsum[1] + wsum[2] + wsum[3];
                }
                __syncthreads();
                token = pick != INT32_MAX ? pick : last;  // the sums' last bits: none passed the target
            }
        }
    }
    for (int64_t i = threadIdx.x; i < a.max_q; i += kThreads)
        a.tokens[b * a.max_q + i] = d.n == 0 || i > d.kept ? -1 : i == d.kept ? token : a.ids[d.row - d.kept + i + 1];
    if (threadIdx.x == 0) {
        a.counts[b] = d.n == 0 ? 0 : d.kept + 1;
        if (a.new_lens) {
            const int64_t all = min(max(a.offsets[b + 1], int64_t{0}), a.T) - min(max(a.offsets[b], int64_t{0}), a.T);
            a.new_lens[b] = a.lens[b] - max(all, int64_t{0}) + (d.n == 0 ? 0 : d.kept + 1);
        }
    }
}

int64_t bytes_for(int64_t B, int64_t T, int64_t V) {
    const int64_t parts = (V + kPart - 1) / kPart;
    return 2 * T * parts * static_cast<int64_t>(sizeof(Stat)) + B * parts * 8;
}

void check_sizes(int64_t B, int64_t T, int64_t V) {
    AIC_CHECK(B >= 0 && T >= 0 && B <= INT32_MAX && T <= INT32_MAX, InvalidArgument,
              "verify_drafts: B and T must be 0 .. 2^31 - 1");
    AIC_CHECK(V >= 1 && V <= (1 << 30), InvalidArgument, "verify_drafts: the vocabulary must be 1 .. 2^30, got ", V);
}

}  // namespace

int64_t verify_drafts_workspace(int64_t B, int64_t T, int64_t V) {
    check_sizes(B, T, V);
    return bytes_for(B, T, V);
}

void verify_drafts(const void* logits, int64_t ld, const void* draft, int64_t ld_draft, const int64_t* ids, const float* u,
                   const float* u_next, const int64_t* offsets, const int64_t* lens, int64_t B, int64_t T, int64_t max_q,
                   int64_t V, float temperature, int64_t* tokens, int64_t* counts, int64_t* new_lens, void* workspace,
                   int64_t workspace_bytes, DType dt, hipStream_t s) {
    check_sizes(B, T, V);
    AIC_CHECK(dt == DType::Float32 || dt == DType::BFloat16, DTypeMismatch, "verify_drafts: logits are float32 or bfloat16");
    AIC_CHECK(ld >= V && (!draft || ld_draft >= V), InvalidArgument, "verify_drafts: leading dimension below the vocabulary");
    AIC_CHECK(max_q >= 1 && max_q <= INT32_MAX, InvalidArgument, "verify_drafts: max_q must be 1 .. 2^31 - 1, got ", max_q);
    AIC_CHECK(std::isfinite(temperature) && temperature >= 0.0f, InvalidArgument,
              "verify_drafts: the temperature must be finite and not negative, got ", temperature);
    AIC_CHECK(workspace_bytes >= 0, InvalidArgument, "verify_drafts: negative workspace size");
    if (B == 0) return;
    AIC_CHECK(offsets && tokens && counts && (!new_lens || lens), InvalidArgument, "verify_drafts: null pointer");
    const bool greedy = temperature <= 0.001f;  // as aic_lm_generate
    AIC_CHECK(T == 0 || (logits && ids && (greedy || (u && u_next))), InvalidArgument, "verify_drafts: null pointer");

    const int64_t need = bytes_for(B, T, V), parts = (V + kPart - 1) / kPart;
    const StreamScratchUse use(s);
    if (workspace) {
        AIC_CHECK(workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, InvalidArgument,
                  "verify_drafts: the workspace must be 16-byte aligned and hold ", need, " bytes, got ", workspace_bytes);
    } else {
        AIC_CHECK(stream_scratch_ready(s), InvalidState, "verify_drafts: a captured call needs a workspace of its own");
        workspace = stream_scratch(static_cast<size_t>(need), s);
    }
    DraftArgs a{};
    a.z = logits, a.y = greedy ? nullptr : draft;
    a.ldz = ld, a.ldy = ld_draft;
    a.ids = ids, a.u = u, a.u_next = u_next, a.offsets = offsets, a.lens = lens;
    a.B = static_cast<int>(B), a.V = static_cast<int>(V), a.parts = static_cast<int>(parts);
    a.T = T, a.max_q = max_q;
    a.c = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temperature);
    a.tokens = tokens, a.counts = counts, a.new_lens = new_lens;
    a.sz = static_cast<Stat*>(workspace);
    a.sy = a.sz + T * parts;
    a.left = reinterpret_cast<double*>(a.sy + T * parts);
    const int64_t size = static_cast<int64_t>(dtype_size(dt));
    a.vec_z = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * size % 16 == 0;
    a.vec_y = reinterpret_cast<uintptr_t>(draft) % 16 == 0 && ld_draft * size % 16 == 0;
    const int64_t rows = T * (a.y ? 2 : 1) * parts, seqs = B * parts;
    AIC_CHECK(rows <= INT32_MAX && seqs <= INT32_MAX, OutOfRange, "verify_drafts: too many rows in one call");
    auto run = [&](auto t) {
        using X = decltype(t);
        if (rows > 0) draft_stats_k<X><<<static_cast<unsigned>(rows), kThreads, 0, s>>>(a);
        if (!greedy) draft_residual_k<X><<<static_cast<unsigned>(seqs), kThreads, 0, s>>>(a);
        draft_pick_k<X><<<static_cast<unsigned>(B), kThreads, 0, s>>>(a);
    };
    if (dt == DType::Float32) run(float{});
    else run(bf16{});
    AIC_LAUNCH_CHECK("verify_drafts");
}

}  // namespace aic::hip
