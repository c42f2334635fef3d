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
// to a neighbouring token).
//
// Three launches: the rows' statistics by parts of kPart logits, a wave each, in one pass over all
// logits (the only work that grows with the batch's bytes; the parts need no barrier); then per
// sequence the decision and the residual's sums by runs of kRun; then the draw inside the one run it falls into.
// Nothing is returned to the host.  (Two launches, the draw by the last block of a sequence, came to the same:
// 33.3 us for 33.6, for the counting is another trip to memory.)
//
// 64 sequences of up to 7 drafts, 32000 fp32 logits: 33.6 us; statistics 19.5 us (75 MB at 3.8 TB/s, and as long for bf16
// logits: 64-bit products, vector units busy about 60% of the time and waves waiting for issue half of theirs),
// residual 11.7 us, draw 4.9 us.  One sequence of 4 drafts: 14.2 us, three chains of latencies of 3.8, 6.9 and 4.4 us.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "kernels.hpp"
#include "wave_dpp.hpp"
#include "../runtime/memory_pool.hpp"

namespace aic::hip {

namespace {

constexpr int kPer = 16;             // logits per lane
constexpr int kPart = kWave * kPer;  // logits of a part: one wave's
constexpr int kStatWaves = 4;        // waves of a block: statistics
constexpr int kWaves = 8;            // decision: rows looked at side by side
// Logits per lane and per wave of the residual: few, for the weights are straight-line code that each launch
// fetches anew (16 per lane: 12.4 us for one sequence, 4 per lane: 7.0 us).
constexpr int kFew = 4;
constexpr int kRun = kWave * kFew;

struct Stat {
    double sum;    // of the weights against max over the part
    float max;
    int32_t best;  // lowest index of the maximum (target rows)
};
// A row's maximum and the sum of its weights.
struct Whole {
    double sum;
    float max;
    int32_t best;
};
struct Decision {
    int64_t row;   // the packed row whose distribution the new token comes from
    int64_t off;   // the token taken out of it (a refused one-hot draft), -1: none
    int n, kept;
    int minus;     // the draft's distribution is taken off
    Whole p, d;
};

struct DraftArgs {
    const void *z, *y;
    int64_t ldz, ldy;
    const int64_t* ids;
    const float *u, *u_next;
    const int64_t *offsets, *lens;
    int B, V, parts, runs;
    int64_t T, max_q;
    double c;  // log2(e) / temperature; 0: greedy
    // logits below the maximum less reach weigh under 2^-1000; maxima under plain_top, 8 reaches, times c are below 2^13
    float reach, plain_top;
    int64_t *tokens, *counts, *new_lens;
    Stat *sz, *sy;       // [T][parts]
    double* left;        // [B][runs]: residual sums
    Decision* decided;   // [B]
    bool vec_z, vec_y;
};

// 2^x for x <= 0, to 1e-12 of the value: x = n + f with |f| <= 1/2 by adding and taking off 1.5 2^52 (whose
// low word then is n), a polynomial of 2^f (Chebyshev interpolation of degree 8 on [-1/2, 1/2], off by at most
// 1.07e-12), and n into the exponent.  x >= -1001.
__device__ __forceinline__ double exp2_poly(double x) {
    const double big = x + 6755399441055744.0, f = x - (big - 6755399441055744.0);
    double p = 1.3255394667825251e-06;
    p = fma(p, f, 1.531008371327383e-05);
    p = fma(p, f, 0.00015403455050654204);
    p = fma(p, f, 0.0013333450549365335);
    p = fma(p, f, 0.009618129160545788);
    p = fma(p, f, 0.055504109412293744);
    p = fma(p, f, 0.24022650695808107);
    p = fma(p, f, 0.6931471805459256);
    p = fma(p, f, 1.0000000000000004);
    return ldexp(p, static_cast<int>(static_cast<uint32_t>(__double_as_longlong(big))));
}
__device__ __forceinline__ double exp2_neg(double x) { return x < -1000.0 ? 0.0 : exp2_poly(fmax(x, -1000.0)); }
// Weight of a logit against its row's maximum.  An infinite maximum shares the mass among the infinities.
__device__ __forceinline__ double weight(float z, float top, double c) {
    if (top == INFINITY) return z == top ? 1.0 : 0.0;
    return z > -INFINITY ? exp2_neg((static_cast<double>(z) - static_cast<double>(top)) * c) : 0.0;
}

// This lane's PER logits of a run that starts at i0: groups of kWave vectors of up to 16 bytes.
// -infinity past the row's end.
template <typename T, int PER> constexpr int vec_width = PER < 16 / static_cast<int>(sizeof(T)) ? PER : 16 / static_cast<int>(sizeof(T));
template <typename T, int PER>
__device__ __forceinline__ void load_logits(const T* row, int i0, int V, bool vec, float (&z)[PER]) {
    constexpr int W = vec_width<T, PER>;
    typedef T vec_t __attribute__((ext_vector_type(W)));
    const int i = i0 + static_cast<int>(threadIdx.x & 63) * W;
    if (vec && i0 + PER * kWave <= V) {  // wave-uniform: the loads go out together
        vec_t x[PER / W];
#pragma unroll
        for (int g = 0; g < PER / W; ++g) x[g] = *reinterpret_cast<const vec_t*>(row + i + g * W * kWave);
#pragma unroll
        for (int j = 0; j < PER; ++j) z[j] = static_cast<float>(x[j / W][j % W]);
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int at = i + j / W * W * kWave + j % W;
            const float x = static_cast<float>(row[min(at, V - 1)]);
            z[j] = at < V ? x : -INFINITY;
        }
    }
}
template <typename T, int PER>
__device__ __forceinline__ int logit_index(int i0, int j) {
    constexpr int W = vec_width<T, PER>;
    return i0 + (j / W) * W * kWave + static_cast<int>(threadIdx.x & 63) * W + j % W;
}
struct Max {
    template <typename X> __device__ __forceinline__ X operator()(X a, X b) const { return a > b ? a : b; }
};
struct Min {
    template <typename X> __device__ __forceinline__ X operator()(X a, X b) const { return a < b ? a : b; }
};
struct Sum {
    template <typename X> __device__ __forceinline__ X operator()(X a, X b) const { return a + b; }
};

template <typename T>
__global__ __launch_bounds__(kStatWaves * kWave) void draft_stats_k(DraftArgs a) {
    const int lane = threadIdx.x & 63, blocks = (a.parts + kStatWaves - 1) / kStatWaves;
    const int part = static_cast<int>(blockIdx.x) % blocks * kStatWaves + static_cast<int>(threadIdx.x >> 6);
    int64_t row = static_cast<int64_t>(blockIdx.x) / blocks;
    if (part >= a.parts) return;
    const bool draft = row >= a.T;
    if (draft) {
        row -= a.T;
        if (a.B <= 256) {  // a sequence's last row judges no draft (more sequences: the search costs more than the row)
            bool end = false;
            for (int b = lane; b < a.B; b += kWave) end |= a.offsets[b + 1] == row + 1;
            if (__any(end)) return;
        }
    }
    const T* src = draft ? static_cast<const T*>(a.y) + row * a.ldy : static_cast<const T*>(a.z) + row * a.ldz;
    float z[kPer];
    load_logits<T, kPer>(src, part * kPart, a.V, draft ? a.vec_y : a.vec_z, z);
    float mx = -INFINITY;  // a NaN does not count
#pragma unroll
    for (int j = 0; j < kPer; ++j) mx = fmaxf(mx, z[j]);
    mx = wave_all(mx, Max{});
    Stat st{0.0, mx, -1};
    if (mx > -INFINITY) {
        if (a.c == 0.0) {
            int best = INT32_MAX;
#pragma unroll
            for (int j = 0; j < kPer; ++j) best = z[j] == mx ? min(best, logit_index<T, kPer>(part * kPart, j)) : best;
            st.best = wave_all(best, Min{});
        } else {
            double sum = 0.0;
            // Clamped at 2^-1000 of the maximum, also NaN.  One product with mx * c rounded beforehand: that rounding, 2^-41
            // for maxima up to 8 reaches, moves all weights of the part by 3e-13 of themselves.  It would be 1e-7 for the largest
            // maxima, and another one in p than in d: those take the exact difference.
            if (fabsf(mx) < a.plain_top) {
                const float low = mx - a.reach;
                const double top = -static_cast<double>(mx) * a.c;
#pragma unroll
                for (int j = 0; j < kPer; ++j) sum += exp2_poly(fma(static_cast<double>(fmaxf(z[j], low)), a.c, top));
            } else {
#pragma unroll 1
                for (int j = 0; j < kPer; ++j) sum += weight(z[j], mx, a.c);
            }
            st.sum = wave_all(sum, Sum{});
        }
    }
    if (lane == 0) (draft ? a.sy : a.sz)[row * a.parts + part] = st;
}

// A row's whole from its parts, by a wave; x: this lane's part, loaded by the caller, if there is one.
__device__ __forceinline__ Whole whole(const Stat* s, Stat x, int parts, double c) {
    const int lane = threadIdx.x & 63;
    float m = x.max;
    for (int i = lane + kWave; i < parts; i += kWave) m = fmaxf(m, s[i].max);
    Whole w{0.0, wave_all(m, Max{}), INT32_MAX};
    if (c == 0.0) {
        int best = x.max == w.max ? x.best : INT32_MAX;
        for (int i = lane + kWave; i < parts; i += kWave)
            if (s[i].max == w.max) best = min(best, s[i].best);
        w.best = wave_all(best, Min{});
    } else if (w.max > -INFINITY) {
        double sum = x.max > -INFINITY ? x.sum * weight(x.max, w.max, c) : 0.0;
        for (int i = lane + kWave; i < parts; i += kWave)
            if (s[i].max > -INFINITY) sum += s[i].sum * weight(s[i].max, w.max, c);
        w.sum = wave_all(sum, Sum{});
    }
    return w;
}
// p of a logit; exp2 of the library: down to the smallest number.
__device__ __forceinline__ double prob(float z, const Whole& w, double c) {
    if (!(z > -INFINITY)) return 0.0;
    const double v = w.max == INFINITY ? (z == w.max ? 1.0 : 0.0) : exp2((static_cast<double>(z) - static_cast<double>(w.max)) * c);
    return v / w.sum;
}

// How many drafts of sequence b are kept, and where its new token comes from.  The block's waves take its rows
// in turn, kWaves at a time, up to the first draft that is refused.  What a row needs is loaded before its
// statistics are joined: the chain of dependent loads is offsets, ids, logits.
template <typename T>
__device__ __forceinline__ Decision decide(const DraftArgs& a, int b) {
    __shared__ Whole ps[kWaves], ds[kWaves];
    __shared__ int bad[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t lo = min(max(a.offsets[b], int64_t{0}), a.T);
    const int64_t hi = min(max(a.offsets[b + 1], lo), a.T);
    Decision d{lo, -1, static_cast<int>(min(hi - lo, a.max_q)), 0, 0, {}, {}};
    for (int i0 = 0; i0 < d.n; i0 += kWaves) {
        const int i = i0 + wave;
        const int64_t t = lo + i;
        if (i < d.n) {
            const bool judges = i + 1 < d.n, two = judges && a.y;  // the last row gives one token more
            const Stat none{0.0, -INFINITY, INT32_MAX};
            const Stat *sz = a.sz + t * a.parts, *sy = a.sy + t * a.parts;
            const Stat xz = lane < a.parts ? sz[lane] : none, xy = two && lane < a.parts ? sy[lane] : none;
            int64_t x = -1;
            float zx = -INFINITY, yx = -INFINITY, u = 0.0f;
            if (judges) {
                x = a.ids[t + 1];
                if (a.c > 0.0) u = a.u[t];
                if (a.c > 0.0 && x >= 0 && x < a.V) {
                    zx = static_cast<float>(static_cast<const T*>(a.z)[t * a.ldz + x]);
                    if (two) yx = static_cast<float>(static_cast<const T*>(a.y)[t * a.ldy + x]);
                }
            }
            const Whole p = whole(sz, xz, a.parts, a.c);
            Whole q{0.0, -INFINITY, -1};
            if (two) q = whole(sy, xy, a.parts, a.c);
            if (lane == 0) {
                int refuse = 1;
                if (judges && a.c == 0.0) refuse = !(p.max > -INFINITY && x == p.best);
                else if (judges) refuse = !(static_cast<double>(u) * (two ? prob(yx, q, a.c) : 1.0) < prob(zx, p, a.c));
                ps[wave] = p;
                ds[wave] = q;
                bad[wave] = refuse;
            }
        } else if (lane == 0) {
            bad[wave] = 0;
        }
        __syncthreads();
        int first = 0;
        while (first < kWaves && !bad[first]) ++first;
        if (first < kWaves) {
            d.kept = i0 + first;
            d.row = lo + d.kept;
            d.p = ps[first];
            d.d = ds[first];
            if (d.kept + 1 < d.n) {
                d.minus = a.y != nullptr;
                if (!a.y) d.off = a.ids[d.row + 1];
            }
            break;
        }
        __syncthreads();
    }
    return d;
}

// This lane's target and draft logits of a run that starts at i0.
template <int PER>
struct Pair {
    float z[PER], y[PER];
};
template <typename T, int PER>
__device__ __forceinline__ Pair<PER> load_pair(const DraftArgs& a, const Decision& d, int i0) {
    Pair<PER> x;
    load_logits<T, PER>(static_cast<const T*>(a.z) + d.row * a.ldz, i0, a.V, a.vec_z, x.z);
    if (d.minus) load_logits<T, PER>(static_cast<const T*>(a.y) + d.row * a.ldy, i0, a.V, a.vec_y, x.y);
    return x;
}
// Their residual weights max(0, p - d), both rounded before they are taken off: where p and d are equal nothing is
// left (an fma would leave p's rounding error).
template <typename T, int PER>
__device__ __forceinline__ void residual(const DraftArgs& a, const Decision& d, int i0, const Pair<PER>& x, double (&r)[PER]) {
#pragma clang fp contract(off)
    const double ip = d.p.max > -INFINITY ? 1.0 / d.p.sum : 0.0, iq = d.minus && d.d.max > -INFINITY ? 1.0 / d.d.sum : 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) r[j] = weight(x.z[j], d.p.max, a.c) * ip;
    if (iq > 0.0) {
#pragma unroll
        for (int j = 0; j < PER; ++j) r[j] = fmax(0.0, r[j] - weight(x.y[j], d.d.max, a.c) * iq);
    }
    if (d.off >= 0) {
#pragma unroll
        for (int j = 0; j < PER; ++j) r[j] = logit_index<T, PER>(i0, j) == d.off ? 0.0 : r[j];
    }
}

template <typename T>
__global__ __launch_bounds__(kWaves * kWave) void draft_residual_k(DraftArgs a, int blocks) {
    const int group = static_cast<int>(blockIdx.x) % blocks, b = static_cast<int>(blockIdx.x) / blocks;
    const Decision d = decide<T>(a, b);
    if (group == 0 && threadIdx.x == 0) a.decided[b] = d;
    if (d.n == 0 || a.c == 0.0) return;
    int run = group * kWaves + static_cast<int>(threadIdx.x >> 6);
    if (run >= a.runs) return;
    Pair<kFew> x = load_pair<T, kFew>(a, d, run * kRun);
    while (true) {
        const int next = run + blocks * kWaves;
        Pair<kFew> y = x;
        if (next < a.runs) y = load_pair<T, kFew>(a, d, next * kRun);
        double r[kFew], sum = 0.0;
        residual<T, kFew>(a, d, run * kRun, x, r);
#pragma unroll
        for (int j = 0; j < kFew; ++j) sum += r[j];
        sum = wave_all(sum, Sum{});
        if ((threadIdx.x & 63) == 0) a.left[static_cast<int64_t>(b) * a.runs + run] = sum;
        if (next >= a.runs) return;
        x = y;
        run = next;
    }
}

// One wave per sequence: the run, then the token, whose running sum first passes the target.
template <typename T>
__global__ __launch_bounds__(kWave) void draft_pick_k(DraftArgs a) {
    constexpr int W = vec_width<T, kFew>;
    static_assert(W == kFew, "a lane's logits of a run are neighbours");
    const int b = static_cast<int>(blockIdx.x), lane = threadIdx.x;
    double* left = a.left + static_cast<int64_t>(b) * a.runs;
    Decision d = a.decided[b];
    int64_t token = -1;
    if (d.n > 0 && d.p.max > -INFINITY) {
        if (a.c == 0.0) {
            token = d.p.best;
        } else {
            int run = -1;  // runs of weight zero hold no token
            double below = 0.0, target = 0.0;
            // once; and again where p - d left nothing in 64 bits, which then tell p from d nowhere: from p
#pragma unroll 1
            for (int again = 0; again < 2 && run < 0; ++again) {
                if (again) {
                    d.minus = 0;
                    d.off = -1;
                    for (int i = 0; i < a.runs; ++i) {
                        double r[kFew], sum = 0.0;
                        residual<T, kFew>(a, d, i * kRun, load_pair<T, kFew>(a, d, i * kRun), r);
#pragma unroll
                        for (int j = 0; j < kFew; ++j) sum += r[j];
                        sum = wave_all(sum, Sum{});
                        if (lane == 0) left[i] = sum;
                    }
                    __syncthreads();
                }
                double total = 0.0;
                for (int i = lane; i < a.runs; i += kWave) total += left[i];
                target = wave_all(total, Sum{}) * static_cast<double>(a.u_next[b]);
                double sofar = 0.0;
                for (int i0 = 0; i0 < a.runs; i0 += kWave) {
                    const double w = i0 + lane < a.runs ? left[i0 + lane] : 0.0;
                    const double upto = sofar + wave_running_sum(w);
                    const uint64_t some = __ballot(w > 0.0), past = __ballot(w > 0.0 && upto > target);
                    if (some) {
                        const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
                        run = i0 + l;
                        below = __shfl(upto - w, l, kWave);
                    }
                    if (past) break;
                    sofar = __shfl(upto, kWave - 1, kWave);
                }
            }
            if (run >= 0) {
                double r[kFew], mine = 0.0;
                residual<T, kFew>(a, d, run * kRun, load_pair<T, kFew>(a, d, run * kRun), r);
#pragma unroll
                for (int j = 0; j < kFew; ++j) mine += r[j];
                double at = below + (wave_running_sum(mine) - mine);
                int pick = INT32_MAX, last = -1;
#pragma unroll
                for (int j = 0; j < kFew; ++j) {
                    at += r[j];
                    const int i = logit_index<T, kFew>(run * kRun, j);
                    const bool some = r[j] > 0.0;
                    last = some ? max(last, i) : last;
                    pick = some && at > target ? min(pick, i) : pick;
                }
                pick = wave_all(pick, Min{});
                last = wave_all(last, Max{});
                token = pick != INT32_MAX ? pick : last;  // the sums' last bits: none passed the target
            }
        }
    }
    for (int64_t i = lane; i < a.max_q; i += kWave)
        a.tokens[b * a.max_q + i] = d.n == 0 || i > d.kept ? -1 : i == d.kept ? token : a.ids[d.row - d.kept + i + 1];
    if (lane == 0) {
        a.counts[b] = d.n == 0 ? 0 : d.kept + 1;
        if (a.new_lens) {
            const int64_t all = min(max(a.offsets[b + 1], int64_t{0}), a.T) - min(max(a.offsets[b], int64_t{0}), a.T);
            a.new_lens[b] = a.lens[b] - max(all, int64_t{0}) + (d.n == 0 ? 0 : d.kept + 1);
        }
    }
}

int64_t bytes_for(int64_t B, int64_t T, int64_t V) {
    const int64_t parts = (V + kPart - 1) / kPart;
    return 2 * T * parts * static_cast<int64_t>(sizeof(Stat)) + B * ((V + kRun - 1) / kRun) * 8 + B * static_cast<int64_t>(sizeof(Decision));
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

    const int64_t need = bytes_for(B, T, V), parts = (V + kPart - 1) / kPart, runs = (V + kRun - 1) / kRun;
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
    a.B = static_cast<int>(B), a.V = static_cast<int>(V), a.parts = static_cast<int>(parts), a.runs = static_cast<int>(runs);
    a.T = T, a.max_q = max_q;
    a.c = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(temperature);
    a.reach = 1000.0f * temperature * 0.6931f;  // under 1000 / c: 2^-999.9
    a.plain_top = a.reach < 1e30f ? a.reach * 8.0f : 0.0f;
    a.tokens = tokens, a.counts = counts, a.new_lens = new_lens;
    a.sz = static_cast<Stat*>(workspace);
    a.sy = a.sz + T * parts;
    a.left = reinterpret_cast<double*>(a.sy + T * parts);
    a.decided = reinterpret_cast<Decision*>(a.left + B * runs);
    const int64_t size = static_cast<int64_t>(dtype_size(dt));
    a.vec_z = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld * size % 16 == 0;
    a.vec_y = reinterpret_cast<uintptr_t>(draft) % 16 == 0 && ld_draft * size % 16 == 0;
    const int64_t rows = T * (a.y ? 2 : 1) * ((parts + kStatWaves - 1) / kStatWaves);
    // a block decides anew, so large batches give a sequence fewer blocks with several runs per wave
    const int64_t share = greedy ? 1 : std::min((runs + kWaves - 1) / kWaves, std::max<int64_t>(4, 256 / B)), seqs = B * share;
    AIC_CHECK(rows <= INT32_MAX && seqs <= INT32_MAX, OutOfRange, "verify_drafts: too many rows in one call");
    auto run = [&](auto t) {
        using X = decltype(t);
        if (rows > 0) draft_stats_k<X><<<static_cast<unsigned>(rows), kStatWaves * kWave, 0, s>>>(a);
        draft_residual_k<X><<<static_cast<unsigned>(seqs), kWaves * kWave, 0, s>>>(a, static_cast<int>(share));
        draft_pick_k<X><<<static_cast<unsigned>(B), kWave, 0, s>>>(a);
    };
    if (dt == DType::Float32) run(float{});
    else run(bf16{});
    AIC_LAUNCH_CHECK("verify_drafts");
}

}  // namespace aic::hip
