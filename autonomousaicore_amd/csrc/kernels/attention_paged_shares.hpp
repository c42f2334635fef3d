// Attention over the paged cache for few query rows per key/value head: how the keys of a batch are shared among blocks,
// and how what a share has divided is joined (attention_paged_few.hip, attention_paged_e2m1.hip).
#pragma once

#include "attention_paged.hpp"

namespace aic::hip {

template <typename A>
struct FewArgs {
    A a;
    int group;         // query rows of a group, at most 32
    int shares;        // 0: a block per sequence and key/value head, nothing divided
    int least;         // steps of a share at least, of a batch of up to kFewSteps
    int64_t* plan;     // [B + 1], as find_share leaves it
    float2* part_ml;   // [2 shares][group]: a share's first group's, then its last one's
    float* part_o;     // [2 shares][group][hd]
};

namespace {

constexpr int kIds = 512;    // page ids in LDS at a time
constexpr int kStep = 128;   // keys: a tile for each wave
constexpr int kLeast = 4;    // steps of a share at least: a part costs a block about as much as three steps
constexpr int kFewSteps = 256;  // a batch that leaves most CUs without a block even so
// A sequence's place in the list of steps.
struct Steps {
    Seq sq;
    int lo, steps, groups;  // first key (a multiple of kStep), steps over its keys, row groups
};
template <typename A>
__device__ __forceinline__ Steps steps_of(const FewArgs<A>& f, const Seq& sq) {
    Steps x;
    x.sq = sq;
    const int first = max(x.sq.len - x.sq.n, 0);
    x.lo = f.a.window > 0 ? max(0, first - f.a.window + 1) & ~(kStep - 1) : 0;
    x.steps = max(1, (x.sq.len - x.lo + kStep - 1) / kStep);  // also of a sequence without keys: its rows are zeros
    x.groups = (x.sq.n * f.a.G + f.group - 1) / f.group;
    return x;
}
// Steps of a share, of `total` in at most `cuts`.
template <typename A>
__device__ __forceinline__ int64_t share_of(const FewArgs<A>& f, double total, int cuts) {
    return max(static_cast<int64_t>(total <= kFewSteps ? f.least : kLeast), static_cast<int64_t>((total + cuts - 1) / cuts));
}
// Parts of a group of `steps` steps that is cut by itself.
__device__ __forceinline__ int parts_of(int steps, int64_t share) {
    return share >= steps ? 1 : (steps + static_cast<int>(share) - 1) / static_cast<int>(share);
}
// Whole numbers below 2^53, added over the block's threads: what comes before each, and all of them.
__device__ __forceinline__ void block_scan(double mine, double (&sums)[4], double& before, double& total) {
    const int wave = threadIdx.x >> 6;
    const double upto = wave_running_sum(mine);
    if ((threadIdx.x & 63) == 63) sums[wave] = upto;
    __syncthreads();
    before = upto - mine;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        before += w < wave ? sums[w] : 0.0;
        total += sums[w];
    }
}
// The part of block g: its sequence, the steps before it there and its own.  False: nothing is left for it.
// plan: for each sequence the steps (or, where groups are cut by themselves, the blocks) before it; behind
// them a share's steps, negative in the second case.
template <typename A>
__device__ __forceinline__ bool find_share(const FewArgs<A>& f, int g, int& b, Steps& x, int64_t& before, int64_t& count) {
    __shared__ double sums[2][4], pair_sums[4];
    __shared__ int at_b;
    __shared__ Steps at_x;
    __shared__ int64_t at_before;
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    // what is left once the sequence is known
    auto within = [&](bool by_group, int64_t share, int64_t in, double begin, double total) {
        if (by_group) {
            const int part = same(static_cast<int>(in)), n = parts_of(x.steps, share);
            const int gi = same(part / n), i = part - gi * n;
            // floor(steps i / n), in 32 bits also for 2^24 steps in 512 parts
            const uint32_t steps = static_cast<uint32_t>(x.steps), parts = static_cast<uint32_t>(n), each = steps / parts, rest = steps % parts;
            auto upto = [&](uint32_t k) { return same(static_cast<int>(each * k + rest * k / parts)); };
            const int u0 = upto(static_cast<uint32_t>(i)), u1 = upto(static_cast<uint32_t>(i) + 1);
            before = static_cast<int64_t>(gi) * x.steps + u0;
            count = u1 - u0;
        } else {
            before = in;
            count = min(share, static_cast<int64_t>(total - begin));
        }
    };
    if (f.a.B <= 64) {
        // a lane per sequence, every wave for itself
        const int lane = threadIdx.x & 63;
        Steps own{};
        if (lane < f.a.B) own = steps_of(f, sequence(f.a, lane));
        const double groups = lane < f.a.B ? static_cast<double>(own.groups) * grid_heads(f.a) : 0.0;
        auto sum = [](double p, double q) { return p + q; };
        double size = own.steps * groups, total = wave_all(size, sum);
        const double pairs = wave_all(groups, sum);
        const bool by_group = pairs * 4 <= f.shares;
        const int cuts = f.shares - (by_group ? static_cast<int>(pairs) : 0);  // every group ends one part early
        const int64_t share = share_of(f, total, cuts);
        if (by_group) {
            size = lane < f.a.B ? parts_of(own.steps, share) * groups : 0.0;
            total = wave_all(size, sum);
        }
        const double start = wave_running_sum(size) - size, begin = by_group ? g : static_cast<double>(g) * share;
        if (g == 0 && threadIdx.x < f.a.B) f.plan[lane] = static_cast<int64_t>(start);
        if (g == 0 && threadIdx.x == 0) f.plan[f.a.B] = by_group ? -share : share;
        const uint64_t here = __ballot(begin >= start && begin < start + size);
        if (!here) return false;
        b = __builtin_ctzll(here);
        auto at = [&](int v) { return __builtin_amdgcn_readlane(v, b); };
        const uint64_t row0 = static_cast<uint64_t>(own.sq.row0), in = static_cast<uint64_t>(static_cast<int64_t>(begin - start));
        auto at64 = [&](uint64_t v) {
            return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(at(static_cast<int>(v >> 32)))) << 32 |
                                        static_cast<uint32_t>(at(static_cast<int>(v))));
        };
        x.sq = {at64(row0), at(own.sq.n), at(own.sq.len)};
        x.lo = at(own.lo), x.steps = at(own.steps), x.groups = at(own.groups);
        within(by_group, share, at64(in), begin, total);
        return true;
    }
    const int per = (f.a.B + 255) / 256, tid = threadIdx.x;
    const int first = min(tid * per, f.a.B), last = min(first + per, f.a.B);
    Steps own;  // the last of this thread's sequences: its only one in batches of up to 256
    if (first < last) own = steps_of(f, sequence(f.a, first));
    auto load = [&](int i) {
        if (per > 1) own = steps_of(f, sequence(f.a, i));
    };
    auto groups = [&] { return static_cast<double>(own.groups) * grid_heads(f.a); };
    double mine = 0.0, mine_pairs = 0.0, start, pairs_start, total, pairs;
    for (int i = first; i < last; ++i) {
        load(i);
        mine += own.steps * groups();
        mine_pairs += groups();
    }
    block_scan(mine_pairs, pair_sums, pairs_start, pairs);
    block_scan(mine, sums[0], start, total);
    const bool by_group = pairs * 4 <= f.shares;
    const int cuts = f.shares - (by_group ? static_cast<int>(pairs) : 0);  // every group ends one part early
    const int64_t share = share_of(f, total, cuts);
    auto size = [&] { return (by_group ? parts_of(own.steps, share) : own.steps) * groups(); };
    if (by_group) {
        mine = 0.0;
        for (int i = first; i < last; ++i) {
            load(i);
            mine += size();
        }
        block_scan(mine, sums[1], start, total);
    }
    const double begin = by_group ? g : static_cast<double>(g) * share;
    double s = start;
    for (int i = first; i < last; ++i) {
        load(i);
        const double n = size();
        if (g == 0) f.plan[i] = static_cast<int64_t>(s);
        if (begin >= s && begin < s + n) {
            at_b = i;
            at_x = own;
            at_before = static_cast<int64_t>(begin - s);
        }
        s += n;
    }
    if (g == 0 && tid == 0) f.plan[f.a.B] = by_group ? -share : share;
    if (begin >= total) return false;
    __syncthreads();
    b = same(at_b);
    x.sq = {at_x.sq.row0, same(at_x.sq.n), same(at_x.sq.len)};
    x.lo = same(at_x.lo), x.steps = same(at_x.steps), x.groups = same(at_x.groups);
    within(by_group, share, at_before, begin, total);
    return true;
}

// A group's keys, or a block's share of them; one for the whole block.
struct Part {
    Seq sq;
    int b, kvh, r0;  // the group's sequence, key/value head and first row
    int first, end;  // keys
    int slot;        // of its state in the workspace
    int whole;       // all of the group's keys
};

// A block's parts, one after another.  work(part, down): all of a thread's work on one, true where a sum of this thread's has left fp32's
// range; then once more, with the weights' down.  SHARES: whether the launch may have cut the keys into shares.
template <bool SHARES, typename A, typename F>
__device__ __forceinline__ void work_on_parts(const FewArgs<A>& f, F work) {
    const A& a = f.a;
    __shared__ int past;
    const int Hkv = grid_heads(a);
    if (threadIdx.x == 0) past = 0;

    int b;
    Steps x;
    int64_t before, count;
    if (SHARES && f.shares > 0) {
        if (!find_share(f, static_cast<int>(blockIdx.x), b, x, before, count)) return;
    } else {
        b = static_cast<int>(blockIdx.x) / Hkv;
        x = steps_of(f, wave_sequence(f.a, b));
        before = 0;
        count = INT64_MAX;
    }
    for (bool first_part = true; count > 0 && b < a.B;) {
        const Seq sq = x.sq;
        // groups of a sequence: all of them (shares), or those of the block's head
        const int64_t groups = static_cast<int64_t>(x.groups) * (f.shares > 0 ? Hkv : 1);
        if (before >= groups * x.steps) {
            if (f.shares == 0) return;
            before -= groups * x.steps;
            if (++b < a.B) x = steps_of(f, wave_sequence(f.a, b));
            continue;
        }
        // (a 64-bit division takes a microsecond's worth of instructions)
        const int gi = before >> 31 ? static_cast<int>(before / x.steps)
                                    : __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(before) / static_cast<uint32_t>(x.steps)));
        const int u0 = static_cast<int>(before - static_cast<int64_t>(gi) * x.steps);
        const int u1 = static_cast<int>(min(static_cast<int64_t>(x.steps), u0 + min(count, int64_t{1} << 30)));
        const int kvh = kv_head(a, b, f.shares > 0 ? gi % Hkv : static_cast<int>(blockIdx.x) % Hkv), r0 = (f.shares > 0 ? gi / Hkv : gi) * f.group;
        const Part pt{sq, b, kvh, r0, x.lo + u0 * kStep, u1 < x.steps ? x.lo + u1 * kStep : INT32_MAX,
                      2 * static_cast<int>(blockIdx.x) + (first_part ? 0 : 1), u0 == 0 && u1 == x.steps};
        first_part = false;
        before += u1 - u0;
        count -= u1 - u0;

        bool again = false;
        do {
            const bool over = work(pt, again ? kDown : 0.0f);
            if (over && !again) past = 1;
            lds_barrier();  // also: before the next part's tiles
            again = !again && past;
            if (__builtin_expect(again, 0)) {
                lds_barrier();
                if (threadIdx.x == 0) past = 0;
            }
        } while (__builtin_expect(again, 0));
    }
}

// The groups that shares divided: one wave per row adds the parts of its group.
template <int HD, typename A>
__global__ __launch_bounds__(256) void attn_paged_few_join_k(FewArgs<A> f) {
    const A& a = f.a;
    const int Hkv = grid_heads(a), grid_head = static_cast<int>(blockIdx.x) % Hkv, b = static_cast<int>(blockIdx.x) / Hkv;
    const int kvh = kv_head(a, b, grid_head);
    const int lane = threadIdx.x & 63, qr = static_cast<int>(blockIdx.y) * 4 + static_cast<int>(threadIdx.x >> 6);
    if (qr >= f.group) return;
    const int64_t planned = f.plan[a.B], share = planned < 0 ? -planned : planned, base_step = f.plan[b];
    const bool by_group = planned < 0;
    const Steps x = steps_of(f, wave_sequence(f.a, b));
    for (int g = 0; g < x.groups; ++g) {
        const int r = g * f.group + qr;
        if (r >= x.sq.n * a.G) return;
        // the group's first block and its parts; a block's second slot holds a group that begins behind its own begin
        const int64_t group = static_cast<int64_t>(g) * Hkv + grid_head;
        int64_t s0;
        int parts, first_slot = 0;
        if (by_group) {
            parts = parts_of(x.steps, share);
            s0 = base_step + group * parts;
        } else {
            const int64_t from = base_step + group * x.steps;
            s0 = from / share;
            parts = static_cast<int>((from + x.steps - 1) / share - s0) + 1;
            first_slot = from != s0 * share;
        }
        if (parts == 1) continue;  // undivided: written already
        auto at = [&](int i) { return (2 * (s0 + i) + (i == 0 ? first_slot : 0)) * f.group + qr; };
        auto state = [&](int i) { return i < parts ? f.part_ml[at(i)] : make_float2(-INFINITY, 0.0f); };
        const float2 first = state(lane);
        float M = first.y != 0.0f ? first.x : -INFINITY;
        bool any = first.y != 0.0f;
        for (int i = lane + 64; i < parts; i += 64) {
            const float2 ml = state(i);
            any |= ml.y != 0.0f;
            M = ml.y != 0.0f ? fmaxf(M, ml.x) : M;
        }
        any = __any(any);
        M = wave_all(M, [](float p, float q) { return fmaxf(p, q); });
        const float base = M == -INFINITY ? 0.0f : M;
        constexpr int PL = HD >= 64 ? HD / 64 : 1, kAhead = 8;
        // a part's weight, of its row divided by its own sum
        auto weigh = [&](float2 ml) { return ml.y != 0.0f && ml.y != -1.0f ? __builtin_amdgcn_exp2f((ml.x - base) * a.c) * ml.y : 0.0f; };
        float own = weigh(first), o[PL] = {}, l = own;
        for (int i = lane + 64; i < parts; i += 64) l += weigh(state(i));
        l = wave_all(l, [](float p, float q) { return p + q; });
        const float inv = 1.0f / l;
        for (int i0 = 0; i0 < parts; i0 += 64) {
            if (i0 > 0) own = weigh(state(i0 + lane));
            const float w = own * inv;
            uint64_t left = __ballot(own != 0.0f);
            while (left) {  // eight parts' rows at a time
                int j[kAhead];
                float v[kAhead][PL], ws[kAhead];
                bool live[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    live[k] = left != 0;
                    j[k] = live[k] ? __builtin_ctzll(left) : j[k > 0 ? k - 1 : 0];
                    ws[k] = __shfl(w, j[k], 64);
                    left &= left - 1;
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
#pragma unroll
                    for (int u = 0; u < PL; ++u)
                        if (lane * PL < HD) v[k][u] = f.part_o[at(i0 + j[k]) * HD + lane * PL + u];
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
#pragma unroll
                    for (int u = 0; u < PL; ++u) o[u] = live[k] ? fmaf(ws[k], v[k][u], o[u]) : o[u];
            }
        }
        const int64_t t = x.sq.row0 + r / a.G;
        const int head = kvh * a.G + r % a.G;
        bf16* op = static_cast<bf16*>(a.o) + t * a.ldo + static_cast<int64_t>(head) * HD;
#pragma unroll
        for (int u = 0; u < PL; ++u)
            if (lane * PL < HD) st(op, lane * PL + u, any && l == 0.0f ? NAN : o[u]);  // only scores of -infinity: NaN
        if (a.lse && lane == 0) a.lse[t * a.H + head] = any ? log_sum(base, l, a.c) : -INFINITY;
    }
}

}  // namespace

// Single tokens and a few drafted ones on e2m1 caches (attention_paged_e2m1.hip).
template <typename A>
void attn_paged_e2m1_few(const FewArgs<A>& f, int head_dim, hipStream_t s);

}  // namespace aic::hip
