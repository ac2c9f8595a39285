// Verification of drafted tokens against the target's probabilities
// (include/leafq.h, leafq_verify_drafts).
//
// A request's rows are a tree; row 0 is certain.  With p the distribution that the
// logits of row u give, softmax(logits / T), and q the one that the children of u were
// drawn from, a walk from row 0 takes the first child c, in row order, with
//   accept[c] q(x_c) < p(x_c),   after every child that is not taken  p <- norm(max(p - q, 0)),
// and where no child is left draws from p: then the tokens follow the target's
// distribution whatever the drafts were.  Nothing of p is kept: a pass computes a value's weight
// anew and takes it through the rejections so far, each a difference and a factor, the sum's
// inverse.  (In closed form, max(0, a p0 - b q), a and b grow with every rejection and their
// difference loses what they have: eight rejections that leave a hundredth each took all 53 bits.
// Kept in shared memory, 8 bytes a value, they left one block a SM.)  Where q is one at x_c, p is
// p0 without the rejected tokens, and only their weights are needed.
//
// A cluster of blocks walks one request, each warp on its part of the vocabulary, and
// reads only the rows that the walk comes to.  The decisions are made by every warp for
// itself, from the same numbers in the same order: the warps exchange sums through the
// blocks' shared memory, one barrier of the cluster each.  A comparison of a row's first child
// takes the softmax's sum from 32-bit exponentials: with u = 2^-24, of the exponent 3.25 u times its
// mean under p (at most the logarithm of the vocabulary), of ex2 4 u, 5 u for every rescaling, u for
// every addition, at most 92 u = 2^-17.5 up to 2^17 tokens and 267 u = 2^-15.9 for 2^20 (temperatures
// from 1e-30 on, differences of logits below 3.4e38).  What follows a rejection, and a draw, which has
// a border at each token, compare with a sum over the vocabulary in 64 bits, one more pass over the row.  (All rows' sums in 64 bits, which saves that pass, took 113 us instead of 105 for 200
// requests over 100,003 tokens: some 45 instructions a value against 8.)
//
// Bound: the walk, whose rows and rejections depend on one another.  One chain of 5 rows of
// 32,000: 18 us, in a trace of clocks of some 30 thousand: 4 until the cluster is there, 6.9 the
// first pass over all rows, 4.1 their sums' exchange, 5.3 two rows' children, 8.2 the 64-bit sum
// for the draw, 1.2 the draw.  64 trees of 26 rows with probabilities: 75 us, every rejected child that another follows being a pass over its
// row and q (of 426 MB 39 are read from memory; issue slots 40 % used, the most frequent stalls
// are loads, 3.6 warps an issue, and the cluster's barrier, 3.3).  200 ragged requests over
// 100,003 tokens: 110 us, 1.0 TB/s of the 114 MB that the walks need: latency, of blocks that ask
// for 256 or 512 of a warp's 1,560 values of a row at a time and work on these before they ask again
// (a draw's 45 instructions a value are about 24 us at the issue rate).
#include <algorithm>
#include <cfloat>
#include <climits>

#include "leafq_device.cuh"
#include "leafq_internal.h"

namespace leafq {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMostBlocks = 8, kBlocksPerSm = 4;
// Rows whose sums are taken at once where there are no more: one exchange then does for a
// whole chain of few drafts.
constexpr int kRowsAhead = 8;
constexpr int kEach = kMostBlocks * kWarps / 32;  // warps' sums a lane, when they are added up
constexpr float kLog2e = 1.4426950408889634f;

struct VerifyArgs {
    const float* logits;
    const float* probs;  // null: every draft was certain
    int64_t logits_stride, probs_stride;
    const int32_t* ids;
    const int32_t* parents;
    const int32_t* token_offsets;
    const float* accept;
    const float* sample;
    const float* temperature;
    int32_t* path;
    int32_t* tokens_out;
    int32_t* kept;
    int32_t* next;
    int64_t tokens;
    int vocab, most;
    bool ahead;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}

__device__ __forceinline__ void st_cluster(uint32_t addr, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float2 v) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}

// A row as aligned groups of four values: group k has elements 4 k - off ..; those outside
// the row are `none`.
struct Row {
    const float* begin;
    int off, vocab;
    __device__ __forceinline__ Row(const float* row, int v)
        : begin(row), off(static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 2) & 3), vocab(v) {}
    __device__ __forceinline__ int groups() const { return (off + vocab + 3) / 4; }
    __device__ __forceinline__ int first(int k) const { return 4 * k - off; }
    // Groups k, k + kStep, ..., those before k1, of another row's grouping (shift: its `off`).  All loads are under way at once: the row's two ragged groups come after.
    template <int kStep, int kCount>
    __device__ __forceinline__ void load(float4 (&to)[kCount], int k, int k1, int shift, float none) const {
        const bool whole = shift == off;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int e = 4 * (k + kStep * i) - shift;
            const bool inside = k + kStep * i < k1 && e >= 0 && e + 4 <= vocab;
            to[i] = make_float4(none, none, none, none);
            if (whole) {
                if (inside) to[i] = *reinterpret_cast<const float4*>(begin + e);
            } else if (inside) {
                to[i] = make_float4(begin[e], begin[e + 1], begin[e + 2], begin[e + 3]);
            }
        }
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const int e = 4 * (k + kStep * i) - shift;
            if (k + kStep * i >= k1 || (e >= 0 && e + 4 <= vocab)) continue;
            const auto one = [&](int j) { return j >= 0 && j < vocab ? begin[j] : none; };
            to[i] = make_float4(one(e), one(e + 1), one(e + 2), one(e + 3));
        }
    }
};

// (A NaN counts as -inf.)
__device__ __forceinline__ float number(float x) { return fmaxf(x, -INFINITY); }
__device__ __forceinline__ double chance(float q) { return static_cast<double>(fmaxf(q, 0.0f)); }  // (a NaN: 0)

// 2^(d / 32) for d <= 0, within 2^-48: d = 32 n + j + r, 2^(j / 32) from a table (`powers`, of
// which each lane has its own copy, 32 doubles apart), 2^(r / 32) by its series (|r| <= 1/2: the
// term after the fifth is below 2^-48).  Conversions and comparisons of doubles take four to six
// times a multiplication's time: there is one conversion a value, and what is too small is told
// by the upper word (of a number that is not above zero).
constexpr int kPowers = 32;
__device__ __forceinline__ double exp_of(double d, const double* powers) {
    constexpr double kShift = 6755399441055744.0, u = 0.021660849392498290;  // 1.5 2^52: whole numbers in the low bits; ln 2 / 32
    const double whole = d + kShift;
    const int k = __double2loint(whole);
    const double r = d - (whole - kShift);
    double p = fma(r, u * u * u * u * u / 120.0, u * u * u * u / 24.0);
    p = fma(p, r, u * u * u / 6.0);
    p = fma(p, r, u * u / 2.0);
    p = fma(p, r, u);
    p = fma(p, r, 1.0) * powers[(k & (kPowers - 1)) * 32];
    const bool small = static_cast<uint32_t>(__double2hiint(d)) > 0xc0df4000u;  // below -32000
    return __hiloint2double(small ? 0 : __double2hiint(p) + ((k >> 5) << 20), small ? 0 : __double2loint(p));
}

// max(0, x), of a number.
__device__ __forceinline__ double positive_of(double x) {
    const bool below = __double2hiint(x) < 0;
    return __hiloint2double(below ? 0 : __double2hiint(x), below ? 0 : __double2loint(x));
}

// Weights relative to a row's largest value (not -inf): e^((x - top) / T), in 64 bits.
struct Weigher {
    double top64, cold;
    const double* powers;
    bool endless;  // only values of +inf have any weight
    __device__ __forceinline__ Weigher(float top, double c, const double* p)
        : top64(top == INFINITY ? 0.0 : static_cast<double>(top)), cold(c), powers(p), endless(top == INFINITY) {}
    __device__ __forceinline__ float mapped(float x) const { return !endless ? number(x) : x == INFINITY ? 0.0f : -INFINITY; }
    // Of a value that is mapped.
    __device__ __forceinline__ double operator()(float x) const { return exp_of((static_cast<double>(x) - top64) * cold, powers); }
};

// What the warps of a cluster tell one another: two places in turn, so that one barrier a
// turn is enough.
struct Shared {
    float2 stats[kRowsAhead][kMostBlocks * kWarps];  // {top, sum} of a row's parts: of the first rows, or of the walk's last two in turn
    double told[2][kMostBlocks * kWarps];
    double powers[kPowers][32];          // 2^(j / 32), a copy a lane
    double factor[LEAFQ_KV8_TREE_MOST];  // of the rejections (every warp writes the same)
    int32_t parent[LEAFQ_KV8_TREE_MOST], id[LEAFQ_KV8_TREE_MOST];
};

struct Cluster {
    Shared* shared;
    int rank, blocks, warp, lane, turn;
    __device__ __forceinline__ int voices() const { return blocks * kWarps; }
    __device__ __forceinline__ int voice() const { return rank * kWarps + warp; }
    // Leaves a warp's sum with every block.
    __device__ __forceinline__ void tell(double sum) {
        ++turn;
        if (lane < blocks) st_cluster(mapa_shared(smem_u32(&shared->told[turn & 1][voice()]), lane), sum);
        cluster_sync_all();
    }
    __device__ __forceinline__ const double* heard() const { return shared->told[turn & 1]; }
    __device__ __forceinline__ double heard_sum() const {
        double mine = 0.0;
        for (int i = lane; i < voices(); i += 32) mine += heard()[i];
        return warp_sum(mine);
    }
};

// A thread's share of a row's largest value and of the sum of the weights relative to it; of a
// greedy request, of the first place of the largest.  slope: log2 e / T.
struct Share {
    float top = -INFINITY, part = 0.0f;
    int best = INT_MAX;
    // Values x of the groups k, k + 32, ...
    __device__ __forceinline__ void take(float4 (&x)[4], const Row& row, int k, int k1, bool greedy, float slope) {
        float most = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = make_float4(number(x[i].x), number(x[i].y), number(x[i].z), number(x[i].w));
            most = fmaxf(most, fmaxf(fmaxf(x[i].x, x[i].y), fmaxf(x[i].z, x[i].w)));
        }
        if (greedy) {
            if (most > top || best == INT_MAX) {
#pragma unroll
                for (int i = 3; i >= 0; --i) {
                    const int e = row.first(k + 32 * i);
                    const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int j = 3; j >= 0; --j)
                        if (v[j] == most && k + 32 * i < k1 && e + j >= 0 && e + j < row.vocab) best = e + j;
                }
                top = most;
            }
            return;
        }
        if (most == -INFINITY) return;
        if (most == INFINITY) {  // only those have any weight
            if (top != most) part = 0.0f;
            top = most;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                part += ((x[i].x == most) + (x[i].y == most)) + ((x[i].z == most) + (x[i].w == most));
            return;
        }
        if (most != top) part *= ex2((top - most) * slope);  // (of nothing: zero)
        top = most;
        float sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto w = [&](float v) { return ex2((v - top) * slope); };
            sums[i] = (w(x[i].x) + w(x[i].y)) + (w(x[i].z) + w(x[i].w));
        }
        part += (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    // The warp's {top, sum}; the place's bits in the sum's stead of a greedy request.
    __device__ __forceinline__ float2 join(bool greedy, float slope) const {
        const float most = warp_max_f32(top);
        if (greedy) return make_float2(most, __int_as_float(__reduce_min_sync(~0u, top == most ? best : INT_MAX)));
        return make_float2(most, warp_sum(top == most ? part : part * ex2((top - most) * slope)));
    }
};

// A row's, from its parts'.
struct Stats {
    float top, sum = 0.0f;
    int best = INT_MAX;  // of a greedy request

    __device__ __forceinline__ Stats(const float2* heard, int parts, int lane, bool greedy, float slope) {
        float2 v[kEach];
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            v[i] = lane + 32 * i < parts ? heard[lane + 32 * i] : make_float2(-INFINITY, greedy ? __int_as_float(INT_MAX) : 0.0f);
            top = fmaxf(top, v[i].x);
        }
        top = warp_max_f32(top);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (greedy) {
                if (v[i].x == top) best = min(best, __float_as_int(v[i].y));
            } else if (v[i].x != -INFINITY) {
                sum += v[i].x == top ? v[i].y : v[i].y * ex2((v[i].x - top) * slope);
            }
        }
        if (greedy) best = __reduce_min_sync(~0u, best);
        else sum = warp_sum(sum);
    }
};

// What is left of a row's values after some of its children were rejected.  (Calls, which keep
// the walk's registers and its loop's code few: most rows are only read.)
struct Rest {
    Row row, draft;
    Weigher weigher;
    const Shared* shared;
    int u, n;  // the row, and the rows of the tree

    // Takes a weight through the first `rejections` of the row's children: p but for a factor.
    __device__ __forceinline__ double through(double w, double q, int rejections) const {
        for (int i = 0; i < rejections; ++i) w = positive_of(fma(w, shared->factor[i], -q));
        return w;
    }
    // Eight values' weights, after the rejections.
    __device__ __forceinline__ void eight(double (&w)[8], float4 (&x)[2], const float4 (&q)[2], int rejections) const {
        if (weigher.endless) {
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = make_float4(weigher.mapped(x[i].x), weigher.mapped(x[i].y), weigher.mapped(x[i].z), weigher.mapped(x[i].w));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[4 * i] = weigher(number(x[i].x));
            w[4 * i + 1] = weigher(number(x[i].y));
            w[4 * i + 2] = weigher(number(x[i].z));
            w[4 * i + 3] = weigher(number(x[i].w));
        }
#pragma unroll 1
        for (int r = 0; r < rejections; ++r) {
            const double factor = shared->factor[r];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w[4 * i] = positive_of(fma(w[4 * i], factor, -chance(q[i].x)));
                w[4 * i + 1] = positive_of(fma(w[4 * i + 1], factor, -chance(q[i].y)));
                w[4 * i + 2] = positive_of(fma(w[4 * i + 2], factor, -chance(q[i].z)));
                w[4 * i + 3] = positive_of(fma(w[4 * i + 3], factor, -chance(q[i].w)));
            }
        }
    }
    // Takes the tokens of the row's children behind row `from` out of the values of groups k ..
    // k + 63, of which a lane has two: k + lane and 32 further, or two in a row.
    __device__ __forceinline__ void leave_out(float4 (&x)[2], int k, bool in_a_row, int from) const {
        const int lane = threadIdx.x & 31;
        for (int r = from + 1; r < n; ++r) {
            const int e = shared->id[r] + row.off, group = (e >> 2) - k;
            if (shared->parent[r] != u || shared->id[r] < 0 || group < 0 || group >= 64) continue;
            if (lane != (in_a_row ? group >> 1 : group & 31)) continue;
            const int at = in_a_row ? group & 1 : group >> 5;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (i != at) continue;
                if ((e & 3) == 0) x[i].x = -INFINITY;
                if ((e & 3) == 1) x[i].y = -INFINITY;
                if ((e & 3) == 2) x[i].z = -INFINITY;
                if ((e & 3) == 3) x[i].w = -INFINITY;
            }
        }
    }
    // The sum over the groups [k0, k1), by a warp; the children's tokens behind row `from` are
    // left out (all rows are at or before INT_MAX - 1).
    __device__ __noinline__ double sum(int k0, int k1, int rejections, int from) const {
        const int lane = threadIdx.x & 31;
        if (from < n) {  // most parts have none of them
            bool some = false;
            for (int r = from + 1 + lane; r < n; r += 32) {
                const int group = (shared->id[r] + row.off) >> 2;
                some |= shared->parent[r] == u && shared->id[r] >= 0 && group >= k0 && group < k1;
            }
            if (!__any_sync(~0u, some)) from = INT_MAX;
        }
        double mine = 0.0;
#pragma unroll 1
        for (int k = k0; k < k1; k += 64) {
            float4 x[2], q[2] = {};
            row.load<32>(x, k + lane, k1, row.off, -INFINITY);
            if (rejections > 0) draft.load<32>(q, k + lane, k1, row.off, 0.0f);
            if (from < n) leave_out(x, k, false, from);
            double w[8];
            eight(w, x, q, rejections);
            mine += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        }
        return warp_sum(mine);
    }
    // The first token of [k0, k1) at which the sum, `at` before them, passes `goal`; the last one
    // with any weight where none does.
    __device__ __noinline__ int first_above(int k0, int k1, int rejections, int from, double at, double goal) const {
        const int lane = threadIdx.x & 31;
        int highest = -1;
#pragma unroll 1
        for (int k = k0; k < k1; k += 64) {
            float4 x[2], q[2] = {};
            row.load<1>(x, k + 2 * lane, k1, row.off, -INFINITY);
            if (rejections > 0) draft.load<1>(q, k + 2 * lane, k1, row.off, 0.0f);
            if (from < n) leave_out(x, k, true, from);
            double w[8];
            eight(w, x, q, rejections);
            const double mine = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            double inclusive = mine;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const double other = __shfl_up_sync(~0u, inclusive, d);
                if (lane >= d) inclusive += other;
            }
            double running = at + (inclusive - mine);
            const int e = row.first(k + 2 * lane);
            int hit = INT_MAX, positive = -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                running += w[j];
                if (w[j] > 0.0) {
                    positive = e + j;
                    if (running > goal && hit == INT_MAX) hit = e + j;
                }
            }
            hit = __reduce_min_sync(~0u, hit);
            if (hit != INT_MAX) return hit;
            highest = max(highest, __reduce_max_sync(~0u, positive));
            at += __shfl_sync(~0u, inclusive, 31);
        }
        return highest;
    }
};

__global__ void __launch_bounds__(kThreads, kBlocksPerSm) verify_drafts_kernel(const VerifyArgs g) {
    __shared__ Shared shared;
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const double* powers = &shared.powers[0][lane];
    Cluster cluster{&shared, static_cast<int>(cluster_ctarank()), static_cast<int>(cluster_size()), warp, lane, 0};
    const int s = static_cast<int>(blockIdx.x) >> (__ffs(cluster.blocks) - 1), vocab = g.vocab, voices = cluster.voices();
    const int64_t begin = max64(0, min64(g.token_offsets[s], g.tokens));
    const int n = static_cast<int>(max64(0, min64(min64(g.token_offsets[s + 1], g.tokens) - begin, g.most)));
    for (int t = tid; t < n; t += kThreads) {
        shared.parent[t] = g.parents[begin + t];
        const int id = g.ids[begin + t];
        if ((id < 0 || id >= vocab) && t > 0 && cluster.rank == 0) record_device_error(kSiteDraftRange);
        shared.id[t] = id;
    }
    for (int i = warp; i < kPowers; i += kWarps) shared.powers[i][lane] = exp2(static_cast<double>(i) / kPowers);
    int32_t *path = g.path + (int64_t)s * g.most, *tokens_out = g.tokens_out + (int64_t)s * g.most;
    const bool writer = cluster.rank == 0 && tid == 0;
    if (n == 0 && writer) {
        g.kept[s] = 0;
        g.next[s] = -1;
    }
    const float heat = g.temperature[s];
    const bool greedy = !(heat > 0.0f);
    const float slope = kLog2e / fminf(fmaxf(heat, 1e-30f), FLT_MAX);
    const double cold = kPowers * 1.4426950408889634074 / static_cast<double>(fminf(heat, FLT_MAX));  // for exp_of
    cluster_sync_all();  // the cluster's blocks are there, and the tree

    // A warp's groups of a row.
    const int voices_log2 = __ffs(voices) - 1;  // (blocks are a power of two)
    const auto bound = [&](const Row& row, int voice) { return static_cast<int>((int64_t)row.groups() * voice >> voices_log2); };
    // Warps that share a row, the r-th of `count`.
    const auto parts_of = [&](int r, int count) { return count > 1 ? (voices - r + count - 1) / count : voices; };
    // The sums of `count` rows from u on: the warps share the rows out, a part of one row each,
    // and leave theirs with every block.
    const auto take_rows = [&](int u, int count, int slot) {
        const int r = count > 1 ? cluster.voice() % count : 0, part = count > 1 ? cluster.voice() / count : cluster.voice();
        const Row row(g.logits + (begin + u + r) * g.logits_stride, vocab);
        const int parts = parts_of(r, count), all = row.groups();
        int k = count > 1 ? static_cast<int>((int64_t)all * part / parts) : bound(row, part);
        const int k1 = count > 1 ? static_cast<int>((int64_t)all * (part + 1) / parts) : bound(row, part + 1);
        Share share;
#pragma unroll 1
        for (; k < k1; k += 128) {
            float4 x[4];
            row.load<32>(x, k + lane, k1, row.off, -INFINITY);
            share.take(x, row, k + lane, k1, greedy, slope);
        }
        const float2 own = share.join(greedy, slope);
        if (lane < cluster.blocks) st_cluster(mapa_shared(smem_u32(&shared.stats[slot + r][part]), lane), own);
        cluster_sync_all();
    };
    // Asks for this warp's part of a row, from its first group at or before `from` on.
    const auto prefetch = [&](const float* from) {
        const Row row(from, vocab);
        const int k = bound(row, cluster.voice()), k1 = bound(row, cluster.voice() + 1);
        if (lane == 0 && k1 > k) bulk_prefetch_l2(row.begin + row.first(k), 16 * (k1 - k));
    };
    const bool ahead = g.ahead && n <= kRowsAhead;

    int u = 0, level = 0;
    for (; n > 0; ++level) {
        if (writer) path[level] = u;
        const Row row(g.logits + (begin + u) * g.logits_stride, vocab);
        const Row draft(g.probs ? g.probs + (begin + u) * g.probs_stride : nullptr, vocab);
        const int k0 = bound(row, cluster.voice()), k1 = bound(row, cluster.voice() + 1);

        // The children are looked at 32 rows at a time, a lane each; the first rows' values are
        // asked for ahead of the row's sums.
        bool child;
        float child_x, child_q, child_u;
        const auto ask = [&](int c) {
            child = c < n && shared.parent[c] == u && shared.id[c] >= 0 && shared.id[c] < vocab;
            child_x = child ? row.begin[shared.id[c]] : 0.0f;
            child_q = child && g.probs ? draft.begin[shared.id[c]] : 1.0f;
            child_u = child ? g.accept[begin + c] : 0.0f;
        };
        ask(u + 1 + lane);

        if (!ahead) {
            const uint32_t children = __ballot_sync(~0u, child);
            if (children != 0) prefetch(g.logits + (begin + u + __ffs(children)) * g.logits_stride);
        }
        if (!ahead || level == 0) take_rows(u, ahead ? n : 1, ahead ? 0 : level & 1);
        const int parts = ahead ? parts_of(u, n) : voices;
        const Stats stats(shared.stats[ahead ? u : level & 1], parts, lane, greedy, slope);
        const bool any = stats.top != -INFINITY;  // a row without a number has nothing to draw, and no child is taken
        const Weigher weigher(stats.top, cold, powers);
        const auto weight = [&](float x) { return weigher(weigher.mapped(x)); };

        const Rest rest{row, draft, weigher, &shared, u, n};
        int reset = -1;  // rows up to it do not count as rejected any more
        // What a rejection leaves is summed up only when another child is looked at, or by the
        // draw itself.
        int found = -1, steps = 0;       // factors that are known: the row's own, then of each rejection
        bool pending = false;            // the last rejection's sum is not known yet
        double gone = 0.0, exact = 0.0;  // weight of the rejected tokens; the row's sum in 64 bits (0: not known)
        const auto sum_of = [&](int rejections, int from) {
            cluster.tell(rest.sum(k0, k1, rejections, from));
            return cluster.heard_sum();
        };
        const auto know_exact = [&]() {
            if (exact != 0.0) return;
            if (g.probs) prefetch(draft.begin);
            exact = sum_of(0, INT_MAX);
            if (lane == 0) shared.factor[0] = 1.0 / exact;
            __syncwarp();
            steps = 1;
        };
        for (int first = u + 1; first < n && found < 0 && any; first += 32) {
            if (first != u + 1) ask(first + lane);
            for (uint32_t left = __ballot_sync(~0u, child); left != 0; left &= left - 1) {
                const int at = __ffs(left) - 1, id = shared.id[first + at];
                if (greedy) {
                    if (id != stats.best) continue;
                    found = first + at;
                    break;
                }
                const float cx = __shfl_sync(~0u, child_x, at), cq = __shfl_sync(~0u, child_q, at), cu = __shfl_sync(~0u, child_u, at);
                if (pending) {
                    know_exact();
                    if (g.probs) {
                        const double mass = sum_of(steps, INT_MAX);
                        if (mass > 0.0) {
                            if (lane == 0) shared.factor[steps] = 1.0 / mass;
                            __syncwarp();
                            ++steps;
                        } else {
                            steps = 1;  // nothing left: from the target itself
                        }
                    } else if (!(exact - gone > 0.0)) {
                        gone = 0.0;
                        reset = first + at - 1;
                    }
                    pending = false;
                }
                double own = weight(cx), bar = static_cast<double>(cu);
                if (g.probs) {
                    const double q = chance(cq);
                    // (Bit for bit as in the sums: a sum of one value then gives that value a p of one.)
                    own = steps == 0 ? own / stats.sum : rest.through(own, q, steps - 1) * shared.factor[steps - 1];
                    bar *= q;
                } else {
                    // A token that was rejected already has nothing left.
                    bool again = false;
                    for (int r = max(u, reset) + 1 + lane; r < first + at; r += 32) again |= shared.parent[r] == u && shared.id[r] == id;
                    own = __any_sync(~0u, again) ? 0.0 : own;
                    bar *= (exact == 0.0 ? stats.sum : exact) - gone;
                }
                if (bar < own) {
                    found = first + at;
                    break;
                }
                gone += own;
                pending = true;
            }
        }
        if (found >= 0) {
            if (writer) tokens_out[level] = shared.id[found];
            u = found;
            continue;
        }
        // No child: the draw.
        if (writer) g.kept[s] = level + 1;
        if (!any || greedy) {
            const int drawn = any ? stats.best : -1;
            if (writer) {
                tokens_out[level] = drawn;
                g.next[s] = drawn;
            }
            break;
        }
        // The warps' sums: after the rejections, or without the rejected tokens.
        const bool changed = pending;
        int applied = 0, from = changed && !g.probs ? max(u, reset) : INT_MAX;
        if (g.probs && changed) {
            know_exact();
            applied = steps;
        }
        const double mass = sum_of(applied, from);
        if (changed && !(mass > 0.0)) {  // nothing left: from the target itself
            applied = 0;
            from = INT_MAX;
            sum_of(0, INT_MAX);
        }
        double sums[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) sums[i] = lane * kEach + i < voices ? cluster.heard()[lane * kEach + i] : 0.0;
        // The warp whose part the draw falls into: the last one that begins at or below it.
        double own = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) own += sums[i];
        double upto = own;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const double other = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += other;
        }
        const double total = __shfl_sync(~0u, upto, 31);
        const double goal = static_cast<double>(fminf(fmaxf(g.sample[s], 0.0f), 1.0f - 0x1p-24f)) * total;
        double before = __shfl_up_sync(~0u, upto, 1);
        if (lane == 0) before = 0.0;
        int owner = -1;
        double owner_before = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (before <= goal && sums[i] > 0.0) {
                owner = lane * kEach + i;
                owner_before = before;
            }
            before += sums[i];
        }
        const int part = __reduce_max_sync(~0u, owner);
        const uint32_t has = __ballot_sync(~0u, owner == part);
        const double at = __shfl_sync(~0u, owner_before, __ffs(has) - 1);
        if (part == cluster.voice()) {
            const int drawn = rest.first_above(k0, k1, applied, from, at, goal);
            if (lane == 0) {
                tokens_out[level] = drawn;
                g.next[s] = drawn;
            }
        }
        break;
    }
    if (cluster.rank == 0)
        for (int i = (n > 0 ? level + 1 : 0) + tid; i < g.most; i += kThreads) path[i] = tokens_out[i] = -1;
    cluster_sync_all();  // nobody leaves while others may still write here
}

}  // namespace
}  // namespace leafq

using namespace leafq;

extern "C" int leafq_verify_drafts(void* stream, const float* logits, int64_t logits_stride, int64_t vocab,
                                   const int32_t* ids, const int32_t* parents, const int32_t* token_offsets, int requests,
                                   int64_t tokens, int64_t max_tokens, const float* accept, const float* sample,
                                   const float* temperature, const float* draft_probs, int64_t probs_stride, int32_t* path,
                                   int32_t* tokens_out, int32_t* kept, int32_t* next, uint32_t flags) {
    clear_error();
    const char* what = "leafq_verify_drafts";
    if (vocab <= 0 || requests < 0 || requests > INT_MAX / kMostBlocks || tokens < 0 || tokens > INT_MAX || max_tokens < 0 ||
        (tokens > 1 && (logits_stride < vocab || (draft_probs && probs_stride < vocab)))) {
        set_error("leafq_verify_drafts: invalid sizes, or rows that overlap");
        return LEAFQ_ERR_INVALID;
    }
    if (max_tokens > LEAFQ_KV8_TREE_MOST || vocab > LEAFQ_VERIFY_MOST_VOCAB) {
        set_error("leafq_verify_drafts: a request's tree has at most " + std::to_string(LEAFQ_KV8_TREE_MOST) +
                  " rows, a vocabulary at most " + std::to_string(LEAFQ_VERIFY_MOST_VOCAB) + " tokens");
        return LEAFQ_ERR_UNSUPPORTED;
    }
    if (requests == 0) return LEAFQ_OK;
    if (!token_offsets || !sample || !temperature || !kept || !next || (max_tokens > 0 && (!path || !tokens_out)) ||
        (tokens > 0 && (!logits || !ids || !parents || !accept))) {
        set_error("leafq_verify_drafts: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    // A request's blocks read the inputs while other requests' write.
    const auto rows_span = [&](const float* rows, int64_t stride) { return Span{rows, tokens > 0 && rows ? (tokens - 1) * stride + vocab : 0}; };
    const Span inputs[] = {rows_span(logits, logits_stride), rows_span(draft_probs, probs_stride), {ids, tokens}, {parents, tokens},
                           {token_offsets, int64_t{requests} + 1}, {accept, tokens}, {sample, requests}, {temperature, requests}};
    const Span outputs[] = {{path, requests * max_tokens}, {tokens_out, requests * max_tokens}, {kept, requests}, {next, requests}};
    if (!apart(outputs, inputs)) {
        set_error("leafq_verify_drafts: outputs must not overlap one another or the inputs");
        return LEAFQ_ERR_INVALID;
    }
    // Blocks a request: as many as leave a warp 512 values of a row, which it reads at once.  (A
    // batch's longest walk is what it waits for, so many short ones do not call for fewer.)
    int blocks = kMostBlocks;
    while (blocks > 1 && vocab < (int64_t)blocks * kWarps * 512 * 3 / 4) blocks /= 2;
    const VerifyArgs g{logits, draft_probs, logits_stride, probs_stride, ids, parents, token_offsets, accept, sample, temperature,
                       path, tokens_out, kept, next, tokens, static_cast<int>(vocab), static_cast<int>(max_tokens),
                       requests * blocks <= sm_count()};
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(requests * blocks));
    config.blockDim = dim3(kThreads);
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = blocks;
    attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attributes;
    config.numAttrs = (flags & LEAFQ_FLAG_PDL) != 0 ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&config, verify_drafts_kernel, g), what);
}
