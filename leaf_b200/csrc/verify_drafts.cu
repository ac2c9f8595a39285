// Verification of drafted tokens against the target's probabilities
// (include/leafq.h, leafq_verify_drafts).
//
// A request's rows are a tree; row 0 is certain.  With p the distribution that the
// logits of row u give, softmax(logits / T), and q the one that the children of u were
// drawn from, a walk from row 0 takes the first child c, in row order, with
//   accept[c] q(x_c) < p(x_c),   after every child that is not taken  p <- norm(max(p - q, 0)),
// and where no child is left draws from p: then the tokens follow the target's
// distribution whatever the drafts were.  Nothing of p is kept: a pass computes each value's
// weight anew and takes it through the rejections so far, one subtraction and one factor (the
// sum's inverse) each, until nothing of it is left.  (In closed form, max(0, a p0 - b q), a and b
// grow with every rejection and their difference loses what they have: eight rejections that
// leave a hundredth each took all 53 bits.)  Where q is one at x_c, p is p0 without the rejected
// tokens, and only their weights are needed.
//
// A cluster of blocks walks one request, each block on its part of the vocabulary, and
// reads only the rows that the walk comes to.  The decisions are made by every warp for
// itself, from the same numbers in the same order.  A comparison of one child needs the
// softmax's sum to about 2^-24 (32-bit exponentials, sums of them in 64); the draw compares
// with a sum over the vocabulary, where each of its tokens has a border, and is done in 64 bits.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "leafq_device.cuh"
#include "leafq_internal.h"

namespace leafq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMostBlocks = 8;
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
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
}

__device__ __forceinline__ void st_cluster(uint32_t addr, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
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
    __device__ __forceinline__ float4 at(int e, float none) const {
        if (e >= 0 && e + 4 <= vocab && ((e + off) & 3) == 0) return *reinterpret_cast<const float4*>(begin + e);
        const auto one = [&](int i) { return i >= 0 && i < vocab ? begin[i] : none; };
        return make_float4(one(e), one(e + 1), one(e + 2), one(e + 3));
    }
};

// (A NaN counts as -inf.)
__device__ __forceinline__ float number(float x) { return fmaxf(x, -INFINITY); }

// What the warps of a cluster tell one another: two places in turn, so that one barrier a
// turn is enough.
struct Shared {
    double told[2][kMostBlocks * kWarps][2];
    double factor[LEAFQ_KV8_TREE_MOST];  // of the rejections (every warp writes the same)
    int32_t parent[LEAFQ_KV8_TREE_MOST], id[LEAFQ_KV8_TREE_MOST];
};

struct Cluster {
    Shared* shared;
    int rank, blocks, warp, lane, turn;
    // Leaves a warp's two values with every block.
    __device__ __forceinline__ void tell(double a, double b) {
        ++turn;
        if (lane < blocks) {
            const uint32_t at = mapa_shared(smem_u32(shared->told[turn & 1][rank * kWarps + warp]), lane);
            st_cluster(at, a);
            st_cluster(at + 8, b);
        }
        cluster_sync_all();
    }
    __device__ __forceinline__ const double (*heard() const)[2] { return shared->told[turn & 1]; }
    __device__ __forceinline__ int voices() const { return blocks * kWarps; }
};

__global__ void __launch_bounds__(kThreads) verify_drafts_kernel(const VerifyArgs g) {
    extern __shared__ uint32_t excluded_s[];  // the rejected tokens of the block's part, as bits
    __shared__ Shared shared;
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Cluster cluster{&shared, static_cast<int>(cluster_ctarank()), static_cast<int>(cluster_size()), warp, lane, 0};
    const int s = blockIdx.x / cluster.blocks, vocab = g.vocab;
    const int64_t begin = max64(0, min64(g.token_offsets[s], g.tokens));
    const int n = static_cast<int>(max64(0, min64(min64(g.token_offsets[s + 1], g.tokens) - begin, g.most)));
    for (int t = tid; t < n; t += kThreads) {
        shared.parent[t] = g.parents[begin + t];
        const int id = g.ids[begin + t];
        if ((id < 0 || id >= vocab) && t > 0 && cluster.rank == 0) record_device_error(kSiteDraftRange);
        shared.id[t] = id;
    }
    int32_t *path = g.path + (int64_t)s * g.most, *tokens_out = g.tokens_out + (int64_t)s * g.most;
    const bool writer = cluster.rank == 0 && tid == 0;
    if (n == 0 && writer) {
        g.kept[s] = 0;
        g.next[s] = -1;
    }
    const float heat = g.temperature[s];
    const bool greedy = !(heat > 0.0f);
    const float slope = kLog2e / fminf(fmaxf(heat, 1e-30f), FLT_MAX);
    const double cold = 1.0 / static_cast<double>(fminf(heat, FLT_MAX));
    cluster_sync_all();  // the cluster's blocks are there, and the tree

    int u = 0, level = 0;
    for (; n > 0; ++level) {
        if (writer) path[level] = u;
        const Row row(g.logits + (begin + u) * g.logits_stride, vocab);
        const Row draft(g.probs ? g.probs + (begin + u) * g.probs_stride : nullptr, vocab);
        // This warp's groups of the row.
        const int64_t all = row.groups();
        const int k0 = static_cast<int>(all * (cluster.rank * kWarps + warp) / cluster.voices());
        const int k1 = static_cast<int>(all * (cluster.rank * kWarps + warp + 1) / cluster.voices());

        // The row's largest value, and the sum of the weights relative to it (greedy: where it is).
        float top = -INFINITY;
        double sum = 0.0;
        int best = INT_MAX;
        constexpr int kAhead = 8;
        float part = 0.0f;
        for (int k = k0 + lane; k < k1; k += 32 * kAhead) {
            float4 x[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                x[i] = k + 32 * i < k1 ? row.at(row.first(k + 32 * i), -INFINITY) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                x[i] = make_float4(number(x[i].x), number(x[i].y), number(x[i].z), number(x[i].w));
            }
            float most = top;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) most = fmaxf(most, fmaxf(fmaxf(x[i].x, x[i].y), fmaxf(x[i].z, x[i].w)));
            if (greedy) {
                if (most > top || best == INT_MAX) {
#pragma unroll
                    for (int i = kAhead - 1; i >= 0; --i) {
                        const int e = row.first(k + 32 * i);
                        const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                        for (int j = 3; j >= 0; --j)
                            if (v[j] == most && k + 32 * i < k1 && e + j >= 0 && e + j < vocab) best = e + j;
                    }
                    top = most;
                }
                continue;
            }
            if (most == -INFINITY) continue;
            part = top == -INFINITY ? 0.0f : top == most ? part : part * ex2((top - most) * slope);
            top = most;
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                for (const float v : {x[i].x, x[i].y, x[i].z, x[i].w}) part += v == top ? 1.0f : ex2((v - top) * slope);
        }
        {
            const float most = warp_max_f32(top);
            if (greedy) {
                best = __reduce_min_sync(~0u, top == most ? best : INT_MAX);
                sum = best;
            } else {
                sum = warp_sum(top == -INFINITY ? 0.0 : top == most ? part : static_cast<double>(part) * ex2((top - most) * slope));
            }
            cluster.tell(most, sum);
            const double(*heard)[2] = cluster.heard();
            float all_top = -INFINITY;
            for (int i = lane; i < cluster.voices(); i += 32) all_top = fmaxf(all_top, static_cast<float>(heard[i][0]));
            all_top = warp_max_f32(all_top);
            sum = 0.0;
            best = INT_MAX;
            for (int i = lane; i < cluster.voices(); i += 32) {
                const float their = static_cast<float>(heard[i][0]);
                if (greedy) {
                    if (their == all_top) best = min(best, static_cast<int>(heard[i][1]));
                } else if (their != -INFINITY) {
                    sum += their == all_top ? heard[i][1] : heard[i][1] * ex2((their - all_top) * slope);
                }
            }
            best = __reduce_min_sync(~0u, best);
            sum = warp_sum(sum);
            top = all_top;
        }
        const bool any = top != -INFINITY;  // a row without a number has nothing to draw, and no child is taken

        // A value's weight, in 64 bits.
        const auto weight = [&](float x) {
            x = number(x);
            return x == top ? 1.0 : x == -INFINITY ? 0.0 : exp((static_cast<double>(x) - static_cast<double>(top)) * cold);
        };
        const auto chance = [&](float q) { return static_cast<double>(fmaxf(q, 0.0f)); };  // (a NaN: 0)
        // Sums f(value, draft probability, element) over this warp's groups.
        const auto sum_of = [&](auto&& f) {
            double mine = 0.0;
            for (int k = k0 + lane; k < k1; k += 32) {
                const int e = row.first(k);
                const float4 x = row.at(e, -INFINITY);
                const float4 q = g.probs ? draft.at(e, 0.0f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                mine += f(x.x, q.x, e) + f(x.y, q.y, e + 1) + f(x.z, q.z, e + 2) + f(x.w, q.w, e + 3);
            }
            return warp_sum(mine);
        };
        const auto told_sum = [&]() {
            const double(*heard)[2] = cluster.heard();
            double mine = 0.0;
            for (int i = lane; i < cluster.voices(); i += 32) mine += heard[i][0];
            return warp_sum(mine);
        };

        // The children, a block of 32 rows at a time, each lane with a row.  What a rejection
        // leaves is summed up only when another child is looked at, or by the draw itself.
        int found = -1, reset = -1;            // rows up to `reset` do not count as rejected any more
        bool pending = false;                  // the last rejection's sum is not known yet
        int steps = 0;                         // rejections before it that count
        double gone = 0.0, exact = 0.0;        // weight of the rejected tokens; the row's sum in 64 bits (0: not known)
        // p of a value after the rejections, from its weight.
        const auto through = [&](double w, double q) {
            double p = w / exact;
            for (int i = 0; i < steps && p > 0.0; ++i) p = fmax(0.0, p - q) * shared.factor[i];
            return p;
        };
        const auto know_exact = [&]() {
            if (exact != 0.0) return;
            const double mine = sum_of([&](float v, float, int) { return weight(v); });
            cluster.tell(mine, 0.0);
            exact = told_sum();
        };
        for (int base = u + 1; base < n && found < 0 && any; base += 32) {
            const int c = base + lane;
            const bool child = c < n && shared.parent[c] == u && shared.id[c] >= 0 && shared.id[c] < vocab;
            const float x = child ? row.begin[shared.id[c]] : 0.0f, q = child && g.probs ? draft.begin[shared.id[c]] : 1.0f;
            const float chosen = child ? g.accept[begin + c] : 0.0f;
            for (uint32_t left = __ballot_sync(~0u, child); left != 0; left &= left - 1) {
                const int at = __ffs(left) - 1, id = shared.id[base + at];
                if (greedy) {
                    if (id != best) continue;
                    found = base + at;
                    break;
                }
                const float cx = __shfl_sync(~0u, x, at), cq = __shfl_sync(~0u, q, at), cu = __shfl_sync(~0u, chosen, at);
                double own = weight(cx);
                if (pending) {
                    know_exact();
                    if (g.probs) {
                        const double mine = sum_of([&](float v, float d, int) { return fmax(0.0, through(weight(v), chance(d)) - chance(d)); });
                        cluster.tell(mine, 0.0);
                        const double mass = told_sum();
                        if (lane == 0 && mass > 0.0) shared.factor[steps] = 1.0 / mass;
                        __syncwarp();
                        steps = mass > 0.0 ? steps + 1 : 0;  // nothing left: from the target itself
                    } else if (!(exact - gone > 0.0)) {
                        gone = 0.0;
                        reset = base + at - 1;
                    }
                    pending = false;
                }
                if (g.probs) {
                    own = exact == 0.0 ? own / sum : through(own, chance(cq));
                } else {
                    // A token that was rejected already has nothing left.
                    bool again = false;
                    for (int r = max(u, reset) + 1 + lane; r < base + at; r += 32) again |= shared.parent[r] == u && shared.id[r] == id;
                    own = __any_sync(~0u, again) ? 0.0 : own;
                }
                const double bar = static_cast<double>(cu) * (g.probs ? chance(cq) : (exact == 0.0 ? sum : exact) - gone);
                if (bar < own) {
                    found = base + at;
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
            const int drawn = any ? best : -1;
            if (writer) {
                tokens_out[level] = drawn;
                g.next[s] = drawn;
            }
            break;
        }
        bool holes = !g.probs && gone > 0.0, changed = g.probs && pending;
        if (changed) know_exact();
        const int e0 = max(0, row.first(static_cast<int>(all * (cluster.rank * kWarps) / cluster.voices())));
        if (holes) {
            const int e1 = min(vocab, row.first(static_cast<int>(all * (cluster.rank + 1) * kWarps / cluster.voices())));
            for (int i = tid; i < (e1 - e0 + 31) / 32; i += kThreads) excluded_s[i] = 0;
            __syncthreads();
            for (int r = max(u, reset) + 1 + tid; r < n; r += kThreads)
                if (shared.parent[r] == u && shared.id[r] >= e0 && shared.id[r] < e1)
                    atomicOr(&excluded_s[(shared.id[r] - e0) >> 5], 1u << ((shared.id[r] - e0) & 31));
            __syncthreads();
        }
        const auto mass_of = [&](float v, float d, int e) {
            if (holes && e >= e0 && e < vocab && excluded_s[(e - e0) >> 5] >> ((e - e0) & 31) & 1u) return 0.0;
            const double w = weight(v);
            return changed ? fmax(0.0, through(w, chance(d)) - chance(d)) : w;
        };
        cluster.tell(sum_of(mass_of), 0.0);
        if ((holes || changed) && !(told_sum() > 0.0)) {  // nothing left: from the target itself
            holes = changed = false;
            cluster.tell(sum_of(mass_of), 0.0);
        }
        // The warp whose part the draw falls into: the last one that begins at or below it.
        const double(*heard)[2] = cluster.heard();
        const int each = (cluster.voices() + 31) / 32;
        double own = 0.0;
        for (int i = 0; i < each; ++i)
            if (lane * each + i < cluster.voices()) own += heard[lane * each + i][0];
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
        for (int i = 0; i < each; ++i) {
            const int v = lane * each + i;
            if (v >= cluster.voices()) break;
            if (before <= goal && heard[v][0] > 0.0) {
                owner = v;
                owner_before = before;
            }
            before += heard[v][0];
        }
        const int last = __reduce_max_sync(~0u, owner);
        const uint32_t has = __ballot_sync(~0u, owner == last);
        double at = __shfl_sync(~0u, owner_before, __ffs(has) - 1);
        if (last == cluster.rank * kWarps + warp) {
            int drawn = -1, highest = -1;  // highest: the last token with any weight
            for (int k = k0; k < k1 && drawn < 0; k += 32) {
                const int e = row.first(k + lane);
                double w[4] = {0.0, 0.0, 0.0, 0.0};
                if (k + lane < k1) {
                    const float4 x = row.at(e, -INFINITY), q = g.probs ? draft.at(e, 0.0f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    w[0] = mass_of(x.x, q.x, e);
                    w[1] = mass_of(x.y, q.y, e + 1);
                    w[2] = mass_of(x.z, q.z, e + 2);
                    w[3] = mass_of(x.w, q.w, e + 3);
                }
                double inclusive = w[0] + w[1] + w[2] + w[3];
                const double mine = inclusive;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const double other = __shfl_up_sync(~0u, inclusive, d);
                    if (lane >= d) inclusive += other;
                }
                double running = at + (inclusive - mine);
                int hit = INT_MAX, positive = -1;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    running += w[j];
                    if (w[j] > 0.0) {
                        positive = e + j;
                        if (running > goal && hit == INT_MAX) hit = e + j;
                    }
                }
                hit = __reduce_min_sync(~0u, hit);
                highest = max(highest, __reduce_max_sync(~0u, positive));
                if (hit != INT_MAX) drawn = hit;
                at += __shfl_sync(~0u, inclusive, 31);
            }
            if (drawn < 0) drawn = highest;
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
    if (vocab <= 0 || vocab > LEAFQ_VERIFY_MOST_VOCAB || requests < 0 || requests > INT_MAX / kMostBlocks || tokens < 0 ||
        tokens > INT_MAX || max_tokens < 0 || (tokens > 1 && (logits_stride < vocab || (draft_probs && probs_stride < vocab)))) {
        set_error("leafq_verify_drafts: invalid sizes, or rows that overlap");
        return LEAFQ_ERR_INVALID;
    }
    if (max_tokens > LEAFQ_KV8_TREE_MOST) {
        set_error("leafq_verify_drafts: a request's tree has at most " + std::to_string(LEAFQ_KV8_TREE_MOST) + " rows");
        return LEAFQ_ERR_UNSUPPORTED;
    }
    if (requests == 0) return LEAFQ_OK;
    if (!token_offsets || !sample || !temperature || !kept || !next || (max_tokens > 0 && (!path || !tokens_out)) ||
        (tokens > 0 && (!logits || !ids || !parents || !accept))) {
        set_error("leafq_verify_drafts: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    const VerifyArgs g{logits, draft_probs, logits_stride, probs_stride, ids, parents, token_offsets, accept, sample, temperature,
                       path, tokens_out, kept, next, tokens, static_cast<int>(vocab), static_cast<int>(max_tokens)};
    // As many blocks a request as give every SM one.
    int blocks = kMostBlocks;
    while (blocks > 1 && requests * blocks > sm_count()) blocks /= 2;
    const size_t smem = ((vocab + 8) / blocks + 64) / 32 * 4 + 16;
    const int st = allow_smem(reinterpret_cast<const void*>(verify_drafts_kernel), smem, what);
    if (st) return st;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(requests * blocks));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
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
