// Causal grouped-query attention over the paged INT8 KV cache
// (include/leafq.h, leafq_kv8_attention).
//
// For the query row (request s, new token t, head h) at position
// p = context[s] + t, over keys j < min(p + 1, lengths[s]):
//   x_j = scale * ks * (q . ck_j)      ks, vs: the scales of key j's page
//   out = sum_j exp(x_j - m) vs cv_j / sum_j exp(x_j - m),  m = max x
// in one pass over the keys: when the maximum grows from m to m', the sums so
// far are multiplied by exp(m - m').
#include <algorithm>
#include <type_traits>

#include "kv8_attention.cuh"

namespace leafq {
namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void async_copy4(void* smem_dst, const void* gmem_src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem_dst)), "l"(gmem_src) : "memory");
}
template <int kPending>
__device__ __forceinline__ void wait_async_copies_but() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// ---------------------------------------------------------- split form
// Few query rows, many keys (decode).  A block owns 8 query rows of one kv
// head (rows r = token * group + head-in-group of a request) and a range of the
// keys; its warps take chunks of 32 keys in turn, each warp with its own
// reference, sum and output.
//
// Tensor cores: m16n8k16, fp16 in, fp32 sums.  The codes are exact in fp16.
// An fp32 operand is split into hi + lo, 11 significand bits each, so a
// product loses no more than 2^-22 of it; the eight rows' hi parts are rows
// 0-7 of the 16-row operand and their lo parts rows 8-15, so one MMA does
// both and the two accumulator halves are added in the same thread.
//   S = Q K^T: B is K as stored (a lane's bytes are consecutive elements of
//   one key); the contraction's order over the head is whatever falls out.
//   O = P V: the accumulator layout of S is the operand layout of P; B pairs
//   the bytes of two keys by byte permutes.  A step's columns 2t, 2t+1, 2t+8,
//   2t+9 are keys t, 4+t, 8+t, 12+t, which makes the V reads conflict-free.
// A V scale vs = f 2^e goes half into the exponent, half into the weight:
// u_j = 2^(x_j + e - M) with M a reference near the maximum of x_j + e; O sums
// f u_j cv_j and L sums u_j 2^-e, so O / L is the softmax average over 2^110 of the
// scales' range, and neither half rounds.
//
// The codes are read once, by 16-byte asynchronous copies into a ring per warp,
// laid out so that both fragment reads touch every bank once (with two- and
// four-way conflicts long caches took 115 us instead of 108).  A call's first
// microseconds are round trips, so what does not depend on one another is asked
// for at once: the requests' pages; then a request's lengths and page numbers;
// then its rows and its first chunks (one request 6.0 -> 5.4 us).
//
// Bound: for long caches HBM and the conversions (5 and 7 issue slots per four
// codes of K and V) about alike.  6 requests of 15,000 to 91,000 tokens, 8 heads
// of 128, 468 MB: 104 us (4.5 TB/s); the copies alone take 98 us, the arithmetic
// alone 90 us.  For short ones the round trips: 64 requests of 521 to 765 tokens,
// 4 heads of 64, 21.6 MB, take 13.4 us, of which 6 us pass before the first
// chunk is there, 4 us in the key loop and 1 us in joining the warps; one request
// of 200 tokens takes 5.6 us.  Four warps a block at 64-wide heads took 19.2 us
// instead of 13.5, three blocks of eight warps (80 registers, spilling) 21.8.
//
// kNarrow: blocks of two warps, four or three times as many, for more heads than
// wide blocks: a block that walks several short heads is idle in each one's round
// trips, which the other blocks of the SM then fill.
template <int D, bool kNarrow>
struct Split {
    static constexpr int kWarps = kNarrow ? 2 : D <= 64 ? 8 : 4;
    static constexpr int kBlocksPerSm = (D <= 64 ? 16 : 12) / kWarps;
    static constexpr int kStages = D <= 64 ? 3 : 2;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kBlocks = 148 * kBlocksPerSm;   // key ranges of one row block
    static constexpr int kChunk = 32;                    // keys per warp and turn
    static constexpr int kTile = kChunk * D;             // bytes of K (or V) per chunk
    static constexpr int kStage = 2 * kTile + 32;        // + {ks, vs} of its two 16-key groups
    static constexpr int kRing = kStages * kStage;
    static constexpr int kPart = 8 * (D + 2);            // floats of one partial result: m [8], l [8], O [8][D]
    static constexpr size_t kSmem = (size_t)kWarps * kRing + 8 * D * sizeof(float);
    static_assert(kBlocksPerSm * (kSmem + 1152) <= 228 * 1024, "the blocks share the SM's shared memory");
    static_assert(kRing >= kPart * 4, "a warp's partial result goes through its ring");
    static_assert(kWarps * kRing >= kBlocks * 4, "the requests' pages go through the rings");
    static_assert(kWarps * kRing >= (16 + kThreads * 4 + 8 * D) * 4, "joining goes through the rings");
};

// Values of zero count in L as of a scale with this exponent (2^-63): within 2^126 of
// the others of a cache, and below those that an append gives.
constexpr int kZeroExponent = 127 - 63;

// Layout of a chunk.  K's rows lie in the order of the score tiles' columns:
// row c of eight is key (c >> 1) + 4 (c & 1).  Both functions give where 16-byte
// piece c of row r lies within the row: with them each fragment read (16, 8 or 4
// bytes a lane) touches every bank once.
__device__ __forceinline__ int k_key(int r) { return (r & ~7) + ((r & 7) >> 1) + 4 * (r & 1); }
template <int D>
__device__ __forceinline__ int k_piece(int r, int c) {
    return D == 128 ? c ^ ((r & 1) << 2) : c;
}
template <int D>
__device__ __forceinline__ int v_piece(int r, int c) {
    return D == 128 ? c ^ ((r & 3) << 1) : D == 64 ? c ^ (r & 2) : c;
}

// The last request whose units start at or before u (a search by the warp,
// 32 probes a step).
__device__ __forceinline__ int find_request(const int32_t* page_offsets, int requests, int64_t factor, int64_t u, int lane) {
    int lo = 0, n = requests;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const bool below = lane * step < n && factor * page_offsets[at] <= u;
        const int hit = __popc(__ballot_sync(~0u, below)) - 1;
        lo += hit * step;
        n = min(step, n - hit * step);
    }
    return lo;
}

// The last block of a head to arrive joins its n parts, in their order: part i at
// parts + i stride, the first one `first` floats further.
template <int D, bool kNarrow>
__device__ __forceinline__ void join_parts(uint8_t* smem, const float* parts, int64_t stride, int64_t first, int n, int rows,
                                           int group, int first_row, float* out, int64_t out_stride) {
    using C = Split<D, kNarrow>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const auto other = [&](int i) { return parts + i * stride + (i == 0 ? first : 0); };
    float *top_s = reinterpret_cast<float*>(smem), *total_s = top_s + 8;  // of the rows
    float4* set_s = reinterpret_cast<float4*>(total_s + 8);
    // A part's weight, from its m (one that saw no key counts nothing, but shows an l that is no number).
    const auto weigh = [&](float their, float part_l, float top) {
        return their == -INFINITY ? (part_l == 0.0f ? 0.0f : 1.0f) : ex2(their - top);
    };
    for (int r = warp; r < rows; r += C::kWarps) {
        float top = -INFINITY, total = 0.0f;
        const float m0 = lane < n ? __ldcg(other(lane) + r) : -INFINITY, l0 = lane < n ? __ldcg(other(lane) + 8 + r) : 0.0f;
        for (int i = lane + 32; i < n; i += 32) top = fmaxf(top, __ldcg(other(i) + r));
        top = warp_max_f32(fmaxf(top, m0));
        total = weigh(m0, l0, top) * l0;
        for (int i = lane + 32; i < n; i += 32) {
            const float part_l = __ldcg(other(i) + 8 + r);
            total = fmaf(weigh(__ldcg(other(i) + r), part_l, top), part_l, total);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
        if (lane == 0) {
            top_s[r] = top;
            total_s[r] = total;
        }
    }
    __syncthreads();
    // Four elements and every sets-th part per thread, then the threads' sums.
    constexpr int kAhead = D <= 64 ? 2 : 4;  // (four would have the key loop of 64-wide heads spill)
    const int items = rows * (D / 4), sets = max(1, C::kThreads / items), set = tid / items;
    for (int item = tid % items; item < items && set < sets; item += C::kThreads) {
        const int r = item / (D / 4);
        const float top = top_s[r];
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll kAhead
        for (int i = set; i < n; i += sets) {
            const float weight = weigh(__ldcg(other(i) + r), __ldcg(other(i) + 8 + r), top);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(other(i) + 16) + item);
            sum.x = fmaf(weight, v.x, sum.x);
            sum.y = fmaf(weight, v.y, sum.y);
            sum.z = fmaf(weight, v.z, sum.z);
            sum.w = fmaf(weight, v.w, sum.w);
        }
        set_s[set * items + item] = sum;
    }
    __syncthreads();
    for (int item = tid; item < items; item += C::kThreads) {
        const int r = item / (D / 4), d = 4 * (item - r * (D / 4));
        float4 sum = set_s[item];
        for (int other_set = 1; other_set < sets; ++other_set) {
            const float4 v = set_s[other_set * items + item];
            sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
        }
        const float total = total_s[r];
        const float4 y = total == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                       : make_float4(sum.x / total, sum.y / total, sum.z / total, sum.w / total);
        const int t = (first_row + r) / group, hq = (first_row + r) - t * group;
        *reinterpret_cast<float4*>(out + t * out_stride + hq * D + d) = y;
    }
}

template <int D, bool kNarrow>
__global__ void __launch_bounds__(Split<D, kNarrow>::kThreads, Split<D, kNarrow>::kBlocksPerSm)
kv8_attend_split_kernel(const Kv8AttendArgs g, float* parts, uint32_t* arrivals, int ranges, int row_blocks) {
    using C = Split<D, kNarrow>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int last_s;
    __shared__ struct {  // what the end of a segment needs: kept out of the key loop's registers
        int64_t row0;
        int h, rows, own, parts, first_part;
    } segment_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, tq = lane & 3;
    uint8_t* ring = smem + warp * C::kRing;
    uint4* q_s = reinterpret_cast<uint4*>(smem + C::kWarps * C::kRing);  // the query rows' fragments [D / 16][32]
    __shared__ float factor_s[8];
    grid_dependency_wait();
    grid_launch_dependents();

    // Row blocks of one key range are neighbours, so that they share its codes in L2.
    const int range = blockIdx.x / row_blocks, row_block = blockIdx.x - range * row_blocks;
    const int page = 1 << g.shift;
    const int requests = g.step.requests, kv_heads = g.cache.kv_heads;
    const int64_t units = (int64_t)kv_heads * g.step.page_offsets[requests];
    // Work.  With no more requests' heads than blocks, each head's pages are cut
    // into equal pieces of at most `piece` pages and every block takes one: the
    // smallest piece, from a warp's chunk each on, that makes no more pieces than
    // blocks.  Otherwise the units (page, head, request) in a row are dealt out in
    // even shares of one unit at least, each block walking the heads in its own.  A
    // head over several blocks costs a partial result each, which the last of them
    // joins: it counts every share between the head's ends, so none may be empty.
    const int64_t segments = (int64_t)requests * kv_heads;
    const bool pieces = segments <= ranges;
    int shares = 1;
    int64_t begin = 0, end = 0;
    int s = 0, h = 0, p0 = 0, p1 = 0;             // the segment: pages [p0, p1) of head h of request s
    int first_block = 0, last_block = 0;          // pieces: the blocks of this block's head
    const int32_t* page_offsets = g.step.page_offsets;
    if (pieces) {
        // The pages of each request (at most one per block), in the rings.
        int32_t* held_pages = reinterpret_cast<int32_t*>(smem);
        for (int r = tid; r < requests; r += C::kThreads)
            held_pages[r] = min(max(page_offsets[r + 1] - page_offsets[r], 0), static_cast<int>(g.step.max_pages));
        __syncthreads();
        int piece = 0;
        // About held / piece rounded up, the same in every block; none of no pages, no more than
        // pages.  One of up to `piece` pages, whatever the inverse's last bit: at the longest
        // head's length there are no more pieces than heads, which have a block each.
        const auto pieces_of = [&piece](int held, float inverse) {
            return min(held, held <= piece ? 1 : max(1, __float2int_ru(static_cast<float>(held) * inverse)));
        };
        const auto held_by = [&](int r) { return r < requests ? held_pages[r] : 0; };
        int longest = 0;
        for (int r = lane; r < requests; r += 32) longest = max(longest, held_by(r));
        longest = max(__reduce_max_sync(~0u, longest), 1);
        // (From here on, so that the units are asked for together with the pages: one request 6.2 -> 5.6 us.)
        shares = static_cast<int>(max64(1, min64(ranges, (units << g.shift) / (C::kWarps * C::kChunk))));
        piece = max(1, static_cast<int>(__fdividef(static_cast<float>(units), static_cast<float>(shares))));
        // Heads that are not much longer than that (by about the time of a join) stay whole.
        if (longest <= piece + ((12 * C::kChunk) >> g.shift)) {
            if (range < segments) {
                s = range / kv_heads;
                h = range - s * kv_heads;
                p1 = held_by(s);
            }
            piece = 0;
        }
        float inverse = 0.0f;
        while (piece > 0) {
            piece = min(piece, longest);
            int count = 0;
            inverse = __fdividef(1.0f, static_cast<float>(piece));
            for (int r = lane; r < requests; r += 32) count += pieces_of(held_by(r), inverse);
            count = __reduce_add_sync(~0u, count) * kv_heads;
            if (count <= ranges || piece == longest) break;
            piece = max(piece + 1, static_cast<int>(__fdividef(static_cast<float>(piece) * count, static_cast<float>(ranges))));
        }
        // The request that piece `range` belongs to, by a scan of the requests' pieces.
        int before = 0;
        for (int base = 0; piece > 0 && base < requests; base += 32) {
            const int own = pieces_of(held_by(base + lane), inverse) * kv_heads;
            int upto = own;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int other = __shfl_up_sync(~0u, upto, d);
                if (lane >= d) upto += other;
            }
            const uint32_t beyond = __ballot_sync(~0u, before + upto > range);
            if (beyond != 0) {
                const int hit = __ffs(beyond) - 1;
                s = base + hit;
                const int index = range - before - __shfl_sync(~0u, upto - own, hit);  // of the request's pieces
                const int held = held_by(s), each = pieces_of(held, inverse), i = index % each;
                const int even = held / each, rest = held - even * each;  // the first `rest` pieces have one page more
                h = index / each;
                p0 = i * even + min(i, rest);
                p1 = p0 + even + (i < rest);
                first_block = range - i;
                last_block = first_block + each - 1;
                break;
            }
            before += __shfl_sync(~0u, upto, 31);
        }
        end = p1 > p0;  // one segment at most
    } else {
        // A bound that falls into a short head moves to the nearer end of it: a join
        // would take longer than the head (2,048 heads of 100 to 400 tokens 47 -> 37 us).
        // A long head's shares stay the same ones.
        const auto bound = [&](int64_t u, int& at) {
            at = find_request(page_offsets, requests, kv_heads, u, lane);
            const int64_t base = (int64_t)kv_heads * page_offsets[at];
            const int held = page_offsets[at + 1] - page_offsets[at];
            if (held <= 0 || held > ((8 * C::kWarps * C::kChunk) >> g.shift) || u < base || u >= base + (int64_t)kv_heads * held) return u;
            const int into = static_cast<int>(u - base), rest = into % held;
            return u - rest + (2 * rest < held ? 0 : held);
        };
        shares = static_cast<int>(max64(1, min64(ranges, units)));
        if (range < shares) {
            int unused;
            end = bound(units * (range + 1) / shares, unused);
            begin = bound(units * range / shares, s);
        }
    }

    for (int64_t u = begin; u < end;) {
        int64_t start = 0;  // shares: the head's first unit
        int held;
        if (pieces) {
            held = reinterpret_cast<const int32_t*>(smem)[s];
            u = end;
        } else {
            int64_t base = (int64_t)kv_heads * page_offsets[s];
            held = page_offsets[s + 1] - page_offsets[s];
            while (u >= base + (int64_t)kv_heads * held && s + 1 < requests) {
                ++s;
                base = (int64_t)kv_heads * page_offsets[s];
                held = page_offsets[s + 1] - page_offsets[s];
            }
            if (held <= 0 || u < base || u >= base + (int64_t)kv_heads * held) break;  // offsets that are no prefix sum
            h = static_cast<int>((u - base) / held);
            start = base + (int64_t)h * held;
            p0 = static_cast<int>(u - start);
            p1 = static_cast<int>(min64(held, end - start));
            u = start + p1;
        }
        // This warp's chunks: keys ka + 32 (warp + kWarps i) and on.  The first page
        // numbers are asked for together with the request's lengths.
        const bool within = p0 < g.step.max_pages;
        const int ka = within ? p0 << g.shift : 0;
        const int32_t* table = g.step.table + (int64_t)s * g.step.max_pages;
        const int pages_end = static_cast<int>(min64(p1, g.step.max_pages));
        const auto page_of = [&](int i) {  // lanes 0-15: the page of the chunk's first group; 16-31: of the second
            const int at = (ka + C::kChunk * (warp + C::kWarps * i) + (lane & 16)) >> g.shift;
            return at < pages_end ? table[at] : INT_MIN;
        };
        int ids[C::kStages];
#pragma unroll
        for (int i = 0; i < C::kStages; ++i) ids[i] = page_of(i);
        const int context = g.step.context[s], length = g.step.lengths[s];
        const int64_t row0 = max64(0, g.step.token_offsets[s]);
        const int new_rows = static_cast<int>(
            max64(0, min64(min64(g.step.token_offsets[s + 1], g.step.tokens) - row0, g.most_tokens)) * g.group);
        if (pieces) __syncthreads();  // the requests' pages are read: the rings are free
        const int first_row = row_block * 8;
        if (first_row >= new_rows) continue;
        const int rows = min(8, new_rows - first_row);
        // Keys [ka, kb) for the block; the last row sees the most.
        const int kb = within ? static_cast<int>(min64(min64((int64_t)p1 << g.shift, length),
                                                       (int64_t)context + (first_row + rows - 1) / g.group + 1))
                              : 0;

        // Loads run kStages - 1 turns ahead, the page numbers they need one turn further.
        // A chunk is two groups of 16 keys, each 16 D consecutive bytes of a page.
        const int chunks = kb > ka ? (kb - ka + C::kChunk - 1) / C::kChunk : 0;
        const int mine = chunks > warp ? (chunks - warp + C::kWarps - 1) / C::kWarps : 0;
        // A lane's 16-byte pieces of a group: n-th from the first, in the ring and (V) in the page.
        constexpr int kPieces = D / 16;  // of a row
        const int lane_row = lane / kPieces, lane_piece = lane % kPieces;
        const int k_to = lane_row * D + 16 * k_piece<D>(lane_row, lane_piece);
        const int v_to = lane_row * D + 16 * v_piece<D>(lane_row, lane_piece);
        const int32_t page_bytes = (kv_heads << g.shift) * D;
        const int8_t* k_from = g.cache.k_codes + ((int64_t)h << g.shift) * D;
        const int8_t* v_from = g.cache.v_codes + ((int64_t)h << g.shift) * D + 16 * lane;
        const float* scale_from = (lane == 0 ? g.cache.k_scales : g.cache.v_scales) + h;
        int k_at[kPieces / 2];
#pragma unroll
        for (int n = 0; n < kPieces / 2; ++n) k_at[n] = D == 96 ? k_key((32 * n + lane) / 6) * D + 16 * ((32 * n + lane) % 6)
                                                      : k_key(lane_row) * D + 16 * lane_piece +
                                                            (D == 128 ? (2 * (n & 1) + 8 * (n >> 1)) * D : n * 512);
        const auto load = [&](int i, int slot, int id) {
            uint8_t* stage = ring + slot * C::kStage;
            if (i < mine) {
                const int key = ka + C::kChunk * (warp + C::kWarps * i);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int page_id = key + 16 * half < kb ? __shfl_sync(~0u, id, 16 * half) : INT_MIN;
                    float* scales = reinterpret_cast<float*>(stage + 2 * C::kTile) + 2 * half;
                    if (page_id >= 0 && page_id < g.cache.pages) {
                        const int64_t src = (int64_t)page_id * page_bytes + ((key + 16 * half) & (page - 1)) * D;
#pragma unroll
                        for (int n = 0; n < kPieces / 2; ++n) {
                            async_copy16(stage + 16 * half * D + k_to + 512 * n, k_from + src + k_at[n]);
                            async_copy16(stage + C::kTile + 16 * half * D + v_to + 512 * n, v_from + src + 512 * n);
                        }
                        if (lane < 2) async_copy4(scales + lane, scale_from + (int64_t)page_id * kv_heads);
                    } else if (lane == 0) {
                        scales[0] = 0.0f;
                        scales[1] = -1.0f;  // the group is not there
                        if (page_id != INT_MIN) record_device_error(kSiteKv8Range);
                    }
                }
            }
            commit_async_copies();
        };
        if (tid == 0) {
            // Its parts' blocks i0 .. i1; a block's parts lie side by side: the head that it
            // ends, then the one that it begins.
            const int i0 = pieces ? first_block : static_cast<int>(((start + 1) * shares - 1) / units);
            const int i1 = pieces ? last_block : static_cast<int>(((start + held) * shares - 1) / units);
            segment_s.row0 = row0;
            segment_s.h = h;
            segment_s.rows = rows;
            segment_s.own = p0 > 0 ? 0 : 1;
            segment_s.parts = p0 > 0 || p1 < held ? i1 - i0 + 1 : 0;
            segment_s.first_part = i0;
        }
        // The query rows and the first chunks are under way together.
        constexpr int kRowThreads = D == 32 ? 4 : D == 64 ? 8 : 16;
        constexpr int kRowPasses = 8 * kRowThreads <= C::kThreads ? 1 : 8 * kRowThreads / C::kThreads;
        static_assert(kRowThreads >= D / 8 && kRowPasses * C::kThreads >= 8 * kRowThreads, "eight values a thread and pass");
        const int item = tid % kRowThreads;
        QueryItem<D> rows_item[kRowPasses];
#pragma unroll
        for (int pass = 0; pass < kRowPasses; ++pass) {
            const int row = tid / kRowThreads + pass * (C::kThreads / kRowThreads);
            if (row < 8 && item < D / 8) {
                const int t = (first_row + row) / g.group, hq = (first_row + row) - t * g.group;
                int64_t pos = (int64_t)context + t;
                if (row < rows && g.rotary > 0 && (pos < 0 || pos >= g.table_rows)) {
                    if (item == 0) record_device_error(kSiteKv8Range);
                    pos = 0;
                }
                rows_item[pass].load(g, row < rows ? g.q + (row0 + t) * g.q_stride + (int64_t)(h * g.group + hq) * D : nullptr, item, pos);
            }
        }
#pragma unroll
        for (int i = 0; i < C::kStages - 1; ++i) load(i, i, ids[i]);
        int next_id = ids[C::kStages - 1];
#pragma unroll
        for (int pass = 0; pass < kRowPasses; ++pass) {
            const int row = tid / kRowThreads + pass * (C::kThreads / kRowThreads);
            if (row >= 8) break;
            // Four elements in a row are one lane's part of one MMA: lane (gq, tq) holds
            // row gq's elements that meet its bytes of a key, 16 of each 64 (D = 64, 128)
            // or D / 4 in a row.
            QueryItem<D>& mine_item = rows_item[pass];
            if (item < D / 8) mine_item.turn();
            uint32_t largest = item < D / 8 ? mine_item.largest() : 0;
#pragma unroll
            for (int d = 1; d < kRowThreads; d *= 2) largest = max(largest, __shfl_xor_sync(~0u, largest, d));
            float up, down;
            row_power(largest, up, down);
            if (item == 0) factor_s[row] = down * g.scale * kLog2e;
            const auto put = [&](int at, float4 x) {
                const int j = D % 64 == 0 ? at / 64 * 4 + at % 16 / 4 : at % (D / 4) / 4;
                const int t = D % 64 == 0 ? at % 64 / 16 : at / (D / 4);
                const float a = x.x * up, b = x.y * up, c = x.z * up, d = x.w * up;
                const uint32_t ab = half2_bits(a, b), cd = half2_bits(c, d);
                const __half2 ab2 = *reinterpret_cast<const __half2*>(&ab), cd2 = *reinterpret_cast<const __half2*>(&cd);
                q_s[j * 32 + row * 4 + t] = make_uint4(ab, half2_bits(a - __low2float(ab2), b - __high2float(ab2)), cd,
                                                       half2_bits(c - __low2float(cd2), d - __high2float(cd2)));
            };
            if (item < D / 8) {
                put(mine_item.at, mine_item.a);
                put(mine_item.to, mine_item.b);
            }
        }
        __syncthreads();
        uint32_t q[D / 16][4];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) *reinterpret_cast<uint4*>(q[j]) = q_s[j * 32 + lane];
        const float factor = factor_s[gq];  // from an MMA sum to x_j / ks
        // Keys that row gq sees; none for a row past the request's.
        const int64_t row_pos = (int64_t)context + (first_row + gq) / g.group;
        const bool seen = gq < rows && row_pos >= 0 && (g.rotary == 0 || row_pos < g.table_rows);
        const int limit = seen ? static_cast<int>(min64(kb, row_pos + 1)) : 0;

        float o[D / 8][2], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = 0.0f;

        int slot = 0;
        for (int i = 0; i < mine; ++i) {
            {
                const int id = next_id, into = slot == 0 ? C::kStages - 1 : slot - 1;
                next_id = page_of(i + C::kStages);
                load(i + C::kStages - 1, into, id);
            }
            wait_async_copies_but<C::kStages - 1>();
            __syncwarp();
            const uint8_t* stage = ring + slot * C::kStage;
            slot = slot + 1 == C::kStages ? 0 : slot + 1;
            const int key = ka + C::kChunk * (warp + C::kWarps * i);
            const float4 scales = *reinterpret_cast<const float4*>(stage + 2 * C::kTile);
            float ks[2], bias[2], frac[2], back[2];  // per group: x / sum, e, f, 2^-e
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float vs = n == 0 ? scales.y : scales.w;
                const bool number = vs >= kLeastScale && vs < INFINITY;
                const int e = number ? __float_as_int(vs) >> 23 : kZeroExponent;
                // A V scale that is no number shows in the scores: where they are hidden it does not.
                ks[n] = fmaf(vs, 0.0f, (n == 0 ? scales.x : scales.z) * factor);
                bias[n] = vs < 0.0f ? -INFINITY : static_cast<float>(e - 127);
                back[n] = __int_as_float((254 - e) << 23);
                frac[n] = number ? vs * back[n] : 0.0f;
            }

            // Scores of keys key + 8 n + {tq, 4 + tq} (n-tile n), in x + e.
            float x[4][2];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const int r = 8 * n + gq;
                uint32_t w[D / 16];
                if constexpr (D % 64 == 0) {
#pragma unroll
                    for (int c = 0; c < D / 64; ++c)
                        *reinterpret_cast<uint4*>(w + 4 * c) =
                            *reinterpret_cast<const uint4*>(stage + r * D + 16 * k_piece<D>(r, 4 * c + tq));
                } else {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c)
                        *reinterpret_cast<uint2*>(w + 2 * c) = *reinterpret_cast<const uint2*>(stage + r * D + tq * (D / 4) + 8 * c);
                }
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const uint32_t biased = w[j] ^ 0x80808080u;
                    mma_f16(acc, q[j], codes_half2(biased, 0x4140u), codes_half2(biased, 0x4342u));
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) x[n][e] = fmaf(acc[e] + acc[e + 2], ks[n >> 1], bias[n >> 1]);
            }
            if (__any_sync(~0u, key + C::kChunk > limit)) {
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (key + 8 * n + tq + 4 * e >= limit) x[n][e] = -INFINITY;
            }
            // The weights count relative to m, a whole power of two that is the same for
            // the row's four lanes.  It comes from the row's first keys; later ones are
            // weighed with it as it stands, and only where weights come out above
            // kHighest is it raised, with O and L scaled down (exactly) to the new one.
            // A row that sees none of them keeps having none: any other would stand above
            // its own keys' where the warps and the parts are joined.
            uint32_t p[2][4];
            float sum;
            bool first = true;
#pragma unroll 1
            for (;;) {
                const float shift = m == -INFINITY ? INFINITY : m - kLift;
                sum = 0.0f;
                float most = 0.0f;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    float hi[2], lo[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float u = ex2(x[n][e] - shift), w = u * frac[n >> 1];
                        most = fmaxf(most, u);
                        sum = fmaf(u, back[n >> 1], sum);
                        hi[e] = __uint_as_float(__float_as_uint(w) & 0xffffe000u);  // 11 bits: exact in fp16
                        lo[e] = w - hi[e];
                    }
                    p[n >> 1][2 * (n & 1)] = half2_bits(hi[0], hi[1]);
                    p[n >> 1][2 * (n & 1) + 1] = half2_bits(lo[0], lo[1]);
                }
                if (!__any_sync(~0u, most > kHighest || (first && m == -INFINITY && key < limit))) break;
                first = false;
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 4; ++n) top = fmaxf(top, fmaxf(x[n][0], x[n][1]));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                const float raised = fmaxf(m, ceilf(top));
                const float down = m == -INFINITY ? 0.0f : ex2(m - raised);
                m = raised;
                l *= down;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    o[j][0] *= down;
                    o[j][1] *= down;
                }
            }
            l += sum;
            // A chunk's products sum up in the MMA, whose additions truncate; the
            // chunks are added in rounded fp32.
            constexpr int kWords = D / 32;
            // Keys 16 step + 4 k + tq, elements gq (D / 8) ..: byte n of word c is n-tile 4 c + n's column gq.
            uint32_t w[2][4][kWords];
#pragma unroll
            for (int step = 0; step < 2; ++step)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = 16 * step + 4 * k + tq;
                    const uint8_t* row = stage + C::kTile + r * D;
                    if constexpr (D == 128) {
                        *reinterpret_cast<uint4*>(w[step][k]) = *reinterpret_cast<const uint4*>(row + 16 * v_piece<D>(r, gq));
                    } else if constexpr (D == 64) {
                        *reinterpret_cast<uint2*>(w[step][k]) =
                            *reinterpret_cast<const uint2*>(row + 16 * v_piece<D>(r, gq >> 1) + 8 * (gq & 1));
                    } else {
#pragma unroll
                        for (int c = 0; c < kWords; ++c)
                            w[step][k][c] = *reinterpret_cast<const uint32_t*>(row + gq * (D / 8) + 4 * c);
                    }
                }
#pragma unroll
            for (int c = 0; c < kWords; ++c) {
                float part[4][4] = {};
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    // Bytes of keys (2t, 2t+1) and (2t+8, 2t+9) side by side.
                    const uint32_t x0 = w[step][0][c] ^ 0x80808080u, x1 = w[step][1][c] ^ 0x80808080u,
                                   x2 = w[step][2][c] ^ 0x80808080u, x3 = w[step][3][c] ^ 0x80808080u;
                    const uint32_t a01 = __byte_perm(x0, x1, 0x5140), a23 = __byte_perm(x0, x1, 0x7362);
                    const uint32_t b01 = __byte_perm(x2, x3, 0x5140), b23 = __byte_perm(x2, x3, 0x7362);
                    mma_f16(part[0], p[step], codes_half2(a01, 0x4140u), codes_half2(b01, 0x4140u));
                    mma_f16(part[1], p[step], codes_half2(a01, 0x4342u), codes_half2(b01, 0x4342u));
                    mma_f16(part[2], p[step], codes_half2(a23, 0x4140u), codes_half2(b23, 0x4140u));
                    mma_f16(part[3], p[step], codes_half2(a23, 0x4342u), codes_half2(b23, 0x4342u));
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    o[4 * c + n][0] += part[n][0] + part[n][2];
                    o[4 * c + n][1] += part[n][1] + part[n][3];
                }
            }
            __syncwarp();  // the stage is read before it is copied into again
        }
        wait_async_copies_but<0>();
        __syncwarp();

        // Join the warps: each leaves m, l and O in its ring.
        float* part = reinterpret_cast<float*>(ring);
        l += __shfl_xor_sync(~0u, l, 1);
        l += __shfl_xor_sync(~0u, l, 2);
        if (tq == 0) {
            part[gq] = m;
            part[8 + gq] = l;
        }
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            // n-tile j's columns 2t, 2t+1 are elements (2t) (D/8) + j and (2t+1) (D/8) + j.
            part[16 + gq * D + 2 * tq * (D / 8) + j] = o[j][0];
            part[16 + gq * D + (2 * tq + 1) * (D / 8) + j] = o[j][1];
        }
        __syncthreads();
        const int count = segment_s.parts, rows_here = segment_s.rows;
        float* out = g.out + segment_s.row0 * g.heads * D + (int64_t)segment_s.h * g.group * D;
        float* own = parts + ((2 * (int64_t)range + segment_s.own) * row_blocks + row_block) * C::kPart;
        for (int item = tid; item < 8 * D; item += C::kThreads) {
            const int r = item / D, d = item - r * D;
            float top = -INFINITY, sum = 0.0f, total = 0.0f;
#pragma unroll
            for (int w = 0; w < C::kWarps; ++w) top = fmaxf(top, reinterpret_cast<const float*>(smem + w * C::kRing)[r]);
#pragma unroll
            for (int w = 0; w < C::kWarps; ++w) {
                const float* other = reinterpret_cast<const float*>(smem + w * C::kRing);
                const float weight = other[r] == -INFINITY ? (other[8 + r] == 0.0f ? 0.0f : 1.0f) : ex2(other[r] - top);
                total = fmaf(weight, other[8 + r], total);
                sum = fmaf(weight, other[16 + item], sum);
            }
            if (count > 0) {
                if (d == 0) {
                    own[r] = top;
                    own[8 + r] = total;
                }
                own[16 + item] = sum;
            } else if (r < rows_here) {
                const int t = (first_row + r) / g.group, hq = (first_row + r) - t * g.group;
                out[t * (int64_t)g.heads * D + hq * D + d] = total == 0.0f ? 0.0f : sum / total;
            }
        }
        if (count > 0) {
            // The last block to arrive joins the segment's parts.
            const int64_t first = (2 * (int64_t)segment_s.first_part * row_blocks + row_block) * C::kPart;
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                uint32_t* arrived = arrivals + (int64_t)segment_s.first_part * row_blocks + row_block;
                last_s = atomicAdd(arrived, 1u) == static_cast<uint32_t>(count - 1);
                if (last_s) *arrived = 0;
                __threadfence();
            }
            __syncthreads();
            if (last_s)
                join_parts<D, kNarrow>(smem, parts + first, 2 * (int64_t)row_blocks * C::kPart, (int64_t)row_blocks * C::kPart, count,
                              rows_here, g.group, first_row, out, (int64_t)g.heads * D);
        }
        __syncthreads();  // the rings and q_s are free for the next segment
    }

    // Requests that hold no page: their rows see no key.
    for (int r = range; r < requests; r += ranges) {
        if (g.step.page_offsets[r + 1] != g.step.page_offsets[r]) continue;
        const int64_t row0 = max64(0, g.step.token_offsets[r]);
        const int64_t count = max64(0, min64(g.step.token_offsets[r + 1], g.step.tokens) - row0) * g.group;
        for (int64_t row = row_block * 8; row < min64(count, row_block * 8 + 8); ++row)
            for (int d = tid; d < kv_heads * D; d += C::kThreads)
                g.out[(row0 + row / g.group) * (int64_t)g.heads * D + ((int64_t)(d / D) * g.group + row % g.group) * D + d % D] =
                    0.0f;
    }
}

// Row blocks of 8, key ranges per row block, and what the workspace holds behind
// the counters (one for every range and row block): two partial results for each.
struct SplitShape {
    int64_t row_blocks, ranges;
    size_t part_bytes;
};

template <int D, bool kNarrow>
SplitShape split_shape(int64_t max_tokens, int group) {
    using C = Split<D, kNarrow>;
    SplitShape f;
    f.row_blocks = (max_tokens * group + 7) / 8;
    if (f.row_blocks < 1) f.row_blocks = 1;
    // About one wave of blocks in all; from there on one block per row block,
    // whose requests it walks alone.
    f.ranges = (C::kBlocks + f.row_blocks - 1) / f.row_blocks;
    static_assert(2 * C::kBlocks <= kSplitCounters, "ranges * row_blocks, where there is more than one range");
    f.part_bytes = f.ranges > 1 ? 2 * static_cast<size_t>(f.ranges * f.row_blocks) * C::kPart * sizeof(float) : 0;
    return f;
}

template <int D, bool kNarrow>
int run_split(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl) {
    using C = Split<D, kNarrow>;
    const SplitShape f = split_shape<D, kNarrow>(g.step.max_tokens, g.group);
    // More heads than wide blocks go to narrow ones.  Wide and narrow, us, 64-wide
    // heads: 256 heads of 521 to 765 tokens 13.5 and 20.3, 1,024 heads of 500 to
    // 1,000 tokens 54.6 and 39.7, 2,048 of 100 to 400 72 and 37; 128-wide: 48 of
    // 15,000 to 91,000 tokens 103 and 124, 512 of 1,000 to 4,000 88 and 90, 1,024 of
    // 500 to 1,500 85 and 76, 2,048 of 200 to 2,000 167 and 138.
    if (!kNarrow && (int64_t)g.step.requests * g.cache.kv_heads > f.ranges) return run_split<D, true>(s, g, workspace, pdl);
    if (f.ranges * f.row_blocks > INT_MAX / 8) {
        set_error("leafq_kv8_attention: max_tokens * group is too large");
        return LEAFQ_ERR_INVALID;
    }
    const auto kernel = kv8_attend_split_kernel<D, kNarrow>;
    const int st = allow_smem(reinterpret_cast<const void*>(kernel), C::kSmem, "leafq_kv8_attention");
    if (st) return st;
    uint32_t* arrivals = static_cast<uint32_t*>(workspace);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
    return launch(kernel, dim3(static_cast<unsigned>(f.ranges * f.row_blocks)), dim3(C::kThreads), C::kSmem, s, pdl,
                  "leafq_kv8_attention", g, parts, arrivals, static_cast<int>(f.ranges), static_cast<int>(f.row_blocks));
}

// The tile form gives 128 rows of a request's kv head to a block, the split form
// 8: the tile form wants a quarter of them at least, and enough rows in all.
// Measured with 8 kv heads of 64 (128) and 8,000 cached tokens, split form and
// tile form, us: 2,048 rows of 8 requests 74 and 84 (172 and 122), 4,096 rows 134
// and 85 (294 and 122), 8,192 rows 384 and 99 (569 and 157); with 1,000 cached
// tokens 2,048 rows 16 and 31 (33 and 42), 4,096 rows 35 and 31 (65 and 44).  Over
// 520 shapes of 256 to 64,000 rows this rule is 1 to 3 % above the better form; in
// all of them the requests bring equally many tokens to equally long caches.  A batch
// takes one form: one-token requests beside a prompt's chunk go to the tiles with it,
// which is right but was not measured.
constexpr int kTileRows = 32;
bool takes_tiles(int64_t tokens, int64_t max_tokens, int heads, int group) {
    return max_tokens * group >= kTileRows && tokens * heads >= 3584;
}

// Calls f(integral constant D) for a supported head size.
template <typename F>
auto with_dim(int dim, F&& f) {
    switch (dim) {
        case 32: return f(std::integral_constant<int, 32>{});
        case 64: return f(std::integral_constant<int, 64>{});
        case 96: return f(std::integral_constant<int, 96>{});
        default: return f(std::integral_constant<int, 128>{});
    }
}

}  // namespace
}  // namespace leafq

using namespace leafq;

extern "C" {

size_t leafq_kv8_attention_workspace_bytes(int64_t max_tokens, int heads, int kv_heads, int dim) {
    if (max_tokens <= 0 || max_tokens > INT_MAX || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
        !kv8_dim_supported(dim))
        return 0;
    return with_dim(dim, [&](auto d) {
        const size_t parts = std::max(split_shape<d(), false>(max_tokens, heads / kv_heads).part_bytes,
                                      split_shape<d(), true>(max_tokens, heads / kv_heads).part_bytes);
        const bool tiles = max_tokens * (heads / kv_heads) >= kTileRows;
        return kCounterBytes + std::max(parts, tiles ? kv8_tile_part_bytes(d()) : 0);
    });
}

int leafq_kv8_attention(void* stream, const float* q, int64_t q_stride, int heads, int rotary_dim,
                        const float* cos_table, const float* sin_table, int64_t table_rows,
                        const leafq_kv8_cache* cache, const leafq_kv8_step* step, float scale, float* out,
                        void* workspace, size_t workspace_bytes, uint32_t flags) {
    clear_error();
    if (!kv8_cache_valid(cache, "leafq_kv8_attention")) return LEAFQ_ERR_INVALID;
    if (!kv8_dim_supported(cache->dim)) {
        set_error("leafq_kv8_attention: head sizes are 32, 64, 96 and 128");
        return LEAFQ_ERR_UNSUPPORTED;
    }
    if (!kv8_rope_valid(cache->dim, rotary_dim, cos_table, sin_table, table_rows, "leafq_kv8_attention"))
        return LEAFQ_ERR_INVALID;
    if (!step || step->tokens < 0 || step->tokens > INT_MAX || step->max_tokens < 0 || step->requests < 0 ||
        step->max_pages < 0 || step->max_pages > INT_MAX / cache->page || heads <= 0 || heads > 65535 ||
        heads % cache->kv_heads != 0 || !(scale > 0.0f) || scale > 3.0e38f) {
        set_error("leafq_kv8_attention: invalid step, heads (a multiple of the cache's) or scale (positive)");
        return LEAFQ_ERR_INVALID;
    }
    if (step->tokens == 0 || step->requests == 0) return LEAFQ_OK;
    if (!q || !out || !step->context || !step->lengths || !step->token_offsets || !step->page_offsets ||
        (step->max_pages > 0 && !step->table)) {
        set_error("leafq_kv8_attention: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    if ((step->tokens > 1 && q_stride < (int64_t)heads * cache->dim) || q_stride % 4 != 0 || !aligned16(q) ||
        !aligned16(out)) {
        set_error("leafq_kv8_attention: q and out rows must be 16-byte aligned and must not overlap");
        return LEAFQ_ERR_INVALID;
    }
    if (step->max_tokens == 0) return LEAFQ_OK;
    const size_t need = leafq_kv8_attention_workspace_bytes(step->max_tokens, heads, cache->kv_heads, cache->dim);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
        set_error("leafq_kv8_attention: this shape needs " + std::to_string(need) +
                  " bytes of 16-byte aligned workspace");
        return LEAFQ_ERR_INVALID;
    }
    Kv8AttendArgs g{q, q_stride, cos_table, sin_table, table_rows, *cache, *step, out, scale, heads,
                 heads / cache->kv_heads, rotary_dim, 0, INT_MAX / (heads / cache->kv_heads)};
    while ((1 << g.shift) < cache->page) ++g.shift;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool pdl = (flags & LEAFQ_FLAG_PDL) != 0;
    if (takes_tiles(step->tokens, step->max_tokens, heads, g.group)) return launch_kv8_tiles(s, g, workspace, pdl);
    return with_dim(cache->dim, [&](auto d) { return run_split<d(), false>(s, g, workspace, pdl); });
}

}  // extern "C"
