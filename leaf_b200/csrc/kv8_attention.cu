// Causal grouped-query attention over the paged INT8 KV cache
// (include/leafq.h, leafq_kv8_attention).
//
// For the query row (request s, new token t, head h) at position
// p = context[s] + t, over keys j < min(p + 1, lengths[s]):
//   x_j = scale * ks * (q . ck_j)      ks, vs: the scales of key j's page
//   out = sum_j exp(x_j - m) vs cv_j / sum_j exp(x_j - m),  m = max x
// in one pass over the keys: when the maximum grows from m to m', the sums so
// far are multiplied by exp(m - m').
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "leafq_device.cuh"
#include "leafq_internal.h"

namespace leafq {
namespace {

struct AttendArgs {
    const float* q;
    int64_t q_stride;
    const float* cos_table;
    const float* sin_table;
    int64_t table_rows;
    leafq_kv8_cache cache;
    leafq_kv8_step step;
    float* out;
    float scale;
    int heads, group, rotary, shift;
};

constexpr float kLog2e = 1.4426950408889634f;
// Weights are held as 2^kLift times their value relative to the largest, so
// that the second half of a weight's fp16 split stays a normal number down to
// 2^-28 of the largest; 2^14 times 127 codes is far from fp32's range.
constexpr float kLift = 14.0f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Bytes s of {a, b} (two 16-bit halves of a prmt selector) as two fp16 codes.
// The codes come biased to 0 .. 255 (sign bit flipped): 0x6400 + u is the
// fp16 number 1024 + u, exact, and subtracting 1152 leaves the code.
__device__ __forceinline__ uint32_t codes_half2(uint32_t biased, uint32_t selector) {
    uint32_t r;
    asm("{\n\t.reg .b32 x;\n\t"
        "prmt.b32 x, %1, 0x64646464, %2;\n\t"
        "sub.rn.f16x2 %0, x, %3;\n\t}"
        : "=r"(r)
        : "r"(biased), "r"(selector), "r"(0x64806480u));
    return r;
}

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

// Eight values of a query row, its item j of D / 8 (a rotation pair's quarters
// as in the append): a at `at`, b at `to`.
template <int D>
__device__ __forceinline__ void query_item(const AttendArgs& g, const float* row, int j, int64_t pos, int& at, int& to,
                                           float4& a, float4& b) {
    const int half = g.rotary >> 1;
    const bool turned = 4 * j < half;
    at = turned ? 4 * j : 2 * half + 4 * (j - half / 4);
    to = turned ? at + half : at + ((D - 2 * half) >> 1);
    a = *reinterpret_cast<const float4*>(row + at);
    b = *reinterpret_cast<const float4*>(row + to);
    if (turned) {
        const float4 c = *reinterpret_cast<const float4*>(g.cos_table + pos * half + at);
        const float4 s = *reinterpret_cast<const float4*>(g.sin_table + pos * half + at);
        const float4 x = a, y = b;
        a = make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x)), __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y)),
                        __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z)), __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w)));
        b = make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(x.x, s.x)), __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(x.y, s.y)),
                        __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(x.z, s.z)), __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(x.w, s.w)));
    }
}

// The power of two that brings a row's largest magnitude into [256, 512), as
// a float and its inverse (1 for a row of zeros): exact, and fp16's range
// then holds the row whatever its own.
__device__ __forceinline__ void row_power(uint32_t largest_bits, float& up, float& down) {
    const int e = static_cast<int>(largest_bits >> 23);
    int k = 262 - e;
    k = k > 253 ? 253 : (k < 1 ? 1 : k);
    if (largest_bits == 0) k = 127;
    up = __uint_as_float(static_cast<uint32_t>(k) << 23);
    down = __uint_as_float(static_cast<uint32_t>(254 - k) << 23);
}

// ---------------------------------------------------------- split form
// Few query rows, many keys (decode).  A block owns 8 query rows of one kv
// head (rows r = token * group + head-in-group of a request) and a range of the keys; its warps take chunks of 32 keys in
// turn, each warp with its own running maximum, sum and output.
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
// u_j = 2^(x_j + e - M) with M the running maximum of x_j + e; O sums f u_j cv_j
// and L sums u_j 2^-e, so O / L is the softmax average whatever the scales'
// range, and neither half rounds.
//
// Bound: HBM (the codes are read once: cp.async into a ring per warp, 16-byte
// pieces, rows swizzled so that both fragment reads touch every bank once);
// behind it the conversions, 5 and 7 issue slots per four codes of K and V.
template <int D>
struct Split {
    static constexpr int kWarps = D <= 64 ? 8 : 4;
    static constexpr int kBlocksPerSm = D <= 64 ? 2 : 3;
    static constexpr int kStages = D <= 64 ? 3 : 2;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kBlocks = 148 * kBlocksPerSm;   // key ranges of one row block
    static constexpr int kChunk = 32;                    // keys per warp and turn
    static constexpr int kTile = kChunk * D;             // bytes of K (or V) per chunk
    static constexpr int kStage = 2 * kTile + 32;        // + {ks, vs} of its two 16-key groups
    static constexpr int kRing = kStages * kStage;
    static constexpr int kPart = 8 * (D + 2);            // floats of one partial result: m [8], l [8], O [8][D]
    static constexpr size_t kSmem = (size_t)kWarps * kRing + 8 * D * sizeof(float);
    static_assert(kRing >= kPart * 4, "a warp's partial result goes through its ring");
    static_assert(kWarps * kRing >= (kBlocks + 1) * 8 * 4 + (kThreads * 4 + 8 * D) * 4, "joining goes through the rings");
};

// Where 16-byte piece c of row r of a chunk lies within the row.
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

template <int D>
__global__ void __launch_bounds__(Split<D>::kThreads, Split<D>::kBlocksPerSm)
kv8_attend_split_kernel(const AttendArgs g, float* parts, uint32_t* arrivals, int ranges, int row_blocks) {
    using C = Split<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int last_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, tq = lane & 3;
    uint8_t* ring = smem + warp * C::kRing;
    float* q_s = reinterpret_cast<float*>(smem + C::kWarps * C::kRing);
    grid_dependency_wait();
    grid_launch_dependents();

    // Row blocks of one key range are neighbours, so that they share its codes in L2.
    const int range = blockIdx.x / row_blocks, row_block = blockIdx.x - range * row_blocks;
    const int page = 1 << g.shift;
    const int requests = g.step.requests, kv_heads = g.cache.kv_heads;
    const int64_t units = (int64_t)kv_heads * g.step.page_offsets[requests];
    // Work: units (page, head, request) in a row, an even share per block --
    // a request's head may then be split over blocks, which costs a partial
    // result each -- or one block for each request's head where that is no
    // longer than an even share and the joining (about 12 chunks' time).
    int64_t shares = min64(ranges, (units << g.shift) / (C::kWarps * C::kChunk));
    if (shares < 1) shares = 1;
    const int64_t segments = (int64_t)requests * kv_heads;
    bool whole = false;
    if (segments <= ranges) {
        int longest = 0;
        for (int s = lane; s < requests; s += 32) longest = max(longest, g.step.page_offsets[s + 1] - g.step.page_offsets[s]);
        longest = __reduce_max_sync(~0u, longest);
        whole = (int64_t)longest << g.shift <= (units << g.shift) / shares + 12 * C::kChunk;
    }
    int64_t begin = 0, end = 0;
    int s = 0;
    if (whole) {
        if (range < segments) {
            s = range / kv_heads;
            const int64_t first = g.step.page_offsets[s], held = g.step.page_offsets[s + 1] - first;
            begin = first * kv_heads + (range - (int64_t)s * kv_heads) * held;
            end = begin + held;
        }
    } else if (range < shares) {
        begin = units * range / shares;
        end = units * (range + 1) / shares;
        s = find_request(g.step.page_offsets, requests, kv_heads, begin, lane);
    }

    for (int64_t u = begin; u < end;) {
        // Segment: pages [p0, p1) of head h of request s.
        int64_t base = (int64_t)kv_heads * g.step.page_offsets[s];
        int held = g.step.page_offsets[s + 1] - g.step.page_offsets[s];
        while (u >= base + (int64_t)kv_heads * held && s + 1 < requests) {
            ++s;
            base = (int64_t)kv_heads * g.step.page_offsets[s];
            held = g.step.page_offsets[s + 1] - g.step.page_offsets[s];
        }
        if (held <= 0 || u < base || u >= base + (int64_t)kv_heads * held) break;  // offsets that are no prefix sum
        const int h = static_cast<int>((u - base) / held);
        const int64_t start = base + (int64_t)h * held;  // the segment's first unit
        const int p0 = static_cast<int>(u - start), p1 = static_cast<int>(min64(held, end - start));
        u = start + p1;
        const int context = g.step.context[s];
        const int64_t row0 = max64(0, g.step.token_offsets[s]);
        const int new_rows = static_cast<int>(
            max64(0, min64(min64(g.step.token_offsets[s + 1], g.step.tokens) - row0, INT_MAX / g.group)) * g.group);
        const int first_row = row_block * 8;
        if (first_row >= new_rows) continue;
        const int rows = min(8, new_rows - first_row);
        // Keys [ka, kb) for the block; the last row sees the most.
        const int ka = p0 << g.shift;
        const int kb = static_cast<int>(min64(min64((int64_t)p1 << g.shift, g.step.lengths[s]),
                                              (int64_t)context + (first_row + rows - 1) / g.group + 1));

        // The rows, rotated, in shared memory.
        for (int item = tid; item < 8 * (D / 8); item += C::kThreads) {
            const int r = item / (D / 8), j = item - r * (D / 8);
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
            int at = 4 * j, to = at + D / 2;
            if (r < rows) {
                const int t = (first_row + r) / g.group, hq = (first_row + r) - t * g.group;
                int64_t pos = (int64_t)context + t;
                if (g.rotary > 0 && (pos < 0 || pos >= g.table_rows)) {
                    if (j == 0) record_device_error(kSiteKv8Range);
                    pos = 0;
                }
                query_item<D>(g, g.q + (row0 + t) * g.q_stride + (int64_t)(h * g.group + hq) * D, j, pos, at, to, a, b);
            }
            *reinterpret_cast<float4*>(q_s + r * D + at) = a;
            *reinterpret_cast<float4*>(q_s + r * D + to) = b;
        }

        // This warp's chunks: keys ka + 32 (warp + kWarps i) and on.  Loads run
        // kStages - 1 turns ahead, the page numbers they need one turn further.
        // A chunk is two groups of 16 keys, each 16 D consecutive bytes of a page.
        const int32_t* table = g.step.table + (int64_t)s * g.step.max_pages;
        const int chunks = kb > ka ? (kb - ka + C::kChunk - 1) / C::kChunk : 0;
        const int mine = chunks > warp ? (chunks - warp + C::kWarps - 1) / C::kWarps : 0;
        const auto page_of = [&](int i) {  // lanes 0-15: the page of the chunk's first group; 16-31: of the second
            const int key = ka + C::kChunk * (warp + C::kWarps * i) + (lane & 16);
            return i < mine && key < kb && (key >> g.shift) < g.step.max_pages ? table[key >> g.shift] : INT_MIN;
        };
        constexpr int kPieces = D / 16;  // 16-byte pieces of a row
        const auto load = [&](int i, int slot, int id) {
            uint8_t* stage = ring + slot * C::kStage;
            if (i < mine) {
                const int key = ka + C::kChunk * (warp + C::kWarps * i);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int page_id = __shfl_sync(~0u, id, 16 * half);
                    const int64_t tile = (int64_t)page_id * kv_heads + h;
                    float* scales = reinterpret_cast<float*>(stage + 2 * C::kTile) + 2 * half;
                    if (page_id >= 0 && page_id < g.cache.pages) {
                        const int64_t src = ((tile << g.shift) + ((key + 16 * half) & (page - 1))) * D + lane * 16;
#pragma unroll
                        for (int n = 0; n < kPieces / 2; ++n) {
                            const int c = n * 32 + lane, r = 16 * half + c / kPieces, cc = c % kPieces;
                            async_copy16(stage + r * D + 16 * k_piece<D>(r, cc), g.cache.k_codes + src + n * 512);
                            async_copy16(stage + C::kTile + r * D + 16 * v_piece<D>(r, cc), g.cache.v_codes + src + n * 512);
                        }
                        if (lane == 0) async_copy4(scales, g.cache.k_scales + tile);
                        if (lane == 1) async_copy4(scales + 1, g.cache.v_scales + tile);
                    } else if (lane == 0) {
                        scales[0] = 0.0f;
                        scales[1] = -1.0f;  // the group is not there
                        if (page_id != INT_MIN) record_device_error(kSiteKv8Range);
                    }
                }
            }
            commit_async_copies();
        };
        int next_id = page_of(0);
#pragma unroll
        for (int i = 0; i < C::kStages - 1; ++i) {
            const int id = next_id;
            next_id = page_of(i + 1);
            load(i, i, id);
        }

        __syncthreads();
        // Query fragments: lane (gq, tq) holds row gq's elements that meet its
        // bytes of a key: 16 of each 64 (D = 64, 128), else D / 4 in a row.
        uint32_t q[D / 16][4];
        float factor;  // from an MMA sum to x_j / ks
        {
            const float* row = q_s + gq * D;
            uint32_t largest = 0;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const int at = D % 64 == 0 ? (j / 4) * 64 + tq * 16 + (j % 4) * 4 : tq * (D / 4) + j * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) largest = max(largest, __float_as_uint(row[at + e]) & 0x7fffffffu);
            }
            largest = max(largest, __shfl_xor_sync(~0u, largest, 1));
            largest = max(largest, __shfl_xor_sync(~0u, largest, 2));
            float up, down;
            row_power(largest, up, down);
            factor = down * g.scale * kLog2e;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const int at = D % 64 == 0 ? (j / 4) * 64 + tq * 16 + (j % 4) * 4 : tq * (D / 4) + j * 4;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = row[at + 2 * e] * up, y = row[at + 2 * e + 1] * up;
                    const uint32_t hi = half2_bits(x, y);
                    const __half2 h2 = *reinterpret_cast<const __half2*>(&hi);
                    q[j][2 * e] = hi;
                    q[j][2 * e + 1] = half2_bits(x - __low2float(h2), y - __high2float(h2));
                }
            }
        }
        // Keys that row gq sees; none for a row past the request's.
        const int64_t row_pos = (int64_t)context + (first_row + gq) / g.group;
        const bool seen = gq < rows && row_pos >= 0 && (g.rotary == 0 || row_pos < g.table_rows);
        const int limit = seen ? static_cast<int>(min64(kb, row_pos + 1)) : 0;

        float o[D / 8][4], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;

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
                const int e = (__float_as_int(vs) >> 23) & 255;
                ks[n] = (n == 0 ? scales.x : scales.z) * factor;
                bias[n] = vs < 0.0f ? -INFINITY : static_cast<float>(e - 127);
                back[n] = __int_as_float(max(0, 254 - e) << 23);
                frac[n] = vs * back[n];
            }

            // Scores of keys key + 8 n + {tq, 4 + tq} (n-tile n), in x + e.
            float x[4][2], top = -INFINITY;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                // Column c of the tile is key (c >> 1) + 4 (c & 1): lane gq's key.
                const int r = 8 * n + (gq >> 1) + 4 * (gq & 1);
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
#pragma unroll
            for (int n = 0; n < 4; ++n) top = fmaxf(top, fmaxf(x[n][0], x[n][1]));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            // O and L so far count relative to the maximum so far.
            const float grown = fmaxf(m, top);
            const float old = m == -INFINITY ? 0.0f : ex2(m - grown);
            m = grown;
            l *= old;
            const float shift = m == -INFINITY ? 0.0f : m - kLift;
            uint32_t p[2][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float u = ex2(x[n][e] - shift), w = u * frac[n >> 1];
                    l = fmaf(u, back[n >> 1], l);
                    hi[e] = __uint_as_float(__float_as_uint(w) & 0xffffe000u);  // 11 bits: exact in fp16
                    lo[e] = w - hi[e];
                }
                p[n >> 1][2 * (n & 1)] = half2_bits(hi[0], hi[1]);
                p[n >> 1][2 * (n & 1) + 1] = half2_bits(lo[0], lo[1]);
            }
            // A chunk's products sum up in the MMA, whose additions truncate; the
            // chunks are added (and rescaled) in rounded fp32.
            constexpr int kWords = D / 32;
#pragma unroll
            for (int c = 0; c < kWords; ++c) {
                float part[4][4] = {};
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    // Keys 16 step + 4 k + tq, elements gq (D / 8) ..: byte n of them is n-tile n's column gq.
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = 16 * step + 4 * k + tq;
                        const uint8_t* row = stage + C::kTile + r * D;
                        w[k] = *reinterpret_cast<const uint32_t*>(
                                   D == 128 ? row + 16 * v_piece<D>(r, gq) + 4 * c
                                            : (D == 64 ? row + 16 * v_piece<D>(r, gq >> 1) + 8 * (gq & 1) + 4 * c
                                                       : row + gq * (D / 8) + 4 * c)) ^
                               0x80808080u;
                    }
                    // Bytes of keys (2t, 2t+1) and (2t+8, 2t+9) side by side.
                    const uint32_t a01 = __byte_perm(w[0], w[1], 0x5140), a23 = __byte_perm(w[0], w[1], 0x7362);
                    const uint32_t b01 = __byte_perm(w[2], w[3], 0x5140), b23 = __byte_perm(w[2], w[3], 0x7362);
                    mma_f16(part[0], p[step], codes_half2(a01, 0x4140u), codes_half2(b01, 0x4140u));
                    mma_f16(part[1], p[step], codes_half2(a01, 0x4342u), codes_half2(b01, 0x4342u));
                    mma_f16(part[2], p[step], codes_half2(a23, 0x4140u), codes_half2(b23, 0x4140u));
                    mma_f16(part[3], p[step], codes_half2(a23, 0x4342u), codes_half2(b23, 0x4342u));
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * c + n][e] = fmaf(o[4 * c + n][e], old, part[n][e]);
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
            part[16 + gq * D + 2 * tq * (D / 8) + j] = o[j][0] + o[j][2];
            part[16 + gq * D + (2 * tq + 1) * (D / 8) + j] = o[j][1] + o[j][3];
        }
        __syncthreads();
        const bool split = p0 > 0 || p1 < held;
        const int64_t mine_part = ((2 * (int64_t)range + (p0 > 0 ? 0 : 1)) * row_blocks + row_block) * C::kPart;
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
            if (split) {
                float* to = parts + mine_part;
                if (d == 0) {
                    to[r] = top;
                    to[8 + r] = total;
                }
                to[16 + item] = sum;
            } else if (r < rows) {
                const int t = (first_row + r) / g.group, hq = (first_row + r) - t * g.group;
                g.out[(row0 + t) * (int64_t)g.heads * D + (int64_t)(h * g.group + hq) * D + d] = total == 0.0f ? 0.0f : sum / total;
            }
        }
        if (split) {
            // The last block to arrive joins the segment's parts, in block order.
            const int64_t i0 = ((start + 1) * shares - 1) / units, i1 = ((start + held) * shares - 1) / units;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                uint32_t* arrived = arrivals + i0 * row_blocks + row_block;
                last_s = atomicAdd(arrived, 1u) == static_cast<uint32_t>(i1 - i0);
                if (last_s) *arrived = 0;
            }
            __syncthreads();
            if (last_s) {
                __threadfence();
                // Weights of the parts' rows, then their weighted sums, four elements and
                // every kSets-th part per thread.
                const int n = static_cast<int>(i1 - i0) + 1;
                const auto other = [&](int i) {
                    return parts + ((2 * (i0 + i) + (i == 0 ? 1 : 0)) * row_blocks + row_block) * C::kPart;
                };
                float* weight_s = reinterpret_cast<float*>(smem);  // [n][8], then the rows' sums [8]
                for (int r = warp; r < 8; r += C::kWarps) {
                    float top = -INFINITY, total = 0.0f;
                    for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(other(i) + r));
                    top = warp_max_f32(top);
                    for (int i = lane; i < n; i += 32) {
                        const float their = __ldcg(other(i) + r), part_l = __ldcg(other(i) + 8 + r);
                        const float weight = their == -INFINITY ? (part_l == 0.0f ? 0.0f : 1.0f) : ex2(their - top);
                        weight_s[i * 8 + r] = weight;
                        total = fmaf(weight, part_l, total);
                    }
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(~0u, total, d);
                    if (lane == 0) weight_s[n * 8 + r] = total;
                }
                __syncthreads();
                constexpr int kItems = 8 * D / 4, kSets = C::kThreads > kItems ? C::kThreads / kItems : 1;
                float4* set_s = reinterpret_cast<float4*>(weight_s + (n * 8 + 8));
                for (int item = tid % kItems, set = tid / kItems; item < kItems && set < kSets; item += C::kThreads) {
                    const int r = item / (D / 4);
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int i = set; i < n; i += kSets) {
                        const float weight = weight_s[i * 8 + r];
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(other(i) + 16) + item);
                        sum.x = fmaf(weight, v.x, sum.x);
                        sum.y = fmaf(weight, v.y, sum.y);
                        sum.z = fmaf(weight, v.z, sum.z);
                        sum.w = fmaf(weight, v.w, sum.w);
                    }
                    set_s[set * kItems + item] = sum;
                }
                __syncthreads();
                for (int item = tid; item < rows * (D / 4); item += C::kThreads) {
                    const int r = item / (D / 4), d = 4 * (item - r * (D / 4));
                    float4 sum = set_s[item];
#pragma unroll
                    for (int set = 1; set < kSets; ++set) {
                        const float4 v = set_s[set * kItems + item];
                        sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
                    }
                    const float total = weight_s[n * 8 + r];
                    const float4 y = total == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                                   : make_float4(sum.x / total, sum.y / total, sum.z / total, sum.w / total);
                    const int t = (first_row + r) / g.group, hq = (first_row + r) - t * g.group;
                    *reinterpret_cast<float4*>(g.out + (row0 + t) * (int64_t)g.heads * D + (int64_t)(h * g.group + hq) * D + d) = y;
                }
            }
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

// Row blocks of 8, key ranges per row block, and the workspace: the arrival
// counters of every (range, row block), then two partial results for each.
struct SplitShape {
    int64_t row_blocks, ranges;
    size_t counter_bytes, part_bytes;
};

template <int D>
SplitShape split_shape(int64_t max_tokens, int group) {
    SplitShape f;
    f.row_blocks = (max_tokens * group + 7) / 8;
    if (f.row_blocks < 1) f.row_blocks = 1;
    // About one wave of blocks in all; from there on one block per row block,
    // whose requests it walks alone.
    f.ranges = (Split<D>::kBlocks + f.row_blocks - 1) / f.row_blocks;
    f.counter_bytes = (static_cast<size_t>(f.ranges * f.row_blocks) * sizeof(uint32_t) + 255) / 256 * 256;
    f.part_bytes = f.ranges > 1 ? 2 * static_cast<size_t>(f.ranges * f.row_blocks) * Split<D>::kPart * sizeof(float) : 0;
    return f;
}

template <int D>
int run_split(cudaStream_t s, const AttendArgs& g, void* workspace, bool pdl) {
    const SplitShape f = split_shape<D>(g.step.max_tokens, g.group);
    if (f.ranges * f.row_blocks > INT_MAX / 8) {
        set_error("leafq_kv8_attention: max_tokens * group is too large");
        return LEAFQ_ERR_INVALID;
    }
    const int st = allow_smem(reinterpret_cast<const void*>(kv8_attend_split_kernel<D>), Split<D>::kSmem, "leafq_kv8_attention");
    if (st) return st;
    uint32_t* arrivals = static_cast<uint32_t*>(workspace);
    float* parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + f.counter_bytes);
    return launch(kv8_attend_split_kernel<D>, dim3(static_cast<unsigned>(f.ranges * f.row_blocks)), dim3(Split<D>::kThreads),
                  Split<D>::kSmem, s, pdl, "leafq_kv8_attention", g, parts, arrivals, static_cast<int>(f.ranges),
                  static_cast<int>(f.row_blocks));
}

// ----------------------------------------------------------- tile form
// Many query rows (prompts and long chunks): tcgen05.  A block owns 128 query
// rows of one kv head of a request (rows r = token * group + head-in-group),
// walks the keys in tiles, and two blocks share an SM, so that one's MMAs run
// under the other's softmax.  Roles:
//   warps 0-3  softmax: one row per thread (its TMEM lane)
//   warps 4-7  codes to fp16: 16-byte global loads one tile ahead, byte
//              permutes, 128-byte-swizzled shared memory
//   warp 8     MMA issue (kind::f16, fp32 accumulators in TMEM)
// The arithmetic is the split form's: codes exact in fp16, fp32 operands as
// hi + lo halves, the V scale in the exponent.
//   S [128][keys] = Qhi K^T + Qlo K^T   Q and K K-major in shared memory
//   O [128][D]   += Phi V + Plo V       P from TMEM, V as stored (MN-major)
// Each 32 columns of S are replaced in place by 16 columns of P's hi pairs and
// 16 of its lo pairs.  O is rescaled only when a row's maximum grows by more
// than 2^kSlack since its reference was taken: weights then stay below
// 2^(kTileLift + kSlack) < 65504, fp16's largest.
constexpr float kTileLift = 6.0f, kSlack = 8.0f;

template <int D>
struct TileShape {
    static constexpr int kRows = 128;
    static constexpr int kKeys = D <= 64 ? 128 : 64;
    static constexpr int kBlocks = (D + 63) / 64;        // 64-element (128-byte) column blocks
    static constexpr int kStages = D <= 64 ? 2 : 1;      // of K and of V
    static constexpr int kGroups = kKeys / 16;           // of keys that share a page for certain
    static constexpr int kInfo = 4;                      // ring of the groups' scales
    static constexpr int kQBytes = kBlocks * kRows * 128;
    static constexpr int kKvBytes = kBlocks * kKeys * 128;
    static constexpr int kThreads = 9 * 32;
    static constexpr int kPieces = kKeys * D / 16 / 128; // 16-byte pieces of a K (or V) tile per converting thread
    static constexpr int kOutCols = kBlocks * 64;        // O columns (those past D are not read)
    static constexpr uint32_t kTmemCols = 256;
    static constexpr size_t kSmem = 1024 + 2 * kQBytes + 2 * kStages * kKvBytes + kInfo * kGroups * 16 + kRows * 4 + 256;
    static_assert(kKeys + kOutCols <= 256, "two blocks share the SM's 512 TMEM columns");
    static_assert(2 * kQBytes >= kRows * D * 4, "the output leaves through Q's shared memory");
};

// Bounded wait that other requests' range errors do not end.
__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long start = global_timer_ns();
    for (uint32_t spins = 1;; ++spins) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spins & 255u) == 0u && global_timer_ns() - start > wait_limit_ns()) {
            record_device_error(kSiteKv8Tile);
            return false;
        }
    }
}

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// The A operand from tensor memory: two fp16 per 32-bit column.
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor for kind::f16: fp32 accumulator (1) in [4,6), fp16 A
// and B (0), B MN-major (bit 16) or K-major, N >> 3 in [17,23), M >> 4 in [24,29).
__host__ __device__ constexpr uint32_t umma_idesc_f16(uint32_t m, uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(TileShape<D>::kThreads, 2) kv8_attend_tile_kernel(const AttendArgs g, int row_tiles) {
    using C = TileShape<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* q_hi = smem;
    uint8_t* q_lo = q_hi + C::kQBytes;
    uint8_t* k_tiles = q_lo + C::kQBytes;
    uint8_t* v_tiles = k_tiles + C::kStages * C::kKvBytes;
    float4* info = reinterpret_cast<float4*>(v_tiles + C::kStages * C::kKvBytes);  // [kInfo][kGroups]: ks, log2 vs, 1 / vs
    float* factor_s = reinterpret_cast<float*>(info + C::kInfo * C::kGroups);
    uint64_t* k_full = reinterpret_cast<uint64_t*>(factor_s + C::kRows);
    uint64_t* k_empty = k_full + C::kStages;
    uint64_t* v_full = k_empty + C::kStages;
    uint64_t* v_empty = v_full + C::kStages;
    uint64_t* s_full = v_empty + C::kStages;
    uint64_t* p_full = s_full + 1;
    uint64_t* o_full = p_full + 1;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(o_full + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_dependency_wait();
    grid_launch_dependents();

    // Work item, the rows that see most keys first.  Request s may have row
    // tiles floor(token_offsets[s] * group / 128) + s and on: enough of them.
    const int item = row_tiles - 1 - blockIdx.x / g.cache.kv_heads;
    const int h = blockIdx.x % g.cache.kv_heads;
    const int requests = g.step.requests;
    int s = 0;
    for (int n = requests; n > 1;) {
        const int step = (n + 31) / 32, at = s + lane * step;
        const bool below = lane * step < n && ((int64_t)g.step.token_offsets[at] * g.group >> 7) + at <= item;
        const int hit = max(__popc(__ballot_sync(~0u, below)) - 1, 0);
        s += hit * step;
        n = min(step, n - hit * step);
    }
    const int64_t row0 = max64(0, g.step.token_offsets[s]);
    const int new_rows = static_cast<int>(
        max64(0, min64(min64(g.step.token_offsets[s + 1], g.step.tokens) - row0, INT_MAX / g.group)) * g.group);
    const int64_t tile_index = item - ((row0 * g.group >> 7) + s);
    if (tile_index < 0 || tile_index * C::kRows >= new_rows) return;
    const int first_row = static_cast<int>(tile_index) * C::kRows;
    const int rows = min(C::kRows, new_rows - first_row);
    const int context = g.step.context[s];
    const int64_t held = min64(g.step.page_offsets[s + 1] - g.step.page_offsets[s], g.step.max_pages);
    const int keys = static_cast<int>(max64(0, min64(min64(held << g.shift, g.step.lengths[s]),
                                                     (int64_t)context + (first_row + rows - 1) / g.group + 1)));
    const int tiles = (keys + C::kKeys - 1) / C::kKeys;

    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(s_full, 1);
        mbar_init(p_full, 4);
        mbar_init(o_full, 1);
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(tmem_holder, C::kTmemCols);
        tmem_relinquish();
    } else {
        // The rows: D / 8 lanes per row, eight values each, rotated, scaled by
        // the row's power of two, split, stored swizzled (warps 0-7).
        constexpr int kLanes = D / 8;  // 4, 8, 12, 16: a row's lanes are in one warp
        constexpr int kRowsAtOnce = 32 / kLanes;
        const int sub = lane / kLanes, j = lane - sub * kLanes;
        for (int base = warp * kRowsAtOnce; base < C::kRows; base += 8 * kRowsAtOnce) {
            const int r = base + sub;
            const bool live = sub < kRowsAtOnce && r < C::kRows;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
            int at = 4 * j, to = at + D / 2;
            if (live && r < rows) {
                const int t = (first_row + r) / g.group, hq = (first_row + r) - t * g.group;
                int64_t pos = (int64_t)context + t;
                if (g.rotary > 0 && (pos < 0 || pos >= g.table_rows)) {
                    if (j == 0) record_device_error(kSiteKv8Range);
                    pos = 0;
                }
                query_item<D>(g, g.q + (row0 + t) * g.q_stride + (int64_t)(h * g.group + hq) * D, j, pos, at, to, a, b);
            }
            uint32_t largest = 0;
            const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) largest = max(largest, __float_as_uint(v[e]) & 0x7fffffffu);
            if constexpr (kLanes == 12) {
                uint32_t all = 0;
#pragma unroll
                for (int e = 0; e < kLanes; ++e) all = max(all, __shfl_sync(~0u, largest, min(sub * kLanes + e, 31)));
                largest = all;
            } else {
#pragma unroll
                for (int d = kLanes / 2; d > 0; d >>= 1) largest = max(largest, __shfl_xor_sync(~0u, largest, d));
            }
            float up, down;
            row_power(largest, up, down);
            if (live) {
                if (j == 0) factor_s[r] = down * g.scale * kLog2e;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = half == 0 ? at : to;
                    const float x0 = v[4 * half] * up, x1 = v[4 * half + 1] * up, x2 = v[4 * half + 2] * up, x3 = v[4 * half + 3] * up;
                    uint2 hi, lo;
                    hi.x = half2_bits(x0, x1);
                    hi.y = half2_bits(x2, x3);
                    const __half2 h01 = *reinterpret_cast<const __half2*>(&hi.x), h23 = *reinterpret_cast<const __half2*>(&hi.y);
                    lo.x = half2_bits(x0 - __low2float(h01), x1 - __high2float(h01));
                    lo.y = half2_bits(x2 - __low2float(h23), x3 - __high2float(h23));
                    const int offset = (d >> 6) * (C::kRows * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 4) * 2;
                    *reinterpret_cast<uint2*>(q_hi + offset) = hi;
                    *reinterpret_cast<uint2*>(q_lo + offset) = lo;
                }
            }
        }
        fence_proxy_async_smem();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_holder;
    const uint32_t s_tmem = tmem, o_tmem = tmem + C::kKeys;

    if (warp < 4) {
        // ------------------------------------------------------- softmax
        const int r = tid;
        const int64_t pos = (int64_t)context + (first_row + r) / g.group;
        const bool seen = r < rows && pos >= 0 && (g.rotary == 0 || pos < g.table_rows);
        const int limit = seen ? static_cast<int>(min64(keys, pos + 1)) : 0;
        const float factor = factor_s[r];
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < tiles && ok; ++j) {
            ok = __all_sync(~0u, tile_wait(s_full, j & 1));
            if (!ok) break;
            tcgen05_fence_after();
            const float4* scales = info + (j % C::kInfo) * C::kGroups;
            const int visible = limit - j * C::kKeys;  // columns of this tile that the row sees
            const bool whole = __all_sync(~0u, visible >= C::kKeys);
            float top = -INFINITY;
            uint32_t x[32];
#pragma unroll
            for (int c = 0; c < C::kKeys / 32; ++c) {
                tmem_ld_32x32b_x32(s_tmem + lanes + 32 * c, x);
                tmem_wait_ld();
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e >= visible) x[e] = 0xff800000u;
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float most = __uint_as_float(x[16 * half]);
#pragma unroll
                    for (int e = 1; e < 16; ++e) most = fmaxf(most, __uint_as_float(x[16 * half + e]));
                    const float4 scale = scales[2 * c + half];
                    // A column that is not seen stays -inf whatever the scale.
                    const float value = fmaf(most, scale.x * factor, scale.y);
                    top = fmaxf(top, most == -INFINITY ? most : value);
                }
            }
            if (j == 0) {
                m = top;
            } else if (__any_sync(~0u, top > m + kSlack)) {
                // PV of the tile before has completed with this tile's S.
                const float grown = top > m + kSlack ? top : m;
                const float old = m == -INFINITY ? 0.0f : ex2(m - grown);
                m = grown;
                l *= old;
#pragma unroll
                for (int c = 0; c < C::kOutCols / 32; ++c) {
                    tmem_ld_32x32b_x32(o_tmem + lanes + 32 * c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * old);
                    tmem_st_32x32b_x32(o_tmem + lanes + 32 * c, x);
                }
            }
            const float shift = m == -INFINITY ? 0.0f : m - kTileLift;
#pragma unroll
            for (int c = 0; c < C::kKeys / 32; ++c) {
                tmem_ld_32x32b_x32(s_tmem + lanes + 32 * c, x);
                tmem_wait_ld();
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e >= visible) x[e] = 0xff800000u;
                }
                uint32_t p[32];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float4 scale = scales[2 * c + half];
                    const float a = scale.x * factor, b = scale.y - shift;
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float x0 = __uint_as_float(x[16 * half + e]), x1 = __uint_as_float(x[16 * half + e + 1]);
                        float w0 = ex2(fmaf(x0, a, b)), w1 = ex2(fmaf(x1, a, b));
                        if (!whole) {  // -inf times a scale of zero is no number
                            w0 = 32 * c + 16 * half + e >= visible ? 0.0f : w0;
                            w1 = 32 * c + 16 * half + e + 1 >= visible ? 0.0f : w1;
                        }
                        sum += w0;
                        sum += w1;
                        const float h0 = __uint_as_float(__float_as_uint(w0) & 0xffffe000u);
                        const float h1 = __uint_as_float(__float_as_uint(w1) & 0xffffe000u);
                        p[8 * half + e / 2] = half2_bits(h0, h1);
                        p[16 + 8 * half + e / 2] = half2_bits(w0 - h0, w1 - h1);
                    }
                    l = fmaf(sum, scale.z, l);
                }
                tmem_st_32x32b_x32(s_tmem + lanes + 32 * c, p);
            }
            tmem_wait_st();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        if (ok && tiles > 0) tile_wait(o_full, 0);
        __syncwarp();
        tcgen05_fence_after();
        // Out through shared memory (Q's, no longer read): whole rows per store.
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* stage = smem + warp * (32 * D * 4);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            uint32_t x[32];
            if (tiles > 0) {
                tmem_ld_32x32b_x32(o_tmem + lanes + 32 * c, x);
                tmem_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (tiles > 0 && l != 0.0f)
                    y = make_float4(__uint_as_float(x[e]) * inverse, __uint_as_float(x[e + 1]) * inverse,
                                    __uint_as_float(x[e + 2]) * inverse, __uint_as_float(x[e + 3]) * inverse);
                const int piece = 8 * c + e / 4;  // of the row's D / 4
                *reinterpret_cast<float4*>(stage + lane * (D * 4) + ((piece ^ (lane & 7)) << 4)) = y;
            }
        }
        __syncwarp();
        for (int i = lane; i < 32 * (D / 4); i += 32) {
            const int rr = i / (D / 4), piece = i - rr * (D / 4);
            const int row = warp * 32 + rr;
            if (row >= rows) break;
            const float4 y = *reinterpret_cast<const float4*>(stage + rr * (D * 4) + ((piece ^ (rr & 7)) << 4));
            const int t = (first_row + row) / g.group, hq = (first_row + row) - t * g.group;
            *reinterpret_cast<float4*>(g.out + (row0 + t) * (int64_t)g.heads * D + (int64_t)(h * g.group + hq) * D + 4 * piece) = y;
        }
    } else if (warp < 8) {
        // ---------------------------------------------- codes to fp16
        const int ct = tid - 128;
        constexpr int kRowPieces = D / 16;
        const int32_t* table = g.step.table + (int64_t)s * g.step.max_pages;
        const int page = 1 << g.shift;
        // The page of this thread's piece n of tile j, -1 where there is no key.
        const auto page_of = [&](int j, int n) {
            const int key = j * C::kKeys + (n * 128 + ct) / kRowPieces;
            return key < keys ? table[key >> g.shift] : INT_MIN;
        };
        const auto fetch = [&](int j, const int32_t (&ids)[C::kPieces], const int8_t* codes, uint4 (&w)[C::kPieces]) {
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) {
                const int row = (n * 128 + ct) / kRowPieces, cc = (n * 128 + ct) % kRowPieces;
                const int key = j * C::kKeys + row;
                w[n] = make_uint4(0u, 0u, 0u, 0u);
                if (ids[n] >= 0 && ids[n] < g.cache.pages)
                    w[n] = __ldg(reinterpret_cast<const uint4*>(
                        codes + ((((int64_t)ids[n] * g.cache.kv_heads + h) << g.shift) + (key & (page - 1))) * D + cc * 16));
            }
        };
        const auto convert = [&](const uint4 (&w)[C::kPieces], uint8_t* tile) {
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) {
                const int row = (n * 128 + ct) / kRowPieces, cc = (n * 128 + ct) % kRowPieces;
                const uint32_t b[4] = {w[n].x ^ 0x80808080u, w[n].y ^ 0x80808080u, w[n].z ^ 0x80808080u, w[n].w ^ 0x80808080u};
                uint8_t* line = tile + (cc >> 2) * (C::kKeys * 128) + row * 128;
                const int chunk = (cc & 3) * 2;
                *reinterpret_cast<uint4*>(line + ((chunk ^ (row & 7)) << 4)) =
                    make_uint4(codes_half2(b[0], 0x4140u), codes_half2(b[0], 0x4342u), codes_half2(b[1], 0x4140u), codes_half2(b[1], 0x4342u));
                *reinterpret_cast<uint4*>(line + (((chunk + 1) ^ (row & 7)) << 4)) =
                    make_uint4(codes_half2(b[2], 0x4140u), codes_half2(b[2], 0x4342u), codes_half2(b[3], 0x4140u), codes_half2(b[3], 0x4342u));
            }
        };
        int32_t ids[C::kPieces], next_ids[C::kPieces];
        uint4 k[C::kPieces], v[C::kPieces];
        const auto scales_of = [&](int j) {  // of 16-key group ct, in the first lanes
            float4 f = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);  // hides the group
            const int key = j * C::kKeys + 16 * ct;
            if (ct < C::kGroups && key < keys) {
                const int32_t id = table[key >> g.shift];
                if (id >= 0 && id < g.cache.pages) {
                    const int64_t at = (int64_t)id * g.cache.kv_heads + h;
                    const float vs = __ldg(g.cache.v_scales + at);
                    // A page of zeros counts in the sum as any other.
                    f = vs == 0.0f ? make_float4(0.0f, -126.0f, 0x1p126f, 0.0f) : make_float4(0.0f, log2f(vs), 1.0f / vs, 0.0f);
                    f.x = __ldg(g.cache.k_scales + at);
                } else {
                    record_device_error(kSiteKv8Range);
                }
            }
            return f;
        };
#pragma unroll
        for (int n = 0; n < C::kPieces; ++n) ids[n] = page_of(0, n);
        fetch(0, ids, g.cache.k_codes, k);
        float4 scale = scales_of(0);
        bool ok = true;
        for (int j = 0; j < tiles && ok; ++j) {
            const int stage = j % C::kStages;
            const uint32_t reuse = ((j / C::kStages) - 1) & 1;
            fetch(j, ids, g.cache.v_codes, v);
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) next_ids[n] = page_of(j + 1, n);
            if (j >= C::kStages) ok = __all_sync(~0u, tile_wait(&k_empty[stage], reuse));
            if (!ok) break;
            convert(k, k_tiles + stage * C::kKvBytes);
            if (ct < C::kGroups) info[(j % C::kInfo) * C::kGroups + ct] = scale;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[stage]);
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) ids[n] = next_ids[n];
            if (j + 1 < tiles) {
                fetch(j + 1, ids, g.cache.k_codes, k);
                scale = scales_of(j + 1);
            }
            if (j >= C::kStages) ok = __all_sync(~0u, tile_wait(&v_empty[stage], reuse));
            if (!ok) break;
            convert(v, v_tiles + stage * C::kKvBytes);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[stage]);
        }
    } else if (tiles > 0 && elect_one_sync()) {
        // ------------------------------------------------------ MMA issue
        constexpr uint32_t s_desc = umma_idesc_f16(C::kRows, C::kKeys, false), o_desc = umma_idesc_f16(C::kRows, C::kOutCols, true);
        const uint32_t qh = smem_u32(q_hi), ql = smem_u32(q_lo), kt = smem_u32(k_tiles), vt = smem_u32(v_tiles);
        const auto scores = [&](int stage) {
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    umma_f16(s_tmem,
                             umma_desc_k_sw128((part == 0 ? qh : ql) + (i >> 2) * (C::kRows * 128)) + 2 * (i & 3),
                             umma_desc_k_sw128(kt + stage * C::kKvBytes + (i >> 2) * (C::kKeys * 128)) + 2 * (i & 3), s_desc,
                             part > 0 || i > 0);
            umma_commit(&k_empty[stage]);
            umma_commit(s_full);
        };
        bool ok = tile_wait(&k_full[0], 0);
        tcgen05_fence_after();
        if (ok) scores(0);
        for (int j = 0; j < tiles && ok; ++j) {
            const int stage = j % C::kStages;
            ok = tile_wait(&v_full[stage], (j / C::kStages) & 1) && tile_wait(p_full, j & 1);
            if (!ok) break;
            tcgen05_fence_after();
#pragma unroll
            for (int i = 0; i < C::kKeys / 16; ++i)
#pragma unroll
                for (int part = 0; part < 2; ++part)
                    umma_f16_ta(o_tmem, s_tmem + (i >> 1) * 32 + part * 16 + (i & 1) * 8,
                                umma_desc_mn_sw128(vt + stage * C::kKvBytes + i * 2048, C::kKeys * 128), o_desc,
                                j > 0 || i > 0 || part > 0);
            umma_commit(&v_empty[stage]);
            if (j + 1 < tiles) {
                const int next = (j + 1) % C::kStages;
                ok = tile_wait(&k_full[next], ((j + 1) / C::kStages) & 1);
                tcgen05_fence_after();
                if (ok) scores(next);
            }
        }
        // Whatever was issued has completed before the block ends.
        umma_commit(o_full);
        tile_wait(o_full, 0);
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 8) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

template <int D>
int run_tile(cudaStream_t s, const AttendArgs& g, bool pdl) {
    const int64_t row_tiles = (g.step.tokens * g.group >> 7) + g.step.requests;
    if (row_tiles * g.cache.kv_heads > INT_MAX) {
        set_error("leafq_kv8_attention: too many rows");
        return LEAFQ_ERR_INVALID;
    }
    const int st = allow_smem(reinterpret_cast<const void*>(kv8_attend_tile_kernel<D>), TileShape<D>::kSmem, "leafq_kv8_attention");
    if (st) return st;
    return launch(kv8_attend_tile_kernel<D>, dim3(static_cast<unsigned>(row_tiles * g.cache.kv_heads)),
                  dim3(TileShape<D>::kThreads), TileShape<D>::kSmem, s, pdl, "leafq_kv8_attention", g,
                  static_cast<int>(row_tiles));
}

// The tile form pads a request's rows to 128: it is the faster one from about
// 32 rows of one request on.
bool takes_tiles(int64_t max_tokens, int group) { return max_tokens * group >= 32; }

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
        !kv8_dim_supported(dim) || takes_tiles(max_tokens, heads / kv_heads))
        return 0;
    return with_dim(dim, [&](auto d) {
        const SplitShape f = split_shape<d()>(max_tokens, heads / kv_heads);
        return f.counter_bytes + f.part_bytes;
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
    AttendArgs g{q, q_stride, cos_table, sin_table, table_rows, *cache, *step, out, scale, heads,
                 heads / cache->kv_heads, rotary_dim, 0};
    while ((1 << g.shift) < cache->page) ++g.shift;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool pdl = (flags & LEAFQ_FLAG_PDL) != 0;
    const bool tiles = takes_tiles(step->max_tokens, g.group);
    return with_dim(cache->dim, [&](auto d) { return tiles ? run_tile<d()>(s, g, pdl) : run_split<d()>(s, g, workspace, pdl); });
}

}  // extern "C"
