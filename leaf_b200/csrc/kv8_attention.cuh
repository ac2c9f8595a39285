// Shared by the paged INT8 cache's plan and append (kv8_cache.cu), the two forms of its
// attention (kv8_attention.cu for few query rows, kv8_tile.cu for many) and its trees of
// drafts (kv8_tree.cu).
#pragma once

#include <cuda_fp16.h>

#include <climits>
#include <cmath>

#include "leafq_device.cuh"
#include "leafq_internal.h"

namespace leafq {

inline int page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }

struct Kv8AttendArgs {
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
    int most_tokens;  // of a request: its rows (tokens * group) fit int32
    // Trees of drafts (leafq_kv8_tree_attention): each row's position, and which of the
    // request's new rows it sees, as bits.  Null for causal attention.
    const int32_t* positions;
    const uint32_t* masks;
    int mask_words;
};

constexpr float kLog2e = 1.4426950408889634f;
// Weights are held as 2^kLift times their value relative to a row's reference,
// so that the second half of a weight's fp16 split stays a normal number far
// below it; twice kHighest is below 65504, fp16's largest.
constexpr float kLift = 6.0f, kHighest = 24576.0f;
// A page's weights carry its V scale's exponent, which their sum takes out again: as
// a factor of up to 2^90, so that the sum of 2^17 keys' weights stays below 2^127.
// Smaller scales count as zero.
constexpr float kLeastScale = 0x1p-90f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// Rotates the pairs of a and b, in the rounding steps of leafq_rotary_append.
__device__ __forceinline__ void kv8_turn(float4& a, float4& b, float4 c, float4 s) {
    const float4 x = a, y = b;
    a = make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(y.x, s.x)), __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(y.y, s.y)),
                    __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(y.z, s.z)), __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(y.w, s.w)));
    b = make_float4(__fadd_rn(__fmul_rn(y.x, c.x), __fmul_rn(x.x, s.x)), __fadd_rn(__fmul_rn(y.y, c.y), __fmul_rn(x.y, s.y)),
                    __fadd_rn(__fmul_rn(y.z, c.z), __fmul_rn(x.z, s.z)), __fadd_rn(__fmul_rn(y.w, c.w), __fmul_rn(x.w, s.w)));
}

// Bit i: whether a tree's row with these mask words sees key `at` + i, the request's new
// keys being numbered from 0 (those before them are cached ones, which every row sees;
// the mask's words end with those of the tree).
__device__ __forceinline__ uint32_t tree_window(const uint32_t* row_mask, int words, int at) {
    if (at <= -32) return ~0u;
    const int w = at >> 5;
    const auto word = [&](int i) { return i < 0 ? ~0u : i < words ? row_mask[i] : 0u; };
    return __funnelshift_r(word(w), word(w + 1), at & 31);
}

// Eight values of a query row, its item j of D / 8: four at `at` and four at
// `to`, a rotation pair's quarters where they are turned (as in the append).
template <int D>
struct QueryItem {
    int at, to;
    bool turned;
    float4 a, b, cos, sin;

    // row: null for a row of zeros.
    __device__ __forceinline__ void load(const Kv8AttendArgs& g, const float* row, int j, int64_t pos) {
        const int half = g.rotary >> 1;
        turned = 4 * j < half;
        at = turned ? 4 * j : 2 * half + 4 * (j - half / 4);
        to = turned ? at + half : at + ((D - 2 * half) >> 1);
        a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row == nullptr) {
            turned = false;
            return;
        }
        a = *reinterpret_cast<const float4*>(row + at);
        b = *reinterpret_cast<const float4*>(row + to);
        if (turned) {
            cos = *reinterpret_cast<const float4*>(g.cos_table + pos * half + at);
            sin = *reinterpret_cast<const float4*>(g.sin_table + pos * half + at);
        }
    }
    __device__ __forceinline__ void turn() {
        if (turned) kv8_turn(a, b, cos, sin);
    }
    __device__ __forceinline__ uint32_t largest() const {  // the magnitude's bits
        uint32_t most = 0;
        for (const float x : {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}) most = max(most, __float_as_uint(x) & 0x7fffffffu);
        return most;
    }
};

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

// The workspace: counters that are zero between calls, in places that do not
// depend on the call's shape, so that calls of all shapes may share it; then the
// parts' results.
constexpr int kSplitCounters = 2560, kTileCounters = kSplitCounters, kTileBlocks = 296;
constexpr size_t kCounterBytes = 16384;
static_assert((kTileCounters + 4 + 4 * (kTileBlocks / 2)) * 4 <= kCounterBytes, "the items that have parts, four counters each");

// Many query rows of a request (kv8_tile.cu), and what its parts take.
size_t kv8_tile_part_bytes(int dim);
int launch_kv8_tiles(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl);
// The same for trees (kv8_tree_tile.cu).
size_t kv8_tree_part_bytes(int dim);
int launch_kv8_tree_tiles(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl);

}  // namespace leafq
