// Causal grouped-query attention over the paged INT8 KV cache
// (include/leafq.h, leafq_kv8_attention).
//
// For the query row (request s, new token t, head h) at position
// p = context[s] + t, over keys j < min(p + 1, lengths[s]):
//   x_j = scale * ks * (q . ck_j)      ks, vs: the scales of key j's page
//   out = sum_j exp(x_j - m) vs cv_j / sum_j exp(x_j - m),  m = max x
// in one pass over the keys: when the maximum grows from m to m', the sums so
// far are multiplied by exp(m - m').
#include <climits>

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

// Element d of a query row, rotated by position p.
__device__ __forceinline__ float rotated(const AttendArgs& g, const float* q, int d, int64_t p) {
    const int half = g.rotary >> 1;
    const float x = q[d];
    if (d >= g.rotary) return x;
    const int j = d < half ? d : d - half;
    const float c = g.cos_table[p * half + j], s = g.sin_table[p * half + j];
    return d < half ? __fsub_rn(__fmul_rn(x, c), __fmul_rn(q[d + half], s))
                    : __fadd_rn(__fmul_rn(x, c), __fmul_rn(q[d - half], s));
}

// One warp per query row, lanes over the head's elements.
template <int D>
__global__ void __launch_bounds__(256) kv8_attend_warp_kernel(const AttendArgs g) {
    constexpr int E = D / 32;
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t row = id / g.heads;
    const int head = static_cast<int>(id - row * g.heads);
    if (row >= g.step.tokens || row >= g.step.token_offsets[g.step.requests]) return;
    int lo = 0, hi = g.step.requests - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (g.step.token_offsets[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    const int64_t pos = (int64_t)g.step.context[lo] + row - g.step.token_offsets[lo];
    const int64_t held = min64(g.step.page_offsets[lo + 1] - g.step.page_offsets[lo], g.step.max_pages) << g.shift;
    int64_t keys = min64(min64(pos + 1, g.step.lengths[lo]), held);
    if (pos < 0 || (g.rotary > 0 && pos >= g.table_rows)) {
        if (lane == 0) record_device_error(kSiteKv8Range);
        keys = 0;
    }
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    const float* src = g.q + row * g.q_stride + (int64_t)head * D;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = keys > 0 ? rotated(g, src, lane * E + e, pos) : 0.0f;
        o[e] = 0.0f;
    }
    const int kvh = head / g.group;
    const int64_t page = int64_t{1} << g.shift;
    const int32_t* table = g.step.table + lo * g.step.max_pages;
    for (int64_t j0 = 0; j0 < keys; j0 += page) {
        const int64_t id_page = table[j0 >> g.shift];
        if (id_page < 0 || id_page >= g.cache.pages) {
            if (lane == 0) record_device_error(kSiteKv8Range);
            continue;
        }
        const int64_t tile = id_page * g.cache.kv_heads + kvh;
        const float ks = g.cache.k_scales[tile] * g.scale, vs = g.cache.v_scales[tile];
        const int8_t* kc = g.cache.k_codes + (tile << g.shift) * D + lane * E;
        const int8_t* vc = g.cache.v_codes + (tile << g.shift) * D + lane * E;
        const int n = static_cast<int>(min64(page, keys - j0));
        for (int j = 0; j < n; ++j) {
            float x = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) x = fmaf(q[e], static_cast<float>(kc[j * D + e]), x);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(~0u, x, d);
            x *= ks;
            const float grown = fmaxf(m, x), old = m == -INFINITY ? 0.0f : expf(m - grown);
            const float p = expf(x - grown);
            m = grown;
            l = l * old + p;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = o[e] * old + p * vs * static_cast<float>(vc[j * D + e]);
        }
    }
    float* dst = g.out + row * (int64_t)g.heads * D + (int64_t)head * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = m == -INFINITY && l == 0.0f ? 0.0f : o[e] / l;
}

template <int D>
int run_warp(cudaStream_t s, const AttendArgs& g, bool pdl) {
    const int64_t rows = g.step.tokens * g.heads;
    return launch(kv8_attend_warp_kernel<D>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, s, pdl,
                  "leafq_kv8_attention", g);
}

}  // namespace
}  // namespace leafq

using namespace leafq;

extern "C" {

size_t leafq_kv8_attention_workspace_bytes(int64_t max_tokens, int heads, int kv_heads, int dim) {
    (void)max_tokens, (void)heads, (void)kv_heads, (void)dim;
    return 0;
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
    (void)workspace, (void)workspace_bytes;
    AttendArgs g{q, q_stride, cos_table, sin_table, table_rows, *cache, *step, out, scale, heads,
                 heads / cache->kv_heads, rotary_dim, 0};
    while ((1 << g.shift) < cache->page) ++g.shift;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool pdl = (flags & LEAFQ_FLAG_PDL) != 0;
    switch (cache->dim) {
        case 32: return run_warp<32>(s, g, pdl);
        case 64: return run_warp<64>(s, g, pdl);
        case 96: return run_warp<96>(s, g, pdl);
        default: return run_warp<128>(s, g, pdl);
    }
}

}  // extern "C"
