// Paged INT8 KV cache: the step plan and the append (include/leafq.h).
//
//   kv8_plan_kernel    block tables and slot map from request lengths
//   kv8_append_kernel  RoPE on the keys, quantisation of keys and values into
//                      their pages, the pages' scales grown where they must
#include <climits>

#include "kv8_attention.cuh"

namespace leafq {
namespace {

// ------------------------------------------------------------------- plan
// Two prefix sums over the requests (new tokens, new pages) decide everything:
// a request's first row, the free pages it takes, whether the pool reaches.
// Every block scans all requests itself, a chunk of blockDim.x (two a thread,
// where there are more requests) at a time with a running carry (8 bytes per request from L2), so that no block waits for
// another; block 0 writes the per-request outputs and the blocks share the
// chunk's tokens.  Four consecutive tokens per thread: one search of the
// chunk's prefix, one page lookup per page, 16-byte stores.  A new page's
// table entry is written by the thread that has the page's first token.
//
// Bound: latency, of the launch, the lengths' load, two barriers per chunk and
// the page lookup behind them.  64 requests of one token each take 4.8 us,
// 2,000 requests with 288,042 new tokens 8.7 us (2.5 MB, 287 GB/s; one request a
// thread, in two chunks, 14.7).
struct PlanArgs {
    const int32_t* context;
    const int32_t* fresh;
    int32_t* table;
    const int32_t* free_pages;
    const int32_t* taken;
    int32_t* lengths;
    int32_t* token_offsets;
    int32_t* page_offsets;
    int32_t* positions;
    int32_t* slots;
    int32_t* taken_after;
    int64_t max_pages, free_count, tokens;
    int requests, shift;  // page = 1 << shift
};

constexpr int kPlanMaxThreads = 1024;

// Inclusive scan over the block of two values at once; total of the block in
// the last argument pair.  Every thread calls it.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t& total_a, int64_t& total_b,
                                            int64_t (*part)[2]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int64_t oa = __shfl_up_sync(~0u, a, d), ob = __shfl_up_sync(~0u, b, d);
        if (lane >= d) {
            a += oa;
            b += ob;
        }
    }
    __syncthreads();  // the previous scan's parts have been read
    if (lane == 31) {
        part[warp][0] = a;
        part[warp][1] = b;
    }
    __syncthreads();
    // Every warp scans the warps' totals for itself.
    int64_t pa = lane < warps ? part[lane][0] : 0, pb = lane < warps ? part[lane][1] : 0;
    const int64_t own_a = pa, own_b = pb;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int64_t oa = __shfl_up_sync(~0u, pa, d), ob = __shfl_up_sync(~0u, pb, d);
        if (lane >= d) {
            pa += oa;
            pb += ob;
        }
    }
    total_a = __shfl_sync(~0u, pa, 31);
    total_b = __shfl_sync(~0u, pb, 31);
    a += __shfl_sync(~0u, pa - own_a, warp);
    b += __shfl_sync(~0u, pb - own_b, warp);
}

// kPer: consecutive requests of a chunk per thread.
template <int kPer>
__global__ void __launch_bounds__(kPlanMaxThreads) kv8_plan_kernel(const PlanArgs g) {
    __shared__ int64_t part[32][2];
    __shared__ int64_t first_s[kPlanMaxThreads * kPer + 1];  // first token of each request of the chunk
    __shared__ int64_t source_s[kPlanMaxThreads * kPer];     // free_pages index of table column 0 (if it were new); LLONG_MIN: refused
    __shared__ int32_t context_s[kPlanMaxThreads * kPer];
    __shared__ long long reached_s;                          // pages granted so far
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, threads = blockDim.x, chunk = threads * kPer;
    const int64_t page = int64_t{1} << g.shift;
    const int64_t taken = *g.taken;
    const bool writer = blockIdx.x == 0;
    if (tid == 0) reached_s = 0;
    int64_t token_base = 0, need_base = 0, page_base = 0;
    int32_t next_c[kPer], next_n[kPer];
    const auto ask = [&](int base) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int r = base + tid * kPer + i;
            next_c[i] = r < g.requests ? g.context[r] : 0;
            next_n[i] = r < g.requests ? g.fresh[r] : 0;
        }
    };
    ask(0);
    for (int base = 0; base < g.requests; base += chunk) {
        int64_t c[kPer], n[kPer], before[kPer], need[kPer];
        bool fits[kPer];
        int64_t tn = 0, tp = 0, chunk_tokens, chunk_pages;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            c[i] = next_c[i];
            n[i] = next_n[i];
            if (c[i] < 0 || n[i] < 0) {
                if (writer) record_device_error(kSiteKv8Range);
                c[i] = max64(c[i], 0);
                n[i] = 0;
            }
            before[i] = (c[i] + page - 1) >> g.shift;
            const int64_t after = (c[i] + n[i] + page - 1) >> g.shift;
            fits[i] = after <= g.max_pages;
            need[i] = fits[i] ? after - before[i] : 0;
            tn += n[i];
            tp += need[i];
        }
        ask(base + chunk);
        const int64_t own_tn = tn, own_tp = tp;
        block_scan2(tn, tp, chunk_tokens, chunk_pages, part);
        int64_t first = token_base + tn - own_tn, upto = need_base + tp - own_tp;  // pages wanted by the requests before
        int64_t length[kPer], held = 0, reached = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            upto += need[i];
            const bool granted = fits[i] && (need[i] == 0 || (taken >= 0 && taken + upto <= g.free_count));
            length[i] = granted ? c[i] + n[i] : c[i];
            const int at = tid * kPer + i;
            first_s[at] = first;
            source_s[at] = granted ? taken + upto - need[i] - before[i] : LLONG_MIN;
            context_s[at] = static_cast<int32_t>(c[i]);
            first += n[i];
            if (granted && need[i] > 0) reached = upto;
        }
        if (tid == threads - 1) first_s[chunk] = first;
        if (writer) {
            // Pages held are bounded by the table's row (a context past it is the caller's error).
            int64_t pages[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                pages[i] = base + tid * kPer + i < g.requests ? min64((length[i] + page - 1) >> g.shift, g.max_pages) : 0;
                held += pages[i];
            }
            const int64_t own_held = held;
            int64_t none = 0, chunk_held, unused, end = token_base + tn - own_tn;
            block_scan2(held, none, chunk_held, unused, part);
            held += page_base - own_held;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int r = base + tid * kPer + i;
                end += n[i];
                held += pages[i];
                if (r < g.requests) {
                    g.lengths[r] = static_cast<int32_t>(length[i]);
                    g.token_offsets[r + 1] = static_cast<int32_t>(min64(end, g.tokens));
                    g.page_offsets[r + 1] = static_cast<int32_t>(min64(held, INT_MAX));
                }
            }
            if (reached > 0) atomicMax(&reached_s, static_cast<long long>(reached));
            page_base += chunk_held;
        }
        __syncthreads();
        // Tokens [t0, t1) of the chunk, in aligned groups of four.
        const int64_t t0 = token_base, t1 = min64(token_base + chunk_tokens, g.tokens);
        const int count = min(chunk, g.requests - base);
        for (int64_t u = t0 / 4 + (int64_t)blockIdx.x * threads + tid; u * 4 < t1; u += (int64_t)gridDim.x * threads) {
            const int64_t begin = max64(u * 4, t0), end = min64(u * 4 + 4, t1);
            int lo = 0, hi = count - 1;  // the last request whose first token is at most begin
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (first_s[mid] <= begin) lo = mid;
                else hi = mid - 1;
            }
            int32_t pos4[4], slot4[4];
            int64_t known = -1, id = -1;  // the last page looked up
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t t = u * 4 + i;
                pos4[i] = 0;
                slot4[i] = -1;
                if (t < begin || t >= end) continue;
                while (lo + 1 < count && first_s[lo + 1] <= t) {
                    ++lo;
                    known = -1;
                }
                const int64_t c_r = context_s[lo], p = c_r + (t - first_s[lo]), column = p >> g.shift;
                pos4[i] = static_cast<int32_t>(p);
                if (source_s[lo] == LLONG_MIN) continue;
                if (column != known) {
                    known = column;
                    int32_t* entry = g.table + (int64_t)(base + lo) * g.max_pages + column;
                    if (column >= (c_r + page - 1) >> g.shift) {
                        id = g.free_pages[source_s[lo] + column];
                        if ((p & (page - 1)) == 0) *entry = static_cast<int32_t>(id);
                    } else {
                        id = *entry;
                    }
                }
                slot4[i] = static_cast<int32_t>(id * page + (p & (page - 1)));
            }
            if (begin == u * 4 && end == u * 4 + 4) {
                *reinterpret_cast<int4*>(g.positions + u * 4) = make_int4(pos4[0], pos4[1], pos4[2], pos4[3]);
                *reinterpret_cast<int4*>(g.slots + u * 4) = make_int4(slot4[0], slot4[1], slot4[2], slot4[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (u * 4 + i >= begin && u * 4 + i < end) {
                        g.positions[u * 4 + i] = pos4[i];
                        g.slots[u * 4 + i] = slot4[i];
                    }
            }
        }
        token_base += chunk_tokens;
        need_base += chunk_pages;
        __syncthreads();  // the chunk's arrays are free
    }
    for (int64_t t = token_base + (int64_t)blockIdx.x * threads + tid; t < g.tokens; t += (int64_t)gridDim.x * threads) {
        g.positions[t] = 0;
        g.slots[t] = -1;
    }
    if (writer && tid == 0) {
        g.token_offsets[0] = 0;
        g.page_offsets[0] = 0;
        *g.taken_after = static_cast<int32_t>(taken + reached_s);
        if (token_base > g.tokens) record_device_error(kSiteKv8Range);
    }
}

// ----------------------------------------------------------------- append
// A run is the new rows of one page: consecutive rows with consecutive slots
// inside the page.  A block owns the runs that start among its `span` rows,
// for one kv head, of the keys (blockIdx.z 0) or the values (1).  One pass:
// the run's rows (rotated) stay in registers between the absmax and the
// codes, kAppendItems items of 8 values per thread, blockDim.x * kAppendItems
// items = page * dim / 8.  An item is the two quarters of a rotation pair:
// values a .. a+3 and b .. b+3 with b = a + rotary / 2 (behind the rotated
// part, pairs of the remaining half).  The absmax is a maximum over bit
// patterns, which is exact, order-free and lets a NaN through.
//
// Bound: HBM, 5 bytes a value (4 read, 1 written), once the calls are large; the
// chain slots -> rows -> absmax -> codes is one round trip after another and is
// hidden only by the other blocks of the SM.  4 heads of 64: a decode step of 64
// rows 2.7 us; 64 prompts of 512 tokens, 84 MB, 25.9 us (3.2 TB/s, half of the
// copy rate).  8 heads of 128, 37 requests with 4,737 new tokens in pages of 16,
// 48.5 MB, 17.7 us.
constexpr int kAppendItems = 4;

struct AppendArgs {
    const float* rows[2];
    int64_t stride[2];
    int8_t* codes[2];
    float* scales[2];
    const int32_t* positions;
    const int32_t* slots;
    const float* cos_table;
    const float* sin_table;
    int64_t table_rows, tokens, pages;
    int shift, kv_heads, rotary, span;
};

// Four codes: the products, rounded, plus 1.5 * 2^23, which rounds them to whole
// numbers (half to even) in the low bits, two's complement.  |x| is at most the
// absmax that the multiplier comes from, so no product passes 127.5.  (Scalar
// operations: the paired mul.rn and add.rn came out as one fused rounding.)
__device__ __forceinline__ uint32_t pack_codes(float4 x, float multiplier) {
    const float a = __fadd_rn(__fmul_rn(x.x, multiplier), 12582912.0f), b = __fadd_rn(__fmul_rn(x.y, multiplier), 12582912.0f);
    const float c = __fadd_rn(__fmul_rn(x.z, multiplier), 12582912.0f), d = __fadd_rn(__fmul_rn(x.w, multiplier), 12582912.0f);
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                       __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}

// max |x| that keeps a NaN.
__device__ __forceinline__ float largest_of(float m, float4 v) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v.x)));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v.y)));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v.z)));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v.w)));
    return m;
}

template <int D>
__global__ void __launch_bounds__(512, 2) kv8_append_kernel(const AppendArgs g) {
    __shared__ int32_t slots_s[256], positions_s[256];  // of the span's rows and a page's worth behind them
    __shared__ uint32_t starts_s[4];   // rows of the span that start a run
    __shared__ uint32_t follow_s[16];  // rows behind a start that belong to its run
    __shared__ uint32_t largest_s[16];
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int head = blockIdx.y, which = blockIdx.z;
    const int page = 1 << g.shift;
    const int64_t row0 = (int64_t)blockIdx.x * g.span;
    const int64_t pool = g.pages << g.shift;
    const int32_t before_row0 = row0 > 0 ? g.slots[row0 - 1] : -2;
    for (int i = tid; i < g.span + page; i += blockDim.x) {
        const bool there = row0 + i < g.tokens;
        slots_s[i] = there ? g.slots[row0 + i] : -1;
        positions_s[i] = there && g.rotary > 0 && which == 0 ? g.positions[row0 + i] : 0;
    }
    __syncthreads();
    // span <= page <= blockDim.x: one row per thread.
    bool start = false;
    if (tid < g.span && row0 + tid < g.tokens) {
        const int32_t slot = slots_s[tid];
        if (slot >= 0 && slot < pool) {
            start = (slot & (page - 1)) == 0 || (tid == 0 ? before_row0 : slots_s[tid - 1]) != slot - 1;
        } else if (slot != -1 && head == 0 && which == 0) {
            record_device_error(kSiteKv8Range);
        }
    }
    const uint32_t ballot = __ballot_sync(~0u, start);
    if (lane == 0 && warp < 4) starts_s[warp] = ballot;
    __syncthreads();
    constexpr int per_row = D / 8;  // items
    const bool rotate = which == 0 && g.rotary > 0;
    const int half = rotate ? g.rotary >> 1 : 0;
    for (int word = 0; word < 4 && word * 32 < g.span; ++word) {
        for (uint32_t left = starts_s[word]; left != 0; left &= left - 1) {
            const int at_row = word * 32 + __ffs(left) - 1;
            const int64_t row = row0 + at_row, slot = slots_s[at_row];
            const int first = static_cast<int>(slot & (page - 1));
            // Rows of the run: until the page ends or the slots stop following.
            const bool follows = tid < page - first && slots_s[at_row + tid] == slot + tid;
            const uint32_t mask = __ballot_sync(~0u, follows);
            if (lane == 0) follow_s[warp] = mask;
            __syncthreads();
            int n = 0;
            for (int w = 0; w * 32 < page; ++w) {
                const uint32_t gap = ~follow_s[w];
                if (gap != 0) {
                    n += __ffs(gap) - 1;
                    break;
                }
                n += 32;
            }
            const int64_t tile = (slot >> g.shift) * g.kv_heads + head;
            float* scale_at = g.scales[which] + tile;
            const float before = *scale_at;
            float4 a[kAppendItems], b[kAppendItems];
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < kAppendItems; ++i) {
                const int item = tid + i * blockDim.x, r = item / per_row, j = item - r * per_row;
                a[i] = b[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (r >= n) continue;
                const float* src = g.rows[which] + (row + r) * g.stride[which] + (int64_t)head * D;
                const bool turned = 4 * j < half;
                const int at = turned ? 4 * j : 2 * half + 4 * (j - half / 4);
                const int to = turned ? at + half : at + ((D - 2 * half) >> 1);
                a[i] = *reinterpret_cast<const float4*>(src + at);
                b[i] = *reinterpret_cast<const float4*>(src + to);
                if (turned) {
                    int64_t pos = positions_s[at_row + r];
                    if (pos < 0 || pos >= g.table_rows) {
                        if (j == 0 && head == 0) record_device_error(kSiteKv8Range);
                        pos = 0;
                    }
                    kv8_turn(a[i], b[i], *reinterpret_cast<const float4*>(g.cos_table + pos * half + at),
                             *reinterpret_cast<const float4*>(g.sin_table + pos * half + at));
                }
                most = largest_of(largest_of(most, a[i]), b[i]);
            }
            uint32_t largest = __reduce_max_sync(~0u, __float_as_uint(most));
            if (lane == 0) largest_s[warp] = largest;
            __syncthreads();  // also: every thread has read the old scale
            for (int w = 0; w < warps; ++w) largest = max(largest, largest_s[w]);
            float need = __fdiv_rn(__uint_as_float(largest), 127.0f);
            if (need < 1e-12f) need = 1e-12f;  // keeps a NaN
            const float scale = first > 0 && !(need > before) && !isnan(need) ? before : need;
            int8_t* codes = g.codes[which] + ((tile << g.shift) * D);
            if (first > 0 && scale != before) {
                // The page's older codes, rounded to the grown scale.
                const float ratio = __fdiv_rn(before, scale);
                for (int i = tid; i < first * D / 4; i += blockDim.x) {
                    uint32_t* at = reinterpret_cast<uint32_t*>(codes) + i;
                    const uint32_t old = *at;
                    *at = pack_codes(make_float4(static_cast<int8_t>(old), static_cast<int8_t>(old >> 8),
                                                 static_cast<int8_t>(old >> 16), static_cast<int8_t>(old >> 24)), ratio);
                }
            }
            const float multiplier = __fdiv_rn(1.0f, scale);
#pragma unroll
            for (int i = 0; i < kAppendItems; ++i) {
                const int item = tid + i * blockDim.x, r = item / per_row, j = item - r * per_row;
                if (r >= n) continue;
                const bool turned = 4 * j < half;
                const int at = turned ? 4 * j : 2 * half + 4 * (j - half / 4);
                const int to = turned ? at + half : at + ((D - 2 * half) >> 1);
                int8_t* dst = codes + (int64_t)(first + r) * D;
                *reinterpret_cast<uint32_t*>(dst + at) = pack_codes(a[i], multiplier);
                *reinterpret_cast<uint32_t*>(dst + to) = pack_codes(b[i], multiplier);
            }
            if (tid == 0) *scale_at = scale;
            __syncthreads();  // follow_s and largest_s are free
        }
    }
}

}  // namespace

bool kv8_cache_valid(const leafq_kv8_cache* c, const char* what) {
    if (!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || c->pages <= 0 || c->kv_heads <= 0 ||
        c->kv_heads > 65535 || page_shift(c->page) < 0 || c->pages > INT_MAX / c->page) {
        set_error(std::string(what) + ": invalid cache (pages of 16, 32, 64 or 128 tokens, slots within int32)");
        return false;
    }
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes)) {
        set_error(std::string(what) + ": cache codes must be 16-byte aligned");
        return false;
    }
    return true;
}

bool kv8_rope_valid(int dim, int rotary_dim, const float* cos_table, const float* sin_table, int64_t table_rows,
                    const char* what) {
    if (!cos_table && !sin_table && rotary_dim == 0) return true;
    if (!cos_table || !sin_table || rotary_dim <= 0 || rotary_dim > dim || rotary_dim % 8 != 0 || table_rows <= 0 ||
        !aligned16(cos_table) || !aligned16(sin_table)) {
        set_error(std::string(what) +
                  ": rotation needs two 16-byte aligned tables and rotary_dim a multiple of 8 within the head");
        return false;
    }
    return true;
}

}  // namespace leafq

using namespace leafq;

extern "C" {

int leafq_kv8_plan(void* stream, const int32_t* context, const int32_t* new_tokens, int requests, int32_t* table,
                   int64_t max_pages, const int32_t* free_pages, int64_t free_count, const int32_t* taken, int page,
                   int64_t tokens, int32_t* lengths, int32_t* token_offsets, int32_t* page_offsets,
                   int32_t* positions, int32_t* slots, int32_t* taken_after, uint32_t flags) {
    clear_error();
    const int shift = page_shift(page);
    if (requests < 0 || max_pages < 0 || free_count < 0 || tokens < 0 || shift < 0) {
        set_error("leafq_kv8_plan: negative size, or a page that is not 16, 32, 64 or 128 tokens");
        return LEAFQ_ERR_INVALID;
    }
    if (max_pages > INT_MAX / page || tokens > INT_MAX || free_count > INT_MAX) {
        set_error("leafq_kv8_plan: lengths, tokens and pages must fit int32");
        return LEAFQ_ERR_INVALID;
    }
    if (!token_offsets || !page_offsets || !taken || !taken_after ||
        (requests > 0 && (!context || !new_tokens || !lengths || (max_pages > 0 && !table))) ||
        (tokens > 0 && (!positions || !slots)) || (free_count > 0 && !free_pages)) {
        set_error("leafq_kv8_plan: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    if (!aligned16(positions) || !aligned16(slots)) {
        set_error("leafq_kv8_plan: positions and slots must be 16-byte aligned");
        return LEAFQ_ERR_INVALID;
    }
    // Every block reads the inputs while block 0 writes the requests' outputs.
    const Span inputs[] = {{context, requests}, {new_tokens, requests}, {table, requests * max_pages}, {free_pages, free_count}, {taken, 1}};
    const Span outputs[] = {{lengths, requests}, {token_offsets, requests + 1}, {page_offsets, requests + 1}, {positions, tokens},
                            {slots, tokens}, {taken_after, 1}};
    for (const Span& out : outputs)
        for (const Span& in : inputs)
            if (out.overlaps(in)) {
                set_error("leafq_kv8_plan: outputs must not overlap the inputs (taken_after and taken, lengths and context, ...)");
                return LEAFQ_ERR_INVALID;
            }
    PlanArgs g{context, new_tokens, table, free_pages, taken, lengths, token_offsets, page_offsets, positions, slots,
               taken_after, max_pages, free_count, tokens, requests, shift};
    // One block for a decode step; with many tokens one block per 4096 of them.
    const int threads = requests <= 256 && tokens <= 1024 ? 256 : kPlanMaxThreads;
    int64_t blocks = (tokens + 4 * threads - 1) / (4 * threads);
    blocks = blocks < 1 ? 1 : blocks > sm_count() ? sm_count() : blocks;
    return launch(requests > threads ? kv8_plan_kernel<2> : kv8_plan_kernel<1>, dim3(static_cast<unsigned>(blocks)), dim3(threads), 0,
                  static_cast<cudaStream_t>(stream), (flags & LEAFQ_FLAG_PDL) != 0, "leafq_kv8_plan", g);
}

int leafq_kv8_append(void* stream, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                     int64_t tokens, const int32_t* positions, const int32_t* slots, int rotary_dim,
                     const float* cos_table, const float* sin_table, int64_t table_rows,
                     const leafq_kv8_cache* cache, uint32_t flags) {
    clear_error();
    if (!kv8_cache_valid(cache, "leafq_kv8_append")) return LEAFQ_ERR_INVALID;
    if (!kv8_dim_supported(cache->dim)) {
        set_error("leafq_kv8_append: head sizes are 32, 64, 96 and 128");
        return LEAFQ_ERR_UNSUPPORTED;
    }
    if (!kv8_rope_valid(cache->dim, rotary_dim, cos_table, sin_table, table_rows, "leafq_kv8_append"))
        return LEAFQ_ERR_INVALID;
    const int64_t width = (int64_t)cache->kv_heads * cache->dim;
    if (tokens < 0 || tokens > INT_MAX) {
        set_error("leafq_kv8_append: tokens must be between 0 and 2^31 - 1");
        return LEAFQ_ERR_INVALID;
    }
    if (tokens == 0) return LEAFQ_OK;
    if (!k || !v || !slots || (rotary_dim > 0 && !positions)) {
        set_error("leafq_kv8_append: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    if ((tokens > 1 && (k_stride < width || v_stride < width)) || k_stride % 4 != 0 || v_stride % 4 != 0 ||
        !aligned16(k) || !aligned16(v)) {
        set_error("leafq_kv8_append: rows must be 16-byte aligned and must not overlap");
        return LEAFQ_ERR_INVALID;
    }
    AppendArgs g{{k, v}, {k_stride, v_stride}, {cache->k_codes, cache->v_codes}, {cache->k_scales, cache->v_scales},
                 positions, slots, cos_table, sin_table, table_rows, tokens, cache->pages, page_shift(cache->page),
                 cache->kv_heads, rotary_dim, 1};
    // 32 .. 512 threads in whole warps, at least the page.
    const int threads = (cache->page * cache->dim / 8 / kAppendItems + 31) / 32 * 32;
    // Few rows: one per block, so that a decode step's rows run side by side;
    // many: a page's worth, so that most blocks have one whole run.
    int span = 1;
    while (span < cache->page && tokens / (2 * span) * cache->kv_heads * 2 >= 4 * (int64_t)sm_count()) span *= 2;
    g.span = span;
    const auto kernel = cache->dim == 32 ? kv8_append_kernel<32> : cache->dim == 64 ? kv8_append_kernel<64>
                        : cache->dim == 96 ? kv8_append_kernel<96> : kv8_append_kernel<128>;
    return launch(kernel, dim3(static_cast<unsigned>((tokens + span - 1) / span), cache->kv_heads, 2), dim3(threads), 0,
                  static_cast<cudaStream_t>(stream), (flags & LEAFQ_FLAG_PDL) != 0, "leafq_kv8_append", g);
}

}  // extern "C"
