// Drafted tokens over the paged INT8 KV cache (include/leafq.h):
//
//   kv8_tree_kernel     ancestors and positions of the rows of a tree
//   kv8_compact_kernel  the accepted path's rows moved together in the caches
//   kv8_release_kernel  pages behind a request's new length given back
#include <algorithm>
#include <climits>
#include <memory>
#include <new>

#include "kv8_attention.cuh"

namespace leafq {
namespace {

// ------------------------------------------------------------------- tree
// Row t's mask is its parent's and bit t.  A parent comes before its children, so
// the way to the root passes the mask's words from the last to the first, and a
// block does a request's rows in two steps: each row's ancestors inside its own word
// and the row where the way leaves it (at most 32 steps), then from word to word (at
// most 32 more).  A row whose way meets a parent that is none of the rows before it
// sees nothing.
constexpr int kNoRow = -2;  // the way ends at a row that is none; -1: at the request's cached tokens
constexpr int kTreeWords = 8;
static_assert(kTreeWords == 8, "a sector of 32 bytes, and the swizzle");

struct TreeArgs {
    const int32_t* parents;
    const int32_t* context;
    const int32_t* token_offsets;
    int32_t* positions;
    int32_t* masks;
    int64_t tokens;
    int requests, words, most;
};

__global__ void __launch_bounds__(LEAFQ_KV8_TREE_MOST) kv8_tree_kernel(const TreeArgs g) {
    __shared__ int32_t parent_s[LEAFQ_KV8_TREE_MOST], exit_s[LEAFQ_KV8_TREE_MOST];
    __shared__ uint32_t within_s[LEAFQ_KV8_TREE_MOST], tile_s[LEAFQ_KV8_TREE_MOST * kTreeWords];
    grid_dependency_wait();
    grid_launch_dependents();
    const int s = blockIdx.x, t = threadIdx.x;
    // The last block has the rows behind the last request's.
    const int64_t begin = max64(0, min64(g.token_offsets[s], g.tokens));
    const int64_t end = s < g.requests ? max64(begin, min64(g.token_offsets[s + 1], g.tokens)) : g.tokens;
    const int n = s < g.requests ? static_cast<int>(min64(end - begin, g.most)) : 0;
    if (t < n) parent_s[t] = g.parents[begin + t];
    __syncthreads();
    uint32_t within = 0;
    int at = t;
    if (t < n) {
        do {
            within |= 1u << (at & 31);
            const int up = parent_s[at];
            if (up >= at || up < -1) record_device_error(kSiteKv8Range);
            at = up >= at || up < -1 ? kNoRow : up;
        } while (at >= 0 && (at >> 5) == (t >> 5));
        within_s[t] = within;
        exit_s[t] = at;
    }
    __syncthreads();
    bool rooted = false;
    if (t < n) {
        int depth = __popc(within), up = at;
        while (up >= 0) {
            depth += __popc(within_s[up]);
            up = exit_s[up];
        }
        rooted = up != kNoRow;
        g.positions[begin + t] = rooted ? g.context[s] + depth - 1 : -1;
    }
    if (!rooted) at = -1;
    if (g.words == 1) {
        if (t < n) g.masks[begin + t] = static_cast<int32_t>(rooted ? within : 0u);
    }
    const int lane = t & 31, row0 = t - lane, rows = min(32, n - row0);
    uint32_t* tile = tile_s + row0 * kTreeWords;  // word j of lane l at l * 8 + (j ^ (l / 4)): no two lanes in a bank
    if (rows > 0 && g.words > 1) {
        for (int w0 = (g.words - 1) / kTreeWords * kTreeWords; w0 >= 0; w0 -= kTreeWords) {
#pragma unroll
            for (int j = kTreeWords - 1; j >= 0; --j) {
                uint32_t bits = 0;
                if (w0 + j == t >> 5) {
                    bits = rooted ? within : 0;
                } else if (at >= 0 && at >> 5 == w0 + j) {
                    bits = within_s[at];
                    at = exit_s[at];
                }
                tile[lane * kTreeWords + (j ^ lane >> 2)] = bits;
            }
            __syncwarp();
            const int word = w0 + (lane & 7);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = 4 * i + (lane >> 3);
                if (row < rows && word < g.words)
                    g.masks[(begin + row0 + row) * g.words + word] = static_cast<int32_t>(tile[row * kTreeWords + ((lane & 7) ^ i)]);
            }
            __syncwarp();
        }
    }
    // Rows past the bound, or past the last request's.
    if (s < g.requests && end - begin > g.most && t == 0) record_device_error(kSiteKv8Range);
    for (int64_t r = begin + n + t; r < end; r += blockDim.x) {
        g.positions[r] = -1;
        for (int w = 0; w < g.words; ++w) g.masks[r * g.words + w] = 0;
    }
}

// ---------------------------------------------------------------- compact
// The row at context + path[i] goes to context + i, for i < kept.  A path ascends, so
// a row never moves to a place that a later one comes from, and whole pages can be
// done in order: the page's new scale (the largest that its rows from other pages
// need), the rows that stay rounded to it where it grew, then the moved rows.  A warp
// does one request and kv head, of the keys or the values of one layer; a launch does up
// to 32 layers.  Bound by the chain path - table - rows - scales, a few round trips, and where a scale
// grows by the page's older rows, which a warp rounds 128 codes at a time, one after another: 64
// requests, 22 layers of 4 heads of 64, pages of 64, 30 us (12 to 14 of a layer's 344 key scales grow)
// and 9 to 10 where none does, as in caches that were compacted so before; 37 requests, 4 layers of 8
// heads of 128, pages of 16, 18 us and 7.5.
constexpr int kLayersAtOnce = 32;

struct CompactArgs {
    int8_t* codes[kLayersAtOnce][2];
    float* scales[kLayersAtOnce][2];
    const int32_t* context;
    const int32_t* lengths;
    const int32_t* table;
    const int32_t* path;
    const int32_t* kept;
    int64_t max_pages, pages;
    int requests, width, shift, kv_heads;
};

// What takes codes of one scale to another; zeros where the other is zero or no number.
__device__ __forceinline__ double ratio_of(float from, float to) {
    return to > 0.0f ? static_cast<double>(from) / static_cast<double>(to) : 0.0;
}

// Four codes times a ratio that has 64 bits, rounded.  (They fit eight bits, but for scales below
// 2^-126: their own rounding is coarse, and may leave them too small.)
__device__ __forceinline__ uint32_t scale_codes(uint32_t codes, double ratio) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int code = __double2int_rn(static_cast<int8_t>(codes >> (8 * i)) * ratio);
        out |= (static_cast<uint32_t>(min(max(code, -128), 127)) & 0xffu) << (8 * i);
    }
    return out;
}

__device__ __forceinline__ bool same(float a, float b) { return a == b || (isnan(a) && isnan(b)); }

template <int D>
__global__ void __launch_bounds__(128) kv8_compact_kernel(const CompactArgs g) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int s = static_cast<int>(unit / (2 * g.kv_heads));
    if (s >= g.requests) return;
    const int rest = static_cast<int>(unit - (int64_t)s * 2 * g.kv_heads), side = rest & 1, head = rest >> 1, layer = blockIdx.y;
    const int64_t context = g.context[s], fresh = (int64_t)g.lengths[s] - context;
    const int kept = static_cast<int>(max64(0, min64(min64(g.kept[s], g.width), fresh)));
    const int32_t* path = g.path + (int64_t)s * g.width;
    const int32_t* table = g.table + (int64_t)s * g.max_pages;
    const int page = 1 << g.shift;
    // The path: does it ascend inside the request's new rows, in pages that are there, and where does it begin to move?
    int first = kept;
    bool good = context >= 0 && (context + fresh - 1) >> g.shift < g.max_pages;
    const auto page_at = [&](int64_t position) { return table[position >> g.shift]; };
    const auto there = [&](int64_t position) { return static_cast<uint32_t>(page_at(position)) < static_cast<uint64_t>(g.pages); };
    for (int i = lane; i < kept && good; i += 32) {
        const int from = path[i], before = i > 0 ? path[i - 1] : -1;
        if (from <= before || from >= fresh) good = false;
        else if (from != i) {
            first = min(first, i);
            good = there(context + i) && there(context + from);
        }
    }
    good = __all_sync(~0u, good);
    first = __reduce_min_sync(~0u, first);
    if (!good) {
        if (kept > 0 && lane == 0 && rest == 0 && layer == 0) record_device_error(kSiteKv8Range);
        return;
    }
    if (first >= kept) return;
    constexpr int kLanes = D / 16, kAtOnce = 32 / kLanes;  // lanes of a row; rows at once
    const int sub = lane / kLanes, piece = lane - sub * kLanes;
    int8_t* codes = g.codes[layer][side];
    float* scales = g.scales[layer][side];
    const auto tile_of = [&](int id) { return (int64_t)id * g.kv_heads + head; };
    for (int i0 = first; i0 < kept;) {
        const int row0 = static_cast<int>((context + i0) & (page - 1)), i1 = min(kept, i0 + page - row0);
        const int id = page_at(context + i0);
        int8_t* to = codes + (tile_of(id) << g.shift) * D;
        const float before = scales[tile_of(id)];
        // The scale that rows from other pages need: of |code| * scale the largest, by its bits (a NaN is larger than all).
        unsigned long long largest = 0;
        for (int i = i0 + sub; i < i1 && sub < kAtOnce; i += kAtOnce) {
            const int64_t from = context + path[i];
            const int from_id = page_at(from);
            if (from_id == id) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(codes + ((tile_of(from_id) << g.shift) + (from & (page - 1))) * D + 16 * piece);
            uint32_t most = 0;
#pragma unroll
            for (const uint32_t x : {v.x, v.y, v.z, v.w}) most = __vmaxu4(most, __vabsss4(x));
            most = max(max(most & 0xffu, most >> 8 & 0xffu), max(most >> 16 & 0xffu, most >> 24));
            const double product = fabs(static_cast<double>(most) * static_cast<double>(scales[tile_of(from_id)]));
            largest = max(largest, static_cast<unsigned long long>(__double_as_longlong(product)));
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) largest = max(largest, __shfl_xor_sync(~0u, largest, d));
        const float need = static_cast<float>(__longlong_as_double(static_cast<long long>(largest)) / 127.0);
        const float scale = isnan(before) || (!(need > before) && !isnan(need)) ? before : need;
        const bool grown = !same(scale, before);
        if (grown) {
            const double ratio = ratio_of(before, scale);
            for (int i = lane; i < row0 * (D / 4); i += 32) {
                uint32_t* at = reinterpret_cast<uint32_t*>(to) + i;
                *at = scale_codes(*at, ratio);
            }
        }
        for (int i = i0; i < i1; i += kAtOnce) {
            const int mine = i + sub;
            const bool moves = sub < kAtOnce && mine < i1;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (moves) {
                const int64_t from = context + path[mine];
                const int from_id = page_at(from);
                v = *reinterpret_cast<const uint4*>(codes + ((tile_of(from_id) << g.shift) + (from & (page - 1))) * D + 16 * piece);
                const float own = from_id == id ? before : scales[tile_of(from_id)];
                if (!same(own, scale)) {
                    const double ratio = ratio_of(own, scale);
                    v = make_uint4(scale_codes(v.x, ratio), scale_codes(v.y, ratio), scale_codes(v.z, ratio), scale_codes(v.w, ratio));
                }
            }
            __syncwarp();  // rows of this turn may lie where others of it go
            if (moves) *reinterpret_cast<uint4*>(to + (row0 + mine - i0) * D + 16 * piece) = v;
            __syncwarp();
        }
        if (lane == 0 && grown) scales[tile_of(id)] = scale;
        __syncwarp();
        i0 = i1;
    }
}

// ---------------------------------------------------------------- release
// One prefix sum over the requests, of the pages that they give back: request s's go
// to free_pages[taken - upto ... taken - upto + own), below those of the requests
// before it.  Every block scans all requests, a thread each and a chunk at a time, and
// the blocks share the chunk's pages (found by a search of the prefix); block 0 writes
// the requests' outputs.  Launch bound: 64 requests 2.9 us, 2,000 (two chunks) 7.3.
constexpr int kReleaseThreads = 1024;

struct ReleaseArgs {
    const int32_t* context;
    const int32_t* lengths;
    const int32_t* kept;
    const int32_t* table;
    const int32_t* taken;
    int32_t* free_pages;
    int32_t* left;
    int32_t* taken_after;
    int64_t max_pages, free_count;
    int requests, shift;
};

__global__ void __launch_bounds__(kReleaseThreads) kv8_release_kernel(const ReleaseArgs g) {
    __shared__ int64_t upto_s[kReleaseThreads];   // pages given back by the chunk's requests up to this one
    __shared__ int64_t part_s[32];
    __shared__ int32_t after_s[kReleaseThreads];  // pages that it keeps; -1: refused
    __shared__ long long reached_s;
    grid_dependency_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const int64_t page = int64_t{1} << g.shift, taken = *g.taken;
    const bool writer = blockIdx.x == 0;
    if (tid == 0) reached_s = 0;
    int64_t base_pages = 0;
    for (int base = 0; base < g.requests; base += threads) {
        const int r = base + tid;
        int64_t held = 0, after = 0, length = 0, left = 0;
        if (r < g.requests) {
            length = g.lengths[r];
            if (length < 0 || (length + page - 1) >> g.shift > g.max_pages) {
                if (writer) record_device_error(kSiteKv8Range);
                left = length;
                length = 0;
            } else {
                left = max64(0, min64(length, (int64_t)g.context[r] + g.kept[r]));
                held = (length + page - 1) >> g.shift;
                after = (left + page - 1) >> g.shift;
            }
        }
        const int64_t own = held - after;
        int64_t upto = own;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int64_t other = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += other;
        }
        __syncthreads();  // the chunk before is done
        if (lane == 31) part_s[warp] = upto;
        __syncthreads();
        int64_t total = 0;
        for (int w = 0; w < threads / 32; ++w) {
            if (w < warp) upto += part_s[w];
            total += part_s[w];
        }
        // Pages that would go below the list's start, or come from past its end, stay with their request.
        const int64_t at = taken - (base_pages + upto);
        const bool granted = own == 0 || (at >= 0 && taken <= g.free_count);
        upto_s[tid] = upto;
        after_s[tid] = granted ? static_cast<int32_t>(after) : -1;
        if (writer && r < g.requests) {
            g.left[r] = static_cast<int32_t>(granted ? left : length);
            if (!granted) record_device_error(kSiteKv8Range);
            if (granted && own > 0) atomicMax(&reached_s, static_cast<long long>(base_pages + upto));
        }
        __syncthreads();
        const int count = min(threads, g.requests - base);
        for (int64_t i = (int64_t)blockIdx.x * threads + tid; i < total; i += (int64_t)gridDim.x * threads) {
            int lo = 0, hi = count - 1;  // the first request whose pages end behind i
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (upto_s[mid] > i) hi = mid;
                else lo = mid + 1;
            }
            if (after_s[lo] < 0) continue;
            const int64_t begins = lo > 0 ? upto_s[lo - 1] : 0, column = after_s[lo] + (i - begins);
            g.free_pages[taken - (base_pages + upto_s[lo]) + (i - begins)] = g.table[(int64_t)(base + lo) * g.max_pages + column];
        }
        base_pages += total;
    }
    __syncthreads();
    if (writer && tid == 0) *g.taken_after = static_cast<int32_t>(taken - reached_s);
}

// Whether no two pools of the layers share memory.
bool pools_apart(const leafq_kv8_cache* caches, int layers, const char* what) {
    struct Pool {
        uintptr_t begin, end;
    };
    const size_t count = 4 * static_cast<size_t>(layers);
    const std::unique_ptr<Pool[]> pools(new (std::nothrow) Pool[count]);
    if (!pools) {
        set_error(std::string(what) + ": out of host memory");
        return false;
    }
    for (int i = 0; i < layers; ++i) {
        const leafq_kv8_cache& c = caches[i];
        const uintptr_t scales = 4 * static_cast<uintptr_t>(c.pages) * c.kv_heads, codes = scales / 4 * c.page * c.dim;
        const void* begins[4] = {c.k_codes, c.v_codes, c.k_scales, c.v_scales};
        for (int j = 0; j < 4; ++j) {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(begins[j]);
            pools[4 * i + j] = Pool{begin, begin + (j < 2 ? codes : scales)};
        }
    }
    std::sort(pools.get(), pools.get() + count, [](const Pool& a, const Pool& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < count; ++i)
        if (pools[i].begin < pools[i - 1].end) {
            set_error(std::string(what) + ": a cache is there twice, or has memory of another");
            return false;
        }
    return true;
}

// The sizes that the step's arrays have.
bool step_valid(const leafq_kv8_step* step, const char* what) {
    if (!step || step->tokens < 0 || step->tokens > INT_MAX || step->max_tokens < 0 || step->requests < 0 || step->max_pages < 0 ||
        step->max_pages > INT_MAX) {
        set_error(std::string(what) + ": invalid step");
        return false;
    }
    return true;
}

}  // namespace
}  // namespace leafq

using namespace leafq;

extern "C" {

int leafq_kv8_tree(void* stream, const int32_t* parents, const leafq_kv8_step* step, int32_t* positions, int32_t* masks,
                   int words, uint32_t flags) {
    clear_error();
    const char* what = "leafq_kv8_tree";
    if (!step_valid(step, what)) return LEAFQ_ERR_INVALID;
    if (step->tokens == 0) return LEAFQ_OK;
    if (step->max_tokens > LEAFQ_KV8_TREE_MOST || words <= 0 || words > LEAFQ_KV8_TREE_MOST / 32 || step->max_tokens > 32 * (int64_t)words) {
        set_error("leafq_kv8_tree: a request's tree has at most " + std::to_string(LEAFQ_KV8_TREE_MOST) +
                  " rows, and masks have max_tokens / 32 words, rounded up (32 at most)");
        return step->max_tokens > LEAFQ_KV8_TREE_MOST ? LEAFQ_ERR_UNSUPPORTED : LEAFQ_ERR_INVALID;
    }
    if (!parents || !positions || !masks || !step->token_offsets || (step->requests > 0 && !step->context)) {
        set_error("leafq_kv8_tree: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    const Span inputs[] = {{parents, step->tokens}, {step->context, step->requests}, {step->token_offsets, step->requests + 1}};
    const Span outputs[] = {{positions, step->tokens}, {masks, step->tokens * words}};
    if (!apart(outputs, inputs)) {
        set_error("leafq_kv8_tree: outputs must not overlap one another or the inputs");
        return LEAFQ_ERR_INVALID;
    }
    const TreeArgs g{parents, step->context, step->token_offsets, positions, masks, step->tokens, step->requests, words,
                     static_cast<int>(step->max_tokens)};
    const int threads = std::max(32, (g.most + 31) / 32 * 32);
    return launch(kv8_tree_kernel, dim3(static_cast<unsigned>(step->requests) + 1), dim3(threads), 0, static_cast<cudaStream_t>(stream),
                  (flags & LEAFQ_FLAG_PDL) != 0, what, g);
}

int leafq_kv8_compact(void* stream, const leafq_kv8_cache* caches, int layers, const leafq_kv8_step* step, const int32_t* path,
                      int64_t path_width, const int32_t* kept, uint32_t flags) {
    clear_error();
    const char* what = "leafq_kv8_compact";
    if (!step_valid(step, what)) return LEAFQ_ERR_INVALID;
    if (layers < 0 || (layers > 0 && !caches) || path_width < 0 || path_width > LEAFQ_KV8_TREE_MOST) {
        set_error("leafq_kv8_compact: invalid layers, or paths of more than " + std::to_string(LEAFQ_KV8_TREE_MOST) + " rows");
        return LEAFQ_ERR_INVALID;
    }
    for (int i = 0; i < layers; ++i) {
        const leafq_kv8_cache& c = caches[i];
        if (!kv8_cache_valid(&c, what)) return LEAFQ_ERR_INVALID;
        if (!kv8_dim_supported(c.dim)) {
            set_error("leafq_kv8_compact: head sizes are 32, 64, 96 and 128");
            return LEAFQ_ERR_UNSUPPORTED;
        }
        if (c.page != caches[0].page || c.kv_heads != caches[0].kv_heads || c.dim != caches[0].dim || c.pages != caches[0].pages) {
            set_error("leafq_kv8_compact: the layers' caches must have the same pages, kv heads and head size");
            return LEAFQ_ERR_INVALID;
        }
    }
    if (layers == 0 || step->requests == 0 || path_width == 0) return LEAFQ_OK;
    if (!path || !kept || !step->context || !step->lengths || (step->max_pages > 0 && !step->table)) {
        set_error("leafq_kv8_compact: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    if (!pools_apart(caches, layers, what)) return LEAFQ_ERR_INVALID;
    const leafq_kv8_cache& c = caches[0];
    const int64_t blocks = ((int64_t)step->requests * 2 * c.kv_heads + 3) / 4;
    if (blocks > INT_MAX) {
        set_error("leafq_kv8_compact: too many requests");
        return LEAFQ_ERR_INVALID;
    }
    const auto kernel = c.dim == 32 ? kv8_compact_kernel<32> : c.dim == 64 ? kv8_compact_kernel<64>
                        : c.dim == 96 ? kv8_compact_kernel<96> : kv8_compact_kernel<128>;
    for (int first = 0; first < layers; first += kLayersAtOnce) {
        const int count = std::min(kLayersAtOnce, layers - first);
        CompactArgs g = {};
        for (int i = 0; i < count; ++i) {
            const leafq_kv8_cache& layer = caches[first + i];
            g.codes[i][0] = layer.k_codes;
            g.codes[i][1] = layer.v_codes;
            g.scales[i][0] = layer.k_scales;
            g.scales[i][1] = layer.v_scales;
        }
        g.context = step->context;
        g.lengths = step->lengths;
        g.table = step->table;
        g.path = path;
        g.kept = kept;
        g.max_pages = step->max_pages;
        g.pages = c.pages;
        g.requests = step->requests;
        g.width = static_cast<int>(path_width);
        g.shift = page_shift(c.page);
        g.kv_heads = c.kv_heads;
        const int st = launch(kernel, dim3(static_cast<unsigned>(blocks), count), dim3(128), 0, static_cast<cudaStream_t>(stream),
                              (flags & LEAFQ_FLAG_PDL) != 0, what, g);
        if (st) return st;
    }
    return LEAFQ_OK;
}

int leafq_kv8_release(void* stream, const leafq_kv8_step* step, const int32_t* kept, int page, int32_t* free_pages,
                      int64_t free_count, const int32_t* taken, int32_t* lengths, int32_t* taken_after, uint32_t flags) {
    clear_error();
    const char* what = "leafq_kv8_release";
    if (!step_valid(step, what)) return LEAFQ_ERR_INVALID;
    const int shift = page_shift(page);
    if (shift < 0 || free_count < 0 || free_count > INT_MAX || step->max_pages > INT_MAX / page) {
        set_error("leafq_kv8_release: a page that is not 16, 32, 64 or 128 tokens, or sizes that do not fit int32");
        return LEAFQ_ERR_INVALID;
    }
    if (!taken || !taken_after || (free_count > 0 && !free_pages) ||
        (step->requests > 0 && (!kept || !lengths || !step->context || !step->lengths || (step->max_pages > 0 && !step->table)))) {
        set_error("leafq_kv8_release: null pointer");
        return LEAFQ_ERR_INVALID;
    }
    // Every block reads the inputs while others write.
    const Span inputs[] = {{step->context, step->requests}, {step->lengths, step->requests}, {kept, step->requests},
                           {step->table, step->requests * step->max_pages}, {taken, 1}};
    const Span outputs[] = {{free_pages, free_count}, {lengths, step->requests}, {taken_after, 1}};
    if (!apart(outputs, inputs)) {
        set_error("leafq_kv8_release: outputs must not overlap one another or the inputs (lengths and the step's, taken_after and taken, ...)");
        return LEAFQ_ERR_INVALID;
    }
    const ReleaseArgs g{step->context, step->lengths, kept, step->table, taken, free_pages, lengths, taken_after, step->max_pages,
                        free_count, step->requests, shift};
    const int threads = step->requests <= 256 ? 256 : kReleaseThreads;
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(sm_count(), step->requests * step->max_pages / (8 * threads)));
    return launch(kv8_release_kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, static_cast<cudaStream_t>(stream),
                  (flags & LEAFQ_FLAG_PDL) != 0, what, g);
}

}  // extern "C"
