// Attention of trees over the paged INT8 cache, many query rows.
//
// Compiled as a whole program (build.py): setmaxnreg is ignored in relocatable
// device code.
#include <algorithm>
#include <type_traits>

#include "kv8_tile.cuh"

namespace leafq {
namespace {

// The arithmetic is kv8_tile.cu's: codes exact in fp16, fp32 operands as hi + lo halves, the
// V scale in the exponent, S and P in TMEM, O in spans.  What differs is the block's shape.  A
// tree's rows (nodes times query heads of a kv head) are usually more than 128 and see the same
// keys, so one block a SM has 256 of them, two halves of 128, and converts each tile of codes
// once for both.  An item of 128 rows or fewer gives its keys to the halves instead, every
// other tile each, and joins them at its end.
//   warps 0-3, 4-7  softmax of a half: one row per thread (its TMEM lane)
//   warps 8-11      codes to fp16: two warps K, two V
//   warps 12, 13    MMA issue, a half each
//   warps 14, 15    the items and their query rows, the first half's first
// A unit is a tile of keys for one half.  The tensor pipe has one half's units while the other
// is in its softmax; one warp that issued for both halves was itself what they waited for (some
// 250 instructions a unit, one after another).
//
// Bound, 128-wide heads: the hand-offs S - softmax - P - PV of a half, of which the other half's
// fill a part (5 requests of 12 to 18 thousand cached tokens: tensor pipe busy 45 %, issue slots
// 38 %).  6 requests of 9 to 100 thousand cached tokens, trees of 40, 64 / 8 heads: 1,202 us,
// 0.99 PFLOP of MMAs (fp32 operands are two halves) at 825 TFLOP/s, calls back to back in a graph for
// some milliseconds; for two seconds without a rest 1,327 us, in a graph or not, the power limit
// holding the clock at 1.7 GHz.  128 rows a block and two blocks a SM took 1,771.  64-wide heads: the softmax's issue slots, 1.5 to 2.5 us a tile of 96
// keys for 256 rows, and for short caches 6 us for a block's first rows and 2 to 3 for an item's
// output: 64 trees of 26 over 512 to 767 tokens, 32 / 4 heads, 74 us, in 256 items on 148 blocks
// (all cut into even shares 90; kv8_tile.cu's shape, two blocks a SM of 128 rows, 60: that form of
// trees was given up for this one, which is the better one for long caches).
constexpr int kRows = 128, kHalves = 2;

// What the roles need to know of an item: up to 256 query rows of one kv head of a request,
// and, where it is cut into parts along the keys, which one.  tiles < 0: there are no more.
struct TreeItem {
    int row0, first_row, rows, context, keys, tiles, head, request;
    int tile0, parts, part, place;  // its first key tile; the block that has the first part
    int both;                       // 1: both halves have rows; 0: they share the keys
};

// The units of all items in a row (with kItemCost for each item's own sake) are dealt out to
// the blocks in even shares.  An item of more than kShortTiles tiles or more than two shares
// is cut where a share ends; another goes to the block that has its middle, since a join
// would take longer.  Measured with 8 heads of 64, 32 rows a head, us: 16 requests of 700
// tokens, an item of a share and more, whole 21 and cut 35; 4 requests of 3,000 tokens, an
// item of several shares, whole 48 and cut 28.  A share is kLeastShare units at least, so that
// every part of an item has a tile.
constexpr int kTreeBlocks = 148, kTreePlaces = 2 * kTreeBlocks, kShortTiles = 32, kLeastShare = 8;
static_assert((kTileCounters + 4 + 2 * kTreeBlocks) * 4 <= kCounterBytes, "two counters for each block");
static_assert(kTreePlaces % 4 == 0, "the counters are zeroed four at a time");

template <int D>
struct TreeShape {
    static constexpr int kKeys = D <= 64 ? 96 : 64;
    static constexpr int kBlocks = (D + 63) / 64;        // 64-element (128-byte) column blocks
    static constexpr int kStages = D <= 64 ? 4 : 3;      // of K, and of V
    static constexpr int kGroups = kKeys / 16;           // of keys that share a page for certain
    static constexpr int kInfo = 8;                      // ring of the groups' scales: a tile's are read while those of
                                                         // up to kStages + 3 later tiles are written (where halves
                                                         // share the keys: of tile t + 2 the scores are issued then and
                                                         // t + 3 is passed, so that its stage may be filled again)
    static constexpr int kQBytes = kBlocks * kRows * 128;
    static constexpr int kQSlots = D <= 64 ? 2 : 1;      // of query rows: the next item's beside this one's
    static constexpr int kItems = 3;                     // ring of their descriptions
    static constexpr int kKvBytes = kBlocks * kKeys * 128;
    static constexpr int kSpan = (D <= 64 ? 384 : 512) / kKeys;           // a half's tiles between O's additions to the rounded sum
    static constexpr int kItemCost = D <= 64 ? 4 : 6;    // of an item for its own sake, in units
    static constexpr int kThreads = 512;
    // A scheduler has two softmax warps, a converting one and one of the last four.
    static constexpr int kLaunchRegs = 128, kSoftmaxRegs = 152, kConvertRegs = 104, kOtherRegs = 104;
    static constexpr int kPieces = kKeys * D / 16 / 64;  // 16-byte pieces of a K (or V) tile per converting thread
    static constexpr int kOutCols = kBlocks * 64;        // O columns (those past D are not read)
    static constexpr int kHalfCols = 256;
    static constexpr int kPart = kHalves * kRows * (D + 2);  // floats of a part's result: O [D / 4][256][4], m [256], l [256]
    static constexpr size_t kBarriers = 4 * kStages + 6 * kHalves + 3 * kQSlots + kItems + 2 + kHalves;
    static constexpr size_t kSmem = kQSlots * kHalves * 2 * kQBytes + 2 * kStages * kKvBytes + kInfo * kGroups * 16 + kRows * 8 +
                                    kItems * sizeof(TreeItem) + 4 + kQSlots * kHalves * kRows + kBarriers * 8 + 8;
    static_assert(sizeof(TreeItem) * kItems % 8 == 4, "the barriers' alignment");
    static_assert(kRows * D * 4 <= 2 * kQBytes, "a half's output goes through the place of its rows");
    static_assert(kSmem <= 227 * 1024, "a block a SM");
    static_assert(kInfo >= kStages + 4, "no scales are written over that are still read");
    static_assert(2 * kKeys + kOutCols <= kHalfCols, "the halves share the SM's 512 TMEM columns");
    static_assert(2 * kSoftmaxRegs + kConvertRegs + kOtherRegs <= 4 * kLaunchRegs, "the split of what the launch gives each scheduler");
};

template <int D>
__global__ void __launch_bounds__(TreeShape<D>::kThreads, 1)
kv8_attend_tree_kernel(const Kv8AttendArgs g, const DeviceWatch watch, uint32_t* taken, uint32_t* arrivals, float* parts) {
    using C = TreeShape<D>;
    constexpr int kSpan = C::kSpan;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_rows = smem;  // [kQSlots][half]: hi, lo
    uint8_t* k_tiles = q_rows + C::kQSlots * kHalves * 2 * C::kQBytes;
    uint8_t* v_tiles = k_tiles + C::kStages * C::kKvBytes;
    float4* info = reinterpret_cast<float4*>(v_tiles + C::kStages * C::kKvBytes);  // [kInfo][kGroups]: ks, log2 vs, 1 / vs
    float2* join_s = reinterpret_cast<float2*>(info + C::kInfo * C::kGroups);      // [128]: the second half's m, l
    TreeItem* items = reinterpret_cast<TreeItem*>(join_s + kRows);
    uint8_t* power = reinterpret_cast<uint8_t*>(items + C::kItems) + 4;  // [kQSlots][256]: of two, that a row was scaled down by (exponent bits)
    uint64_t* k_full = reinterpret_cast<uint64_t*>(power + C::kQSlots * kHalves * kRows);
    uint64_t* k_empty = k_full + C::kStages;
    uint64_t* v_full = k_empty + C::kStages;
    uint64_t* v_empty = v_full + C::kStages;
    uint64_t* s_full = v_empty + C::kStages;     // [half][S buffer], as p_full
    uint64_t* p_full = s_full + 2 * kHalves;
    uint64_t* o_done = p_full + 2 * kHalves;     // [half]: PV of a unit has completed
    uint64_t* item_done = o_done + kHalves;      // [half]: all MMAs of an item that gave it units have completed
    uint64_t* q_full = item_done + kHalves;      // [slot][half]: an item's rows are there
    uint64_t* q_empty = q_full + C::kQSlots * kHalves;  // its last scores are computed, its description read (its output written), the end before it seen
    uint64_t* found_full = q_empty + C::kQSlots; // by description: it is there
    uint64_t* joined = found_full + C::kItems;   // the second half has left its results to the first
    uint64_t* taken_over = joined + 1;           // and the first has read m and l
    uint64_t* drained = taken_over + 1;          // [half]
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drained + kHalves);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kMmaWarp = 12;
    const auto token_of = [&](int row) { return static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(g.group)); };

    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it; dynamic shared memory starts there
        if (tid == 0) report(watch, kSiteKv8Tile);
        return;
    }
    if (warp == kMmaWarp) {
        if (lane == 0) {
            for (int i = 0; i < C::kStages; ++i) {
                mbar_init(&k_full[i], 2);
                mbar_init(&k_empty[i], kHalves);
                mbar_init(&v_full[i], 2);
                mbar_init(&v_empty[i], kHalves);
            }
            for (int i = 0; i < 2 * kHalves; ++i) {
                mbar_init(&s_full[i], 1);
                mbar_init(&p_full[i], 4);
            }
            for (int i = 0; i < kHalves; ++i) {
                mbar_init(&o_done[i], 1);
                mbar_init(&item_done[i], 1);
                mbar_init(&drained[i], 1);
            }
            for (int i = 0; i < C::kQSlots; ++i) {
                for (int half = 0; half < kHalves; ++half) mbar_init(&q_full[i * kHalves + half], 4);
                mbar_init(&q_empty[i], 5 * kHalves + 2);
            }
            for (int i = 0; i < C::kItems; ++i) mbar_init(&found_full[i], 1);
            mbar_init(joined, 4);
            mbar_init(taken_over, 4);
            fence_barrier_init();
        }
        __syncwarp();
        tmem_alloc(tmem_holder, kHalves * C::kHalfCols);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_holder;
    grid_dependency_wait();
    grid_launch_dependents();

    // Lanes of a row: D / 8, eight values each (a rotation pair's quarters).
    constexpr int kLanes = D / 8;  // 4, 8, 12, 16
    constexpr int kAtOnce = 32 / kLanes;
    const int sub = lane / kLanes, part = lane - sub * kLanes;
    const int pairs = g.rotary >> 1;
    const bool turned = 4 * part < pairs;
    const int at = turned ? 4 * part : 2 * pairs + 4 * (part - pairs / 4);
    const int to = turned ? at + pairs : at + ((D - 2 * pairs) >> 1);
    // Query rows of an item's half, by `warps` warps of which this is the pw-th.  Loads run two turns
    // ahead; rotated, scaled by the row's power of two, split, stored swizzled.  (What lies behind the
    // item's rows is left as it is: every row of S and O is its own.)
    const auto put_rows = [&](const TreeItem& next, int half_of, uint8_t* q_hi, uint8_t* powers, int pw, int warps) {
        const int pass = warps * kAtOnce, first = half_of * kRows, turns = (min(kRows, next.rows - first) + pass - 1) / pass;
        const int step_t = pass / g.group, step_h = pass - step_t * g.group;
        float4 a, b, cs, sn, a1, b1, cs1, sn1;  // this turn's, the next one's
        a = b = cs = sn = a1 = b1 = cs1 = sn1 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const int r0 = next.first_row + first + pw * kAtOnce + sub;
        int t = token_of(r0), hq = r0 - t * g.group;  // of the row two turns ahead
        // Its position is asked for a turn earlier still: the tables' rows depend on it.
        const auto row_there = [&](int i) { return sub < kAtOnce && i < turns && first + i * pass + pw * kAtOnce + sub < next.rows; };
        int pos_next = turned && row_there(0) ? load_now(g.positions + (next.row0 + t)) : 0;
#pragma unroll 2
        for (int i = -2; i < turns; ++i) {
            unsigned long long v[4] = {pack2(a.x, a.y), pack2(a.z, a.w), pack2(b.x, b.y), pack2(b.z, b.w)};
            if (turned) {  // (a product and a sum may be rounded as one)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const unsigned long long x = v[e], y = v[2 + e];
                    const unsigned long long c2 = e == 0 ? pack2(cs.x, cs.y) : pack2(cs.z, cs.w), s2 = e == 0 ? pack2(sn.x, sn.y) : pack2(sn.z, sn.w);
                    v[e] = sub2(mul2(x, c2), mul2(y, s2));
                    v[2 + e] = add2(mul2(y, c2), mul2(x, s2));
                }
            }
            a = a1, b = b1, cs = cs1, sn = sn1;
            a1 = b1 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int64_t pos_asked = pos_next;
            const int t_asked = t, hq_asked = hq;
            t += step_t;
            hq += step_h;
            if (hq >= g.group) {
                hq -= g.group;
                ++t;
            }
            if (turned && row_there(i + 3)) pos_next = load_now(g.positions + (next.row0 + t));
            if (row_there(i + 2)) {
                const float* src = g.q + ((int64_t)next.row0 + t_asked) * g.q_stride + (int64_t)(next.head * g.group + hq_asked) * D;
                a1 = load_now(reinterpret_cast<const float4*>(src + at));
                b1 = load_now(reinterpret_cast<const float4*>(src + to));
                if (turned) {
                    int64_t pos = pos_asked;
                    if (pos < 0 || pos >= g.table_rows) {
                        if (part == 0 && pos >= 0) report(watch, kSiteKv8Range);
                        pos = 0;
                    }
                    cs1 = load_now(reinterpret_cast<const float4*>(g.cos_table + pos * pairs + at));
                    sn1 = load_now(reinterpret_cast<const float4*>(g.sin_table + pos * pairs + at));
                }
            }
            if (i < 0) continue;
            const int r = i * pass + pw * kAtOnce + sub;
            // A NaN is no maximum, but it stays one in its row's products.
            float largest = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 x = unpack2(v[e]);
                largest = fmaxf(largest, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
            if constexpr (kLanes == 12) {
                float all = 0.0f;
#pragma unroll
                for (int e = 0; e < kLanes; ++e) all = fmaxf(all, __shfl_sync(~0u, largest, min(sub * kLanes + e, 31)));
                largest = all;
            } else {
#pragma unroll
                for (int d = kLanes / 2; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor_sync(~0u, largest, d));
            }
            float up, down;
            row_power(__float_as_uint(largest), up, down);
            if (sub < kAtOnce && r < kRows) {
                if (part == 0) powers[r] = static_cast<uint8_t>(__float_as_uint(down) >> 23);
                const unsigned long long up2 = pack2(up, up);
#pragma unroll
                for (int quarter = 0; quarter < 2; ++quarter) {
                    const int d = quarter == 0 ? at : to;
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // 11 bits (exact in fp16), and what is left.
                        const unsigned long long x = mul2(v[2 * quarter + e], up2);
                        const float2 whole = unpack2(x);
                        const float h0 = __uint_as_float(__float_as_uint(whole.x) & 0xffffe000u);
                        const float h1 = __uint_as_float(__float_as_uint(whole.y) & 0xffffe000u);
                        const float2 rest = unpack2(sub2(x, pack2(h0, h1)));
                        hi[e] = half2_bits(h0, h1);
                        lo[e] = half2_bits(rest.x, rest.y);
                    }
                    const int offset = (d >> 6) * (kRows * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 4) * 2;
                    *reinterpret_cast<uint2*>(q_hi + offset) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(q_hi + C::kQBytes + offset) = make_uint2(lo[0], lo[1]);
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
    };

    // Units are counted on over the items, by half (n); barriers of per-unit and per-item
    // phases are waited for in order by every role.
    if (warp < 4 * kHalves) {
        // ------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
        const int side = warp >> 2, r = tid & (kRows - 1);
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t half_tmem = tmem + side * C::kHalfCols, o_tmem = half_tmem + 2 * C::kKeys;
        __align__(16) float o_sum[D];  // the rounded sum
        const uint32_t o_local = local_address(o_sum);
        const auto get_sum = [&](int c) { return load_local(o_local + 16 * c); };  // elements 4 c .. 4 c + 3 of a row
        const auto put_sum = [&](int c, float4 v) { store_local(o_local + 16 * c, v); };
        int n = 0, first_tile = 0, shared_items = 0;  // the half's units, the block's tiles, and the items that shared keys, before
        int worked = 0;                               // items before of which the half had units
        bool ok = true;
        for (int it = 0;; ++it) {
            const int q_slot = it % C::kQSlots;
            const TreeItem* item = items + it % C::kItems;
            ok = ok && __all_sync(~0u, tile_wait(watch, &found_full[it % C::kItems], it / C::kItems & 1));
            if (!ok) break;
            const bool both = item->both != 0;
            const int rows_at = q_slot * kHalves + (both ? side : 0);
            if (item->tiles < 0) break;
            // The first item's rows, or all where there is no room beside them, are its softmax warps' own work.
            if (it == 0 || C::kQSlots == 1) {
                if (it > 0) ok = __all_sync(~0u, tile_wait(watch, q_empty, (it - 1) & 1));
                if (!ok) break;
                if (both || side == 0) put_rows(*item, side, q_rows + side * 2 * C::kQBytes, power + side * kRows, warp & 3, 4);
                if (lane == 0) mbar_arrive(&q_full[side]);
            }
            // (A phase is waited for by whoever waits for a later one: the end of the one before would pass for
            // it.  The second half needs the first's rows in some items only.)
            ok = __all_sync(~0u, tile_wait(watch, &q_full[q_slot * kHalves], it / C::kQSlots & 1));
            if (side == 1) ok = ok && __all_sync(~0u, tile_wait(watch, &q_full[q_slot * kHalves + 1], it / C::kQSlots & 1));
            if (!ok) break;
            const int tiles = item->tiles, first_row = item->first_row + (both ? side * kRows : 0);
            const int rows = both ? max(0, min(kRows, item->rows - side * kRows)) : item->rows;
            const int row0 = item->row0, context = item->context, keys = item->keys, head = item->head, tile0 = item->tile0;
            const int count = item->parts, part_index = item->part, place = item->place;
            const float factor = __uint_as_float(static_cast<uint32_t>(power[rows_at * kRows + r]) << 23) * g.scale * kLog2e;
            if (C::kQSlots == 1 && (both || side == 1)) {
                __syncwarp();
                if (lane == 0) mbar_arrive(q_empty);
            }
            // Tiles of this half: first + step i, of its units.
            const int first = both ? 0 : side, step = both ? 1 : 2, units = both ? tiles : (tiles + 1 - side) / 2;
            const int t = token_of(first_row + r), hq = (first_row + r) - t * g.group;
            const int pos = r < rows ? g.positions[row0 + t] : -1;
            const bool seen = r < rows && pos >= 0 && (g.rotary == 0 || pos < g.table_rows);
            const int limit = seen ? min(keys, context + t + 1) : 0;
            const uint32_t* row_mask = g.masks + (int64_t)(row0 + (r < rows ? t : 0)) * g.mask_words;
            float* out = g.out + ((int64_t)row0 + t) * g.heads * D + (int64_t)(head * g.group + hq) * D;
            float m = -INFINITY, l = 0.0f, m_sum = -INFINITY;
            const bool idle = (warp & 3) * 32 >= rows;  // none of the warp's rows is the item's
            for (int j = 0; j < units; ++j, ++n) {
                const int tile = first + step * j;
                const uint32_t s_tmem = half_tmem + (n & 1) * C::kKeys;
                ok = __all_sync(~0u, tile_wait(watch, &s_full[2 * side + (n & 1)], (n >> 1) & 1));
                if (!ok) break;
                if (idle) {
                    if (lane == 0) mbar_arrive(&p_full[2 * side + (n & 1)]);
                    continue;
                }
                tcgen05_fence_after();
                const float4* scales = info + ((first_tile + tile) % C::kInfo) * C::kGroups;
                const int drafted = (tile0 + tile) * C::kKeys - context;  // the tile's first key among the request's new ones
                const int visible = limit - (tile0 + tile) * C::kKeys;    // columns of this tile that the row may see
                const bool whole = __all_sync(~0u, visible >= C::kKeys) && drafted + C::kKeys <= 0;
                uint32_t x[32];
                const auto read = [&](int c) {
                    tmem_ld_32x32b_x32(s_tmem + lanes + 32 * c, x);
                    tmem_wait_ld();
                    if (!whole) {
                        const uint32_t window = tree_window(row_mask, g.mask_words, drafted + 32 * c);
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = 32 * c + e >= visible || !(window >> e & 1u) ? 0xff800000u : x[e];
                    }
                };
                // From an MMA sum to x_j: above zero, so that -inf stays.
                const auto slope = [&](float ks) { return ks * factor == 0.0f ? 1e-37f : ks * factor; };
                const auto largest = [&](int c) {  // x_j of the 32
                    float top = -INFINITY;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float* at = reinterpret_cast<const float*>(x) + 16 * half;
                        float most = at[0];
#pragma unroll
                        for (int e = 1; e < 16; ++e) most = fmaxf(most, at[e]);
                        const float4 scale = scales[2 * c + half];
                        top = fmaxf(top, fmaf(most, slope(scale.x), scale.z == kZeroInverse ? kZeroLog2 + kZeroAbove : scale.y));
                    }
                    return top;
                };
                // The weights count relative to a whole power of two m.  It is taken from
                // the first tile with a key for the row; later tiles are weighed with it as it stands, and
                // only where weights come out above kTileHighest is it raised, with what has
                // been weighed so far scaled down, exactly but for what is lost below
                // 2^-30 of the largest.
                const bool anew = j % kSpan == 0;
                const float m_before = m;
                if (j == 0 || __any_sync(~0u, m == -INFINITY && visible > 0)) {
                    float top = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < C::kKeys / 32; ++c) {
                        read(c);
                        top = fmaxf(top, largest(c));
                    }
                    if (m == -INFINITY) m = ceilf(top);
                }
#pragma unroll 1
                for (int c = 0; c < C::kKeys / 32; ++c) {
                    read(c);
                    uint32_t p[32];
                    float weight;  // L of the 32
#pragma unroll 1
                    for (;;) {
                        const float shift = m == -INFINITY ? 0.0f : m - kTileLift;
                        bool high = false;
                        weight = 0.0f;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const float4 scale = scales[2 * c + half];
                            const float a1 = slope(scale.x), b1 = scale.y - shift;
                            const unsigned long long a = pack2(a1, a1), b = pack2(b1, b1);
                            unsigned long long sum = 0;
#pragma unroll
                            for (int e = 16 * half; e < 16 * half + 16; e += 2) {
                                const float2 y = unpack2(fma2(pack2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), a, b));
                                const float w0 = ex2(y.x), w1 = ex2(y.y);
                                const unsigned long long w = pack2(w0, w1);
                                sum = add2(sum, w);
                                const float h0 = __uint_as_float(__float_as_uint(w0) & 0xffffe000u);
                                const float h1 = __uint_as_float(__float_as_uint(w1) & 0xffffe000u);
                                const float2 low = unpack2(sub2(w, pack2(h0, h1)));
                                p[e / 2] = half2_bits(h0, h1);
                                p[16 + e / 2] = half2_bits(low.x, low.y);
                            }
                            const float2 both = unpack2(sum);
                            high |= both.x + both.y > kTileHighest;
                            weight = fmaf(both.x + both.y, scale.z, weight);
                        }
                        if (!__any_sync(~0u, high)) break;
                        // Raise m: the weights of this tile so far, O and L come down.
                        const float raised = high ? fmaxf(m, ceilf(largest(c))) : m;
                        const float down = m == -INFINITY ? 0.0f : ex2(m - raised);  // of a whole number: exact
                        float left = m == -INFINITY ? 42.0f : fminf(raised - m, 42.0f);
                        if (!(raised > m)) left = 0.0f;
                        m = raised;
                        l *= down;
                        if (!anew) {
                            // This tile's S means that PV of tile n - 2 is done, so o_done is
                            // waited for one phase on at most, here and below.
                            ok = __all_sync(~0u, tile_wait(watch, &o_done[side], (n - 1) & 1));
                            tcgen05_fence_after();
                        }
                        uint32_t y[32];
                        tmem_wait_st();
#pragma unroll 1
                        for (int cc = 0; cc < c; ++cc) {
                            tmem_ld_32x32b_x32(s_tmem + lanes + 32 * cc, y);
                            tmem_wait_ld();
#pragma unroll
                            for (int third = 0; third < 3; ++third) {
                                const float part = ex2(-fminf(fmaxf(left - 14.0f * third, 0.0f), 14.0f));
                                const uint32_t f = half2_bits(part, part);
#pragma unroll
                                for (int e = 0; e < 32; ++e) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(y[e]) : "r"(f));
                            }
                            tmem_st_32x32b_x32(s_tmem + lanes + 32 * cc, y);
                        }
#pragma unroll 1
                        for (int cc = 0; cc < (anew ? 0 : C::kOutCols / 32); ++cc) {
                            tmem_ld_32x32b_x32(o_tmem + lanes + 32 * cc, y);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * down);
                            tmem_st_32x32b_x32(o_tmem + lanes + 32 * cc, y);
                        }
                        if (!ok) break;
                    }
                    if (!ok) break;
                    l += weight;
                    tmem_st_32x32b_x32(s_tmem + lanes + 32 * c, p);
                }
                if (!ok) break;
                if (anew && j > 0) {
                    // Adds O, complete up to the tile before, to the rounded sum, which is asked
                    // for ahead: local memory of 256 rows is more than L1 holds.
                    const bool first = j == kSpan;
                    const auto ask_sum = [&](float4 (&to)[8], int c) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) to[e] = first ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : get_sum(c + e);
                    };
                    float4 z[8];
                    ask_sum(z, 0);
                    ok = __all_sync(~0u, tile_wait(watch, &o_done[side], (n - 1) & 1));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const float old = first || m_sum == -INFINITY ? 0.0f : ex2(m_sum - m_before);
                    m_sum = m_before;
#pragma unroll 1
                    for (int c = 0; c < D / 4; c += 8) {
                        float4 ahead[8];
                        uint32_t y[32];
                        tmem_ld_32x32b_x32(o_tmem + lanes + 4 * c, y);
                        if (c + 8 < D / 4) ask_sum(ahead, c + 8);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            put_sum(c + e, make_float4(fmaf(z[e].x, old, __uint_as_float(y[4 * e])), fmaf(z[e].y, old, __uint_as_float(y[4 * e + 1])),
                                                       fmaf(z[e].z, old, __uint_as_float(y[4 * e + 2])),
                                                       fmaf(z[e].w, old, __uint_as_float(y[4 * e + 3]))));
                            z[e] = ahead[e];
                        }
                    }
                }
                tmem_wait_st();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * side + (n & 1)]);
            }
            first_tile += tiles;
            // (An item of one tile may have none for the second half: a phase for it would end with the
            // one before, whose end this warp could then miss.)
            if (units > 0) ok = ok && __all_sync(~0u, tile_wait(watch, &item_done[side], worked++ & 1));
            if (!ok) break;
            tcgen05_fence_after();
            // The rows' output: O (and the rounded sum) over L, zeros for a row that
            // sees no key.  A part of an item leaves O, m and l instead; where the halves
            // have shared the keys, the second one leaves them to the first.
            const bool summed = units > kSpan, whole_item = count == 1;
            const float old = !summed || m_sum == -INFINITY ? 0.0f : ex2(m_sum - m);
            uint8_t* slot_rows = q_rows + q_slot * kHalves * 2 * C::kQBytes;
            float4* other = reinterpret_cast<float4*>(slot_rows + 2 * C::kQBytes);  // [D / 4][128]: the second side's O, in the place of its rows
            float own_weight = 1.0f, other_weight = 0.0f;
            if (idle) {  // it has nothing to leave to anyone, but keeps to the others' turns
                if (!both && side == 1 && shared_items > 0) ok = __all_sync(~0u, tile_wait(watch, taken_over, (shared_items - 1) & 1));
                if (!ok) break;
                if (!both && lane == 0) mbar_arrive(side == 1 ? joined : taken_over);
                if ((C::kQSlots > 1 || (!both && side == 0)) && lane == 0) mbar_arrive(&q_empty[q_slot]);
                shared_items += !both;
                continue;
            }
            if (!both && side == 1) {
                // (The halves' units do not wait for one another: the first may be an item behind.)
                if (shared_items > 0) ok = __all_sync(~0u, tile_wait(watch, taken_over, (shared_items - 1) & 1));
                if (!ok) break;
                ++shared_items;
#pragma unroll 1
                for (int c = 0; c < D / 4; c += 8) {
                    uint32_t x[32];
                    tmem_ld_32x32b_x32(o_tmem + lanes + 4 * c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float4 y = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]),
                                               __uint_as_float(x[4 * e + 3]));
                        if (summed) {
                            const float4 z = get_sum(c + e);
                            y = make_float4(fmaf(z.x, old, y.x), fmaf(z.y, old, y.y), fmaf(z.z, old, y.z), fmaf(z.w, old, y.w));
                        }
                        // (Of a row without weights, TMEM may hold anything.)
                        other[(c + e) * kRows + r] = l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : y;
                    }
                }
                join_s[r] = make_float2(m, l);
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(joined);
                    if (C::kQSlots > 1) mbar_arrive(&q_empty[q_slot]);
                }
                continue;
            }
            if (!both) {
                ok = __all_sync(~0u, tile_wait(watch, joined, shared_items++ & 1));
                if (!ok) break;
                const float2 theirs = join_s[r];
                const float top = fmaxf(m, theirs.x);
                // (An l that is no number comes through, whatever its m.)
                own_weight = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2(m - top);
                other_weight = theirs.x == -INFINITY ? (theirs.y == 0.0f ? 0.0f : 1.0f) : ex2(theirs.x - top);
                if (l == 0.0f) own_weight = 0.0f;
                __syncwarp();
                if (lane == 0) mbar_arrive(taken_over);
                l = (own_weight == 0.0f ? 0.0f : own_weight * l) + (other_weight == 0.0f ? 0.0f : other_weight * theirs.y);
                m = top;
            }
            const float inverse = !whole_item ? 1.0f : inverse_of(l);
            const int part_row = (both ? side * kRows : 0) + r;
            // A block has two places: for the part of an item that began before, and of one that goes on behind.
            const auto part_at = [&](int i) { return parts + (int64_t)(i == 0 ? 2 * place + 1 : 2 * (place + i)) * C::kPart; };
            float* own = part_at(part_index);
            // Where there is room beside the next item's rows, whole rows are stored, by
            // way of the place of this item's; permuted so that a row's pieces lie in
            // different banks, as a column's do.
            constexpr bool kStaged = C::kQSlots > 1;
            float4* staged = reinterpret_cast<float4*>(slot_rows + side * 2 * C::kQBytes) + (warp & 3) * (D / 4) * 32;
            const auto put_out = [&](int c, float4 y) {
                if (kStaged) staged[c * 32 + (lane ^ (c & 7))] = y;
                else if (r < rows) *reinterpret_cast<float4*>(out + 4 * c) = y;
            };
#pragma unroll 1
            for (int c = 0; c < D / 4; c += 8) {
                uint32_t x[32];
                tmem_ld_32x32b_x32(o_tmem + lanes + 4 * c, x);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float4 y = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]),
                                           __uint_as_float(x[4 * e + 3]));
                    if (summed) {
                        const float4 z = get_sum(c + e);
                        y = make_float4(fmaf(z.x, old, y.x), fmaf(z.y, old, y.y), fmaf(z.z, old, y.z), fmaf(z.w, old, y.w));
                    }
                    if (!both) {
                        const float4 z = other[(c + e) * kRows + r];
                        if (own_weight == 0.0f) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        y = make_float4(fmaf(z.x, other_weight, y.x * own_weight), fmaf(z.y, other_weight, y.y * own_weight),
                                        fmaf(z.z, other_weight, y.z * own_weight), fmaf(z.w, other_weight, y.w * own_weight));
                    }
                    y = l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                  : make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
                    if (!whole_item) reinterpret_cast<float4*>(own)[(c + e) * (kHalves * kRows) + part_row] = y;
                    else put_out(c + e, y);
                }
            }
            bool there = whole_item;
            if (!whole_item) {
                // The last of the parts' warps to arrive joins its rows' parts, in order.
                own[kHalves * kRows * D + part_row] = m;
                own[kHalves * kRows * (D + 1) + part_row] = l;
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0) {
                    __threadfence();
                    // (Eight bits a warp.)
                    before = atomicAdd(arrivals + 2 * place + side, 1u << (8 * (warp & 3))) >> (8 * (warp & 3)) & 0xffu;
                    __threadfence();
                }
                there = __shfl_sync(~0u, before, 0) == static_cast<uint32_t>(count - 1);
                if (there) {
                    // Eight float4 of the row at a time, two parts' under way.
                    const auto part_m = [&](int i) { return __ldcg(part_at(i) + kHalves * kRows * D + part_row); };
                    const auto part_l = [&](int i) { return __ldcg(part_at(i) + kHalves * kRows * (D + 1) + part_row); };
                    float top = -INFINITY, total = 0.0f;
#pragma unroll 4
                    for (int i = 0; i < count; ++i) top = fmaxf(top, part_m(i));
                    // (An l that is no number comes through, whatever its m.)
                    const auto weigh = [&](float their, float their_l) { return their == -INFINITY ? (their_l == 0.0f ? 0.0f : 1.0f) : ex2(their - top); };
#pragma unroll 4
                    for (int i = 0; i < count; ++i) {
                        const float their_l = part_l(i);
                        total = fmaf(weigh(part_m(i), their_l), their_l, total);
                    }
                    const float over = total == 0.0f ? 0.0f : inverse_of(total);
#pragma unroll 1
                    for (int c = 0; c < D / 4; c += 8) {
                        float4 y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
                        for (int i = 0; i < count; ++i) {
                            const float4* from = reinterpret_cast<const float4*>(part_at(i)) + c * (kHalves * kRows) + part_row;
                            const float weight = weigh(part_m(i), part_l(i));
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float4 v = __ldcg(from + e * (kHalves * kRows));
                                y[e] = make_float4(fmaf(weight, v.x, y[e].x), fmaf(weight, v.y, y[e].y), fmaf(weight, v.z, y[e].z),
                                                   fmaf(weight, v.w, y[e].w));
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            put_out(c + e, total == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                                         : make_float4(y[e].x * over, y[e].y * over, y[e].z * over, y[e].w * over));
                    }
                }
            }
            if (kStaged && there) {
                __syncwarp();
                constexpr int kRowLanes = D / 4;  // 8 or 16 lanes a row
#pragma unroll 4
                for (int i = 0; i < 32; i += 32 / kRowLanes) {
                    const int row = i + lane / kRowLanes, c = lane % kRowLanes;
                    float* to = reinterpret_cast<float*>(__shfl_sync(~0u, reinterpret_cast<uintptr_t>(out), row));
                    const float4 v = staged[c * 32 + (row ^ (c & 7))];
                    if ((warp & 3) * 32 + row < rows) *reinterpret_cast<float4*>(to + 4 * c) = v;
                }
            }
            tcgen05_fence_before();
            if (kStaged || !both) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_empty[q_slot]);
            }
        }
    } else if (warp < kMmaWarp) {
        // ----------------------------------------------------- codes to fp16
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kConvertRegs));
        const int cw = warp - 4 * kHalves;
        const int page = 1 << g.shift;
        const uint32_t page_pieces = (static_cast<uint32_t>(g.cache.kv_heads) << g.shift) * (D / 16);  // 16-byte pieces of a page
        // Warps 8 and 9 convert K, 10 and 11 V, by the same code.
        const bool is_k = cw < 2;
        const int ct = tid & 63;
        const uint4* codes = reinterpret_cast<const uint4*>(is_k ? g.cache.k_codes : g.cache.v_codes);
        uint8_t* tiles_s = is_k ? k_tiles : v_tiles;
        uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
        // This thread's piece i of a tile: its key row and its place in the row.  Four
        // pieces a row and 64-element block at a time, where there are as many: eight
        // lanes then store to eight different bank groups.
        const auto row_of = [&](int i) {
            if (D == 128) return (i & 3) * 16 + (ct >> 2);
            if (D == 64) return i * 16 + (ct >> 2);
            if (D == 32) return i * 32 + (ct >> 1);
            return i < 4 ? i * 16 + (ct >> 2) : (i - 4) * 32 + (ct >> 1);
        };
        const auto piece_of = [&](int i) {
            if (D == 128) return (ct & 3) + 4 * (i >> 2);
            if (D == 64) return ct & 3;
            if (D == 32) return ct & 1;
            return i < 4 ? ct & 3 : 4 + (ct & 1);
        };
        bool ok = true;
        int n = 0;  // tiles of the items before
        for (int it = 0;; ++it) {
            ok = __all_sync(~0u, tile_wait(watch, &found_full[it % C::kItems], it / C::kItems & 1));
            if (!ok) break;
            const TreeItem now = items[it % C::kItems];
            const int keys = now.keys, tiles = now.tiles;
            if (tiles < 0) break;
            const int32_t* table = g.step.table + (int64_t)now.request * g.step.max_pages;
            const uint32_t head_pieces = (static_cast<uint32_t>(now.head) << g.shift) * (D / 16);
            // Loads are asked for where they stand: the page numbers of a tile two
            // tiles ahead, its codes and scales one.
            int32_t ids[C::kPieces], group_id = 0;  // pages of the pieces; of 16-key group ct in the first lanes
            uint4 w[C::kPieces];
            float ks = 0.0f, vs = -1.0f;            // the group's scales; -1: not there
            const auto page_of = [&](int j, int row) {  // of key row `row` of tile j; past the keys: some page
                const int key = min((now.tile0 + j) * C::kKeys + row, keys - 1);
                return keys > 0 ? load_now(table + (key >> g.shift)) : -1;
            };
            const auto ask_pages = [&](int j) {
#pragma unroll
                for (int i = 0; i < C::kPieces; ++i) ids[i] = page_of(j, row_of(i));
                if (is_k && ct < C::kGroups) group_id = page_of(j, 16 * ct);
            };
            const auto fetch = [&](int j) {  // tile j, whose pages are there; zeros where there is no key
#pragma unroll
                for (int i = 0; i < C::kPieces; ++i) {
                    const int key = (now.tile0 + j) * C::kKeys + row_of(i);
                    w[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (key < keys && static_cast<uint32_t>(ids[i]) < static_cast<uint32_t>(g.cache.pages))
                        w[i] = load_now(codes + (ids[i] * page_pieces + (head_pieces + (key & (page - 1)) * (D / 16) + piece_of(i))));
                }
                ks = 0.0f;
                vs = -1.0f;
                if (is_k && ct < C::kGroups && (now.tile0 + j) * C::kKeys + 16 * ct < keys) {
                    if (static_cast<uint32_t>(group_id) < static_cast<uint32_t>(g.cache.pages)) {
                        const int64_t from = (int64_t)group_id * g.cache.kv_heads + now.head;
                        ks = load_now(g.cache.k_scales + from);
                        vs = load_now(g.cache.v_scales + from);
                    } else {
                        report(watch, kSiteKv8Range);
                    }
                }
            };
            ask_pages(0);
            fetch(0);
            ask_pages(1);
#pragma unroll 1
            for (int j = 0; j < tiles; ++j) {
                const int tile = n + j, stage = tile % C::kStages;
                if (tile >= C::kStages) ok = __all_sync(~0u, tile_wait(watch, &empty[stage], (tile / C::kStages - 1) & 1));
                if (!ok) break;
                uint8_t* to_tile = tiles_s + stage * C::kKvBytes;
#pragma unroll
                for (int i = 0; i < C::kPieces; ++i) {
                    const int row = row_of(i), cc = piece_of(i), chunk = (cc & 3) * 2;
                    const uint32_t b[4] = {w[i].x ^ 0x80808080u, w[i].y ^ 0x80808080u, w[i].z ^ 0x80808080u, w[i].w ^ 0x80808080u};
                    uint8_t* line = to_tile + (cc >> 2) * (C::kKeys * 128) + row * 128;
                    *reinterpret_cast<uint4*>(line + ((chunk ^ (row & 7)) << 4)) =
                        make_uint4(codes_half2(b[0], 0x4140u), codes_half2(b[0], 0x4342u), codes_half2(b[1], 0x4140u), codes_half2(b[1], 0x4342u));
                    *reinterpret_cast<uint4*>(line + (((chunk + 1) ^ (row & 7)) << 4)) =
                        make_uint4(codes_half2(b[2], 0x4140u), codes_half2(b[2], 0x4342u), codes_half2(b[3], 0x4140u), codes_half2(b[3], 0x4342u));
                }
                if (is_k && ct < C::kGroups) {
                    float4 f = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);  // hides the group
                    if (vs >= kLeastScale && !isnan(fmaf(vs, 0.0f, ks))) {
                        // log2 vs and 1 / vs from an approximate logarithm a: with
                        // vs 2^-a = 1 + d, log2 vs = a + d log2 e and 1 / vs = 2^-a (1 - d),
                        // to d^2, about 2^-44.
                        const float a = lg2(vs), back = ex2(-a), d = fmaf(vs, back, -1.0f);
                        f = make_float4(ks, fmaf(d, kLog2e, a), fmaf(-d, back, back), 0.0f);
                    } else if (!(vs < 0.0f)) {
                        f = vs < kLeastScale && !isnan(ks) ? make_float4(ks, kZeroLog2, kZeroInverse, 0.0f)
                                                           : make_float4(0.0f, kNoNumberLog2, FLT_MAX, 0.0f);
                    }
                    info[(tile % C::kInfo) * C::kGroups + ct] = f;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[stage]);
                fetch(j + 1);
                ask_pages(j + 2);
            }
            if (!ok) break;
            n += tiles;
        }
    } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));  // (a warpgroup's four warps, by one instruction)
    if (warp < kMmaWarp + kHalves) {
        // ------------------------------------------------------ MMA issue
        // The whole warp keeps the loop, so that addresses stay in uniform registers (REDUX
        // leaves its result in one); one lane issues.
        const auto uniform = [](uint32_t x) { return __reduce_max_sync(~0u, x); };
        const bool leader = elect_one_sync();
        constexpr uint32_t s_desc = umma_idesc_f16(kRows, C::kKeys, false), o_desc = umma_idesc_f16(kRows, C::kOutCols, true);
        const uint32_t half = uniform(warp - kMmaWarp), half_tmem = uniform(tmem) + half * C::kHalfCols;
        const uint64_t qh = umma_desc_k_sw128(smem_u32(q_rows)), kt = umma_desc_k_sw128(smem_u32(k_tiles)),
                       vt = umma_desc_mn_sw128(smem_u32(v_tiles), C::kKeys * 128);
        const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, tile_wait(watch, bar, parity)); };
        const auto commit = [&](uint64_t* bar) {
            if (leader) umma_commit(bar);
        };
        uint32_t n = 0, count = 0, worked = 0;  // tiles of the items before; the half's units whose PV is issued; its items that had some
        bool ok = true;
        for (uint32_t it = 0; ok; ++it) {
            const uint32_t q_slot = it % C::kQSlots;
            if (!wait(&found_full[it % C::kItems], it / C::kItems & 1)) break;
            const TreeItem* item = items + it % C::kItems;
            const int tiles = item->tiles;
            const bool both = item->both != 0;
            if (tiles < 0 || !wait(&q_full[q_slot * kHalves], it / C::kQSlots & 1)) break;
            if (half && !wait(&q_full[q_slot * kHalves + 1], it / C::kQSlots & 1)) break;  // (as the softmax warps)
            const int units = both ? tiles : (tiles + 1 - static_cast<int>(half)) / 2;
            const uint32_t q_at = uniform((q_slot * kHalves + (both ? half : 0)) * (2 * C::kQBytes >> 4));
            // The tiles that are the other half's are let go of, in their turn.
            const auto pass = [&](uint64_t* full, uint64_t* empty, int tile) {
                const uint32_t at = n + tile, stage = at % C::kStages;
                if (!wait(&full[stage], (at / C::kStages) & 1)) return false;
                if (lane == 0) mbar_arrive(&empty[stage]);
                __syncwarp();
                return true;
            };
            // S of unit i, into the buffer that PV of the unit before the last one reads: MMAs of
            // unlike accumulators keep no order, so that one is waited for (an item's first:
            // all of the item before; of o_done, an item's last phase but one may not have been seen,
            // and would pass for the last).
            const auto scores = [&](int i) {
                if (!both && half && !pass(k_full, k_empty, 2 * i)) return false;
                const uint32_t tile = n + (both ? i : 2 * i + half), stage = uniform(tile % C::kStages), unit = count + (i > 0);
                if (!wait(&k_full[stage], (tile / C::kStages) & 1)) return false;
                if (i == 0 ? worked > 0 : unit >= 2)
                    if (!wait(i == 0 ? &item_done[half] : &o_done[half], (i == 0 ? worked - 1 : unit) & 1)) return false;
                tcgen05_fence_after();
                const uint64_t q = qh + q_at, k = kt + stage * (C::kKvBytes >> 4);
                const uint32_t s_tmem = half_tmem + uniform(unit & 1) * C::kKeys;
                if (leader) {
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int e = 0; e < D / 16; ++e)
                            umma_f16(s_tmem, q + (part == 0 ? C::kQBytes >> 4 : 0) + ((e >> 2) * (kRows * 128 >> 4) + 2 * (e & 3)),
                                     k + ((e >> 2) * (C::kKeys * 128 >> 4) + 2 * (e & 3)), s_desc, part > 0 || e > 0);
                }
                __syncwarp();
                commit(&s_full[2 * half + (unit & 1)]);
                commit(&k_empty[stage]);
                return both || half || 2 * i + 1 >= tiles || pass(k_full, k_empty, 2 * i + 1);
            };
            if (!both && half && units == 0) ok = pass(k_full, k_empty, 0) && pass(v_full, v_empty, 0);
#pragma unroll 1
            for (int i = -1; i < units && ok; ++i) {
                if (i + 1 < units) ok = scores(i + 1);
                if (i + 2 == units) {
                    if (ok && !both && half && (tiles & 1)) ok = pass(k_full, k_empty, tiles - 1);
                    commit(&q_empty[q_slot]);
                }
                if (i < 0) continue;
                if (ok && !both && half) ok = pass(v_full, v_empty, 2 * i);
                const uint32_t tile = n + (both ? i : 2 * i + half), stage = uniform(tile % C::kStages), buffer = uniform(count & 1);
                ok = ok && wait(&v_full[stage], (tile / C::kStages) & 1) && wait(&p_full[2 * half + buffer], (count >> 1) & 1);
                if (!ok) break;
                tcgen05_fence_after();
                const uint64_t v = vt + stage * (C::kKvBytes >> 4);
                const uint32_t p_tmem = half_tmem + buffer * C::kKeys, more = uniform(i % kSpan > 0);
                if (leader) {
#pragma unroll
                    for (int e = 0; e < C::kKeys / 16; ++e)
#pragma unroll
                        for (int part = 0; part < 2; ++part)
                            umma_f16_ta(half_tmem + 2 * C::kKeys, p_tmem + (e >> 1) * 32 + part * 16 + (e & 1) * 8, v + e * (2048 >> 4), o_desc,
                                        e > 0 || part > 0 ? 1u : more);
                }
                __syncwarp();
                commit(&v_empty[stage]);
                commit(&o_done[half]);
                ++count;
                if (!both && !half && 2 * i + 1 < tiles) ok = pass(v_full, v_empty, 2 * i + 1);
                if (!both && half && i + 1 == units && (tiles & 1)) ok = pass(v_full, v_empty, tiles - 1);
            }
            if (units == 0) commit(&q_empty[q_slot]);
            n += tiles;
            if (units > 0) {
                commit(&item_done[half]);
                ++worked;
            }
        }
        commit(&drained[half]);  // whatever was issued has completed before the block ends
        wait(&drained[half], 0);
    } else {
        // ------------------------------------------ the items and their rows
        const int pw = warp - kMmaWarp - kHalves;
        const int requests = g.step.requests, heads = g.cache.kv_heads;
        // A request's groups of 256 rows and what is left, its tiles, and its items' units in all.
        struct Cost {
            int full, rest, tiles;
            __device__ __forceinline__ int64_t of_full() const { return 2 * static_cast<int64_t>(tiles) + C::kItemCost; }
            __device__ __forceinline__ int64_t of_rest() const { return rest == 0 ? 0 : (rest > kRows ? 2 : 1) * static_cast<int64_t>(tiles) + C::kItemCost; }
        };
        const auto held_keys = [&](int s) {
            const int held = min(g.step.page_offsets[s + 1] - g.step.page_offsets[s], static_cast<int>(g.step.max_pages));
            return min(held << g.shift, g.step.lengths[s]);
        };
        const auto rows_of = [&](int s) {
            const int begin = max(0, g.step.token_offsets[s]), end = min(g.step.token_offsets[s + 1], static_cast<int>(g.step.tokens));
            return max(0, end - begin) * g.group;
        };
        const auto cost_of = [&](int s) {
            const int rows = rows_of(s);
            const int seen = max(0, min(held_keys(s), g.step.context[s] + rows / g.group));
            return Cost{rows / (kHalves * kRows), rows % (kHalves * kRows), max(1, (seen + C::kKeys - 1) / C::kKeys)};
        };
        int64_t all = 0;
        for (int s = lane; s < requests; s += 32) {
            const Cost c = cost_of(s);
            all += heads * (c.full * c.of_full() + c.of_rest());
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(~0u, all, d);
        // Shares: the first `blocks` blocks have one, block i the units from share(i) on.
        const int64_t blocks = max64(1, min64(gridDim.x, all / kLeastShare));
        const auto share = [&](int64_t i) { return all * i / blocks; };
        const auto first_at = [&](int64_t unit) { return (unit * blocks + all - 1) / all; };  // the first i whose share begins at or behind it
        const int64_t begin = blockIdx.x < blocks ? share(blockIdx.x) : all, end = blockIdx.x < blocks ? share(blockIdx.x + 1) : all;
        int s = -1, index = 0, count = 0, window = 0;  // the request, its next item, its items; where its search goes on
        int64_t base = 0, before = 0;                  // units before the request; before the window
        uint32_t done = 0;                             // requests of the window that are done with
        Cost cost = {};
        const auto advance = [&](int it) {
            TreeItem next = {};
            next.tiles = -1;
#pragma unroll 1
            while (true) {
                if (index >= count) {
                    // The next request that ends behind this block's share's beginning.
                    s = -1;
#pragma unroll 1
                    while (window < requests && before < end) {
                        Cost own = {};
                        if (window + lane < requests) own = cost_of(window + lane);
                        const int64_t units = heads * (own.full * own.of_full() + own.of_rest());
                        int64_t upto = units;
#pragma unroll
                        for (int d = 1; d < 32; d *= 2) {
                            const int64_t other = __shfl_up_sync(~0u, upto, d);
                            if (lane >= d) upto += other;
                        }
                        const uint32_t here = __ballot_sync(~0u, units > 0 && before + upto > begin) & ~done;
                        if (here != 0) {
                            const int hit = __ffs(here) - 1;
                            done |= (2u << hit) - 1;
                            s = window + hit;
                            base = before + __shfl_sync(~0u, upto - units, hit);
                            cost = Cost{__shfl_sync(~0u, own.full, hit), __shfl_sync(~0u, own.rest, hit), __shfl_sync(~0u, own.tiles, hit)};
                            break;
                        }
                        before += __shfl_sync(~0u, upto, 31);
                        window += 32;
                        done = 0;
                    }
                    if (s < 0 || base >= end) break;
                    count = heads * (cost.full + (cost.rest > 0));
                    // Its first item that ends behind the share's beginning.
                    const int64_t into = max64(0, begin - base), full = heads * (cost.full * cost.of_full());
                    index = static_cast<int>(into < full ? into / cost.of_full() : heads * cost.full + (into - full) / max64(1, cost.of_rest()));
                }
                const int group = index / heads, head = index - group * heads;
                const bool rest = group >= cost.full;
                const int64_t unit = base + (rest ? heads * (cost.full * cost.of_full()) + head * cost.of_rest() : index * cost.of_full());
                ++index;
                if (unit >= end) break;
                const int tokens_at = max(0, g.step.token_offsets[s]);
                next.head = head;
                next.row0 = tokens_at;
                next.first_row = group * (kHalves * kRows);
                next.rows = rest ? cost.rest : kHalves * kRows;
                next.both = next.rows > kRows;
                next.context = g.step.context[s];
                next.request = s;
                const int seen = next.context + token_of(next.first_row + next.rows - 1) + 1;  // by the last row
                next.keys = max(0, min(held_keys(s), seen));
                const int tiles = max(1, (next.keys + C::kKeys - 1) / C::kKeys), each = next.both ? 2 : 1;
                next.part = 0;
                next.parts = 1;
                next.place = 0;
                next.tile0 = 0;
                next.tiles = tiles;
                if (tiles <= kShortTiles && (static_cast<int64_t>(each) * tiles + C::kItemCost) * blocks <= 2 * all) {
                    const int64_t middle = unit + (static_cast<int64_t>(each) * tiles + C::kItemCost) / 2;
                    if (middle >= begin && middle < end) break;
                } else {
                    const int64_t first = unit + C::kItemCost;
                    const auto cut = [&](int64_t at) { return static_cast<int>(max64(0, min64(tiles, (at - first) / each))); };  // (towards zero: of those before, none)
                    const int from = cut(begin), to = cut(end);
                    if (from < to) {
                        const int64_t b0 = first_at(first + each) - 1, b1 = first_at(first + static_cast<int64_t>(each) * tiles) - 1;
                        next.place = static_cast<int>(b0);
                        next.parts = static_cast<int>(b1 - b0) + 1;
                        next.part = static_cast<int>(blockIdx.x - b0);
                        next.tile0 = from;
                        next.tiles = to - from;
                        break;
                    }
                }
                next.tiles = -1;
            }
            if (lane == 0) {
                items[it % C::kItems] = next;
                mbar_arrive(&found_full[it % C::kItems]);
            }
            __syncwarp();
        };
        bool ok = true;
        if (pw == 0) advance(0);
#pragma unroll 1
        for (int it = 0;; ++it) {
            const int q_slot = it % C::kQSlots;
            ok = __all_sync(~0u, tile_wait(watch, &found_full[it % C::kItems], it / C::kItems & 1));
            if (!ok) break;
            const TreeItem now = items[it % C::kItems];
            if (now.tiles < 0) break;
            if (it >= C::kQSlots) ok = __all_sync(~0u, tile_wait(watch, &q_empty[q_slot], (it / C::kQSlots - 1) & 1));
            if (!ok) break;
            // (Its phases wait for those who wait for them.)
            if (lane == 0) mbar_arrive(&q_empty[q_slot]);
            // Who is done with the slot's item before is done with its description, and those before it are
            // read by now.
            if (pw == 0) advance(it + 1);
            if (it > 0 && C::kQSlots > 1) {
#pragma unroll 1
                for (int half = 0; half < kHalves; ++half) {
                    const int at_half = q_slot * kHalves + half;
                    if (now.both || half == 0) put_rows(now, half, q_rows + at_half * 2 * C::kQBytes, power + at_half * kRows, pw, kHalves);
                    if (lane < 2) mbar_arrive(&q_full[at_half]);
                }
            }
        }
    }
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, kHalves * C::kHalfCols);
    }
    // The last block leaves the counters at zero, those of the parts also where a wait has
    // run out and some have not arrived.
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(taken, 1u) == gridDim.x - 1) {
            *taken = 0;
            for (int i = 0; i < kTreePlaces / 4; ++i) reinterpret_cast<uint4*>(arrivals)[i] = make_uint4(0, 0, 0, 0);
        }
    }
}

template <int D>
int run_tree(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl) {
    if (g.cache.pages > UINT32_MAX / (((int64_t)g.cache.kv_heads << g.shift) * (D / 16))) {
        set_error("leafq_kv8_tree_attention: code pools of 64 GiB and more are not supported for many rows");
        return LEAFQ_ERR_UNSUPPORTED;
    }
    const int64_t items = (g.step.tokens * g.group >> 8) + g.step.requests;  // of a kv head, at most
    if (items * g.cache.kv_heads > INT_MAX || g.step.tokens * g.group > INT_MAX) {
        set_error("leafq_kv8_tree_attention: too many rows");
        return LEAFQ_ERR_INVALID;
    }
    DeviceWatch watch;
    int st = device_watch(&watch);
    if (st) return st;
    const void* kernel = reinterpret_cast<const void*>(kv8_attend_tree_kernel<D>);
    static const int registers = [kernel] {
        cudaFuncAttributes a;
        return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers != TreeShape<D>::kLaunchRegs) {  // setmaxnreg would wait for registers that the launch does not have
        set_error("leafq_kv8_tree_attention: the kernel was built with " + std::to_string(registers) + " registers a thread, not " +
                  std::to_string(TreeShape<D>::kLaunchRegs));
        return LEAFQ_ERR_CUDA;
    }
    st = allow_smem(kernel, TreeShape<D>::kSmem, "leafq_kv8_tree_attention");
    if (st) return st;
    const int blocks = std::min(kTreeBlocks, sm_count());
    uint32_t* counters = static_cast<uint32_t*>(workspace) + kTileCounters;
    return launch(kv8_attend_tree_kernel<D>, dim3(static_cast<unsigned>(blocks)), dim3(TreeShape<D>::kThreads), TreeShape<D>::kSmem, s, pdl,
                  "leafq_kv8_tree_attention", g, watch, counters, counters + 4,
                  reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes));
}

}  // namespace

size_t kv8_tree_part_bytes(int dim) { return sizeof(float) * kTreePlaces * kHalves * kRows * (dim + 2); }

int launch_kv8_tree_tiles(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl) {
    switch (g.cache.dim) {
        case 32: return run_tree<32>(s, g, workspace, pdl);
        case 64: return run_tree<64>(s, g, workspace, pdl);
        case 96: return run_tree<96>(s, g, workspace, pdl);
        default: return run_tree<128>(s, g, workspace, pdl);
    }
}

}  // namespace leafq
