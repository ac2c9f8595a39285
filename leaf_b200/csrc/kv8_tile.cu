// Attention over the paged INT8 cache, many query rows (prompts, long chunks).
//
// Compiled as a whole program (build.py): setmaxnreg is ignored in relocatable
// device code.
#define LEAFQ_WHOLE_PROGRAM
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv8_attention.cuh"

namespace leafq {
namespace {

// An item is 128 query rows of one kv head of a request (rows r = token * group +
// head-in-group) over its keys in tiles.  Two persistent blocks share an SM, so
// that one's MMAs run under the other's softmax.  Roles:
//   warps 0-3  softmax: one row per thread (its TMEM lane), 32 scores at a time
//   warps 4-7  the items and their query rows; codes to fp16 (two warps K, two
//              V): 16-byte global loads a tile ahead, byte permutes,
//              128-byte-swizzled shared memory
//   warp 8     MMA issue (tcgen05.mma kind::f16, fp32 accumulators in TMEM)
// The softmax warps take registers that the others leave (setmaxnreg).  S has
// two buffers: the next tile's scores are computed under this tile's softmax.
// The arithmetic is the split form's: codes exact in fp16, fp32 operands as
// hi + lo halves, the V scale in the exponent.
//   S [128][keys] = Qhi K^T + Qlo K^T   Q and K K-major in shared memory
//   O [128][D]   += Phi V + Plo V       P from TMEM, V as stored (MN-major)
// Each 32 columns of S are replaced in place by 16 columns of P's hi pairs and
// 16 of its lo pairs.  Weights are 2^kTileLift times their value relative to a
// power of two that follows the row's maximum from below: 16 of them may sum up
// to kTileHighest, so that none passes 65504, fp16's largest, before the reference
// is raised and O rescaled.  The MMA's additions truncate,
// which adds up over long sums (8192 keys: 5.5e-6 of the result), so every
// kSpan tiles O is added to a rounded sum (in local memory) and starts anew -- and
// the lo halves of Q go first, while S is small.
//
// Bound: issue slots, of which 57 % are used (the tensor pipe is busy 21 % of the
// time): about a third go to the softmax (5 to 6 instructions a score), a fifth
// to rotating and splitting query rows, a sixth to the codes' conversion; the
// rest waits on hand-offs between the roles.  4 heads of 64, 8 queries a key: 64
// prompts of 512 tokens 360 us (191 TFLOP/s, twice that in the MMAs, since fp32
// operands are two halves); one of 8,192 tokens 612 us (449 TFLOP/s).  5 chunks
// of 100 to 1,500 tokens, 8 heads of 128, 3 queries a key, 83 us (252 TFLOP/s).
constexpr float kTileLift = 6.0f, kTileHighest = 49152.0f;
// Two kinds of pages need no test in the softmax (one a tile took 2 % of the time): what
// stands for their V scale does it.  Values of zero count in L as any other, as of scale
// 2^kZeroLog2, with a reference that stands kZeroAbove over their scores (below those of
// the scales that an append gives), which leaves their weights at 2^-37, zeros in fp16.
// (Where later scores are 2^12 times as heavy, and no other page's raise the reference,
// they come through as values below 2^-76.)  Scales that are no numbers: every key that
// a row sees weighs one, the reference is out of all others' reach, and L passes
// kNoNumber; a row that sees none of them keeps its own.
constexpr float kZeroLog2 = -83.0f, kZeroInverse = 0x1p83f, kZeroAbove = 43.0f;
constexpr float kNoNumberLog2 = 1e30f, kNoNumber = 3e38f;
// 1 / L: none for a row that sees no key, and for one that sees a scale that is no number.
__device__ __forceinline__ float inverse_of(float l) { return l == 0.0f ? 0.0f : l > kNoNumber ? NAN : __frcp_rn(l); }

// Where there are fewer items than half the blocks, each is cut into parts along
// the keys, of kPartTiles tiles or more; the last part to end joins them.
constexpr int kPartTiles = 4, kMostParts = 16;

// What the roles of a block need to know of an item: 128 query rows of one kv
// head of a request, and, where it is cut into parts, which one.  tiles < 0:
// there are no more.
struct TileItem {
    int row0, first_row, rows, context, keys, tiles, head, request;
    int tile0, parts, part, place;  // its first key tile; the parts' place in the workspace
};

template <int D>
struct TileShape {
    static constexpr int kRows = 128;
    static constexpr int kKeys = D <= 64 ? 96 : 64;
    static constexpr int kBlocks = (D + 63) / 64;        // 64-element (128-byte) column blocks
    static constexpr int kKStages = 2;
    static constexpr int kVStages = D <= 64 ? 2 : 1;
    static constexpr int kGroups = kKeys / 16;           // of keys that share a page for certain
    static constexpr int kInfo = 4;                      // ring of the groups' scales: a tile's are read while those of
                                                         // up to kKStages + 1 later tiles are written
    static constexpr int kQBytes = kBlocks * kRows * 128;
    static constexpr int kQSlots = D <= 64 ? 2 : 1;      // of query rows: the next item's beside this one's
    static constexpr int kItems = 3;                     // ring of their descriptions
    static constexpr int kKvBytes = kBlocks * kKeys * 128;
    static constexpr int kSpan = 512 / kKeys;            // tiles between O's additions to the rounded sum
    // Two warps convert K, two V.  Registers of the launch, of the softmax warps, of
    // the others: nine warps put five on one of the SM's four schedulers, so the
    // launch gives 96 a thread.  They belong to a scheduler: a softmax warp can take
    // only what the converting warp beside it, four warps on, has left.
    static constexpr int kThreads = 9 * 32;
    static constexpr int kLaunchRegs = 96, kSoftmaxRegs = 104, kOtherRegs = 88;
    static constexpr int kPieces = kKeys * D / 16 / 64;  // 16-byte pieces of a K (or V) tile per converting thread
    static constexpr int kOutCols = kBlocks * 64;        // O columns (those past D are not read)
    static constexpr uint32_t kTmemCols = 256;
    static constexpr size_t kSmem = kQSlots * 2 * kQBytes + (kKStages + kVStages) * kKvBytes + kInfo * kGroups * 16 +
                                    kItems * sizeof(TileItem) + kQSlots * kRows + (2 * kKStages + 2 * kVStages + 2 * kQSlots + kItems + 7) * 8 + 8;
    static_assert(kQSlots == 1 || kRows * D * 4 <= 2 * kQBytes, "the output goes through the place of the item's rows");
    static constexpr int kPart = kRows * (D + 2);        // floats of a part's result: O [D / 4][128][4], m [128], l [128]
    static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two blocks share the SM's shared memory");
    static_assert(2 * kKeys + kOutCols <= 256, "two blocks share the SM's 512 TMEM columns");
    static_assert(kSoftmaxRegs + kOtherRegs <= 2 * kLaunchRegs, "the split of what the launch gives each scheduler");
};

// The library's device error word and wait limit (leafq_device.cuh), which this
// file, compiled as a whole program, cannot name.
__device__ __forceinline__ void report(const DeviceWatch& w, unsigned site) {
    atomicCAS(w.error, 0u, (site << 16) | (blockIdx.x & 0xffffu));
}

// Bounded wait that other requests' range errors do not end.
__device__ __forceinline__ bool tile_wait(const DeviceWatch& w, uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long start = global_timer_ns();
    do {
        if (mbar_try_wait(bar, parity)) return true;
    } while (global_timer_ns() - start <= *static_cast<volatile const unsigned long long*>(w.limit_ns));
    report(w, kSiteKv8Tile);
    return false;
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

// Loads of read-only data that stay where they are written, ahead of their use.
__device__ __forceinline__ uint4 load_now(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float4 load_now(const float4* p) {
    float4 v;
    asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ int32_t load_now(const int32_t* p) {
    int32_t v;
    asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float load_now(const float* p) {
    float v;
    asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}

// An array that stays in local memory: its address, and 16 bytes of it.
__device__ __forceinline__ uint32_t local_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_local(p)); }
__device__ __forceinline__ float4 load_local(uint32_t at) {
    float4 v;
    asm volatile("ld.local.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void store_local(uint32_t at, float4 v) {
    asm volatile("st.local.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// kParts: some items are cut into parts (the code that joins them is left out of
// the other kernel, whose loops it would push out of the instruction cache:
// 64 prompts of 512 tokens 368 us without it, 379 us with it).
template <int D, bool kParts>
__global__ void __launch_bounds__(TileShape<D>::kThreads, 2)
kv8_attend_tile_kernel(const Kv8AttendArgs g, const DeviceWatch watch, uint32_t* taken, uint32_t* arrivals, float* parts,
                       int row_tiles, int splits) {
    using C = TileShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_rows = smem;  // [kQSlots]: hi, lo
    uint8_t* k_tiles = q_rows + C::kQSlots * 2 * C::kQBytes;
    uint8_t* v_tiles = k_tiles + C::kKStages * C::kKvBytes;
    float4* info = reinterpret_cast<float4*>(v_tiles + C::kVStages * C::kKvBytes);  // [kInfo][kGroups]: ks, log2 vs, 1 / vs
    TileItem* items = reinterpret_cast<TileItem*>(info + C::kInfo * C::kGroups);
    uint8_t* power = reinterpret_cast<uint8_t*>(items + C::kItems);  // [kQSlots][128]: of two, that a row was scaled down by (exponent bits)
    uint64_t* k_full = reinterpret_cast<uint64_t*>(power + C::kQSlots * C::kRows);
    uint64_t* k_empty = k_full + C::kKStages;
    uint64_t* v_full = k_empty + C::kKStages;
    uint64_t* v_empty = v_full + C::kVStages;
    uint64_t* s_full = v_empty + C::kVStages;    // by S buffer, as p_full
    uint64_t* p_full = s_full + 2;
    uint64_t* q_full = p_full + 2;               // by slot: an item's rows are there
    uint64_t* q_empty = q_full + C::kQSlots;     // its last scores are computed, its description read (its output written)
    uint64_t* found_full = q_empty + C::kQSlots; // by description: it is there
    uint64_t* o_done = found_full + C::kItems;   // PV of a tile has completed
    uint64_t* item_done = o_done + 1;            // all its MMAs have completed
    uint64_t* drained = item_done + 1;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drained + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kMmaWarp = 8;
    const auto token_of = [&](int row) { return static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(g.group)); };

    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it; dynamic shared memory starts there
        if (tid == 0) report(watch, kSiteKv8Tile);
        return;
    }
    if (warp == kMmaWarp) {
        if (lane == 0) {
            for (int i = 0; i < C::kKStages; ++i) {
                mbar_init(&k_full[i], 2);
                mbar_init(&k_empty[i], 1);
            }
            for (int i = 0; i < C::kVStages; ++i) {
                mbar_init(&v_full[i], 2);
                mbar_init(&v_empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&s_full[i], 1);
                mbar_init(&p_full[i], 4);
            }
            for (int i = 0; i < C::kQSlots; ++i) {
                mbar_init(&q_full[i], 4);
                mbar_init(&q_empty[i], 1 + 4);
            }
            for (int i = 0; i < C::kItems; ++i) mbar_init(&found_full[i], 1);
            mbar_init(o_done, 1);
            mbar_init(item_done, 1);
            mbar_init(drained, 1);
            fence_barrier_init();
        }
        __syncwarp();
        tmem_alloc(tmem_holder, C::kTmemCols);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_holder;
    const uint32_t o_tmem = tmem + 2 * C::kKeys;
    grid_dependency_wait();
    grid_launch_dependents();

    // Tiles are counted on over the items (n); barriers of per-tile and per-item
    // phases are waited for in order by every role.
    if (warp < 4) {
        // ------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        __align__(16) float o_sum[D];  // the rounded sum
        const uint32_t o_local = local_address(o_sum);
        const auto get_sum = [&](int c) { return load_local(o_local + 16 * c); };  // elements 4 c .. 4 c + 3 of a row
        const auto put_sum = [&](int c, float4 v) { store_local(o_local + 16 * c, v); };
        int n = 0;
        bool ok = true;
        for (int it = 0;; ++it) {
            const int q_slot = it % C::kQSlots;
            const TileItem* item = items + it % C::kItems;
            ok = ok && __all_sync(~0u, tile_wait(watch, &q_full[q_slot], it / C::kQSlots & 1));
            if (!ok) break;
            const int tiles = item->tiles, first_row = item->first_row, rows = item->rows, row0 = item->row0, context = item->context,
                      keys = item->keys, head = item->head, tile0 = kParts ? item->tile0 : 0;
            const int count = kParts ? item->parts : 1, part_index = kParts ? item->part : 0, place = kParts ? item->place : 0;
            const float factor = __uint_as_float(static_cast<uint32_t>(power[q_slot * C::kRows + tid]) << 23) * g.scale * kLog2e;
            if (tiles < 0) break;
            if (C::kQSlots == 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(q_empty);
            }
            const int r = tid;
            const int t = token_of(first_row + r), hq = (first_row + r) - t * g.group;
            const int pos = context + t;
            const bool seen = r < rows && pos >= 0 && (g.rotary == 0 || pos < g.table_rows);
            const int limit = seen ? min(keys, pos + 1) : 0;
            float* out = g.out + ((int64_t)row0 + t) * g.heads * D + (int64_t)(head * g.group + hq) * D;
            float m = -INFINITY, l = 0.0f, m_sum = -INFINITY;
            for (int j = 0; j < tiles; ++j, ++n) {
                const uint32_t s_tmem = tmem + (n & 1) * C::kKeys;
                ok = __all_sync(~0u, tile_wait(watch, &s_full[n & 1], (n >> 1) & 1));
                if (!ok) break;
                tcgen05_fence_after();
                const float4* scales = info + (n % C::kInfo) * C::kGroups;
                const int visible = limit - (tile0 + j) * C::kKeys;  // columns of this tile that the row sees
                const bool whole = __all_sync(~0u, visible >= C::kKeys);
                // 32 scores at a time, by rolled loops: the roles' loops have to stay in the
                // instruction cache side by side (unrolled, with all scores in registers,
                // the kernel took 1.5 times as long).  What is not seen is -inf.
                uint32_t x[32];
                const auto read = [&](int c) {
                    tmem_ld_32x32b_x32(s_tmem + lanes + 32 * c, x);
                    tmem_wait_ld();
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) x[e] = 32 * c + e >= visible ? 0xff800000u : x[e];
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
                const bool anew = j % C::kSpan == 0;
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
                            ok = __all_sync(~0u, tile_wait(watch, o_done, (n - 1) & 1));
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
                    // Adds O, complete up to the tile before, to the rounded sum.
                    ok = __all_sync(~0u, tile_wait(watch, o_done, (n - 1) & 1));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const bool first = j == C::kSpan;
                    const float old = first || m_sum == -INFINITY ? 0.0f : ex2(m_sum - m_before);
                    m_sum = m_before;
#pragma unroll 1
                    for (int c = 0; c < D / 4; c += 8) {
                        float4 z[8];
                        uint32_t y[32];
                        tmem_ld_32x32b_x32(o_tmem + lanes + 4 * c, y);
#pragma unroll
                        for (int e = 0; e < 8; ++e) z[e] = first ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : get_sum(c + e);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            put_sum(c + e, make_float4(fmaf(z[e].x, old, __uint_as_float(y[4 * e])), fmaf(z[e].y, old, __uint_as_float(y[4 * e + 1])),
                                                       fmaf(z[e].z, old, __uint_as_float(y[4 * e + 2])),
                                                       fmaf(z[e].w, old, __uint_as_float(y[4 * e + 3]))));
                    }
                }
                tmem_wait_st();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[n & 1]);
            }
            ok = ok && __all_sync(~0u, tile_wait(watch, item_done, it & 1));
            if (!ok) break;
            tcgen05_fence_after();
            // The rows' output: O (and the rounded sum) over L, zeros for a row that
            // sees no key.  A part of an item leaves O, m and l instead.
            const bool summed = tiles > C::kSpan, whole_item = !kParts || count == 1;
            const float old = !summed || m_sum == -INFINITY ? 0.0f : ex2(m_sum - m);
            const float inverse = !whole_item ? 1.0f : inverse_of(l);
            float* own = parts + (int64_t)(place + part_index) * C::kPart;
            // Where there is room beside the next item's rows, whole rows are stored, by
            // way of the place of this item's; permuted so that a row's pieces lie in
            // different banks, as a column's do.
            constexpr bool kStaged = C::kQSlots > 1;
            float4* staged = reinterpret_cast<float4*>(q_rows + q_slot * 2 * C::kQBytes) + warp * (D / 4) * 32;
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
                    y = l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                  : make_float4(y.x * inverse, y.y * inverse, y.z * inverse, y.w * inverse);
                    if (kParts && !whole_item) reinterpret_cast<float4*>(own)[(c + e) * C::kRows + tid] = y;
                    else put_out(c + e, y);
                }
            }
            bool there = whole_item;
            if (kParts && !whole_item) {
                // The last of the parts' warps to arrive joins its rows' parts, in order.
                own[C::kRows * D + tid] = m;
                own[C::kRows * (D + 1) + tid] = l;
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0) {
                    __threadfence();
                    before = atomicAdd(arrivals + 4 * (place / splits) + warp, 1u);
                    __threadfence();
                }
                there = __shfl_sync(~0u, before, 0) == static_cast<uint32_t>(count - 1);
                if (there) {
                    const float* first = parts + (int64_t)place * C::kPart;
                    float top = -INFINITY, total = 0.0f;
#pragma unroll 1
                    for (int i = 0; i < count; ++i) top = fmaxf(top, __ldcg(first + i * C::kPart + C::kRows * D + tid));
#pragma unroll 1
                    for (int i = 0; i < count; ++i) {
                        const float* from = first + i * C::kPart;
                        const float their = __ldcg(from + C::kRows * D + tid), part_l = __ldcg(from + C::kRows * (D + 1) + tid);
                        // (An l that is no number comes through, whatever its m.)
                        const float weight = their == -INFINITY ? (part_l == 0.0f ? 0.0f : 1.0f) : ex2(their - top);
                        total = fmaf(weight, part_l, total);
#pragma unroll 4
                        for (int c = 0; c < D / 4; ++c) {
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(from) + c * C::kRows + tid);
                            const float4 z = i == 0 ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : get_sum(c);
                            put_sum(c, make_float4(fmaf(weight, v.x, z.x), fmaf(weight, v.y, z.y), fmaf(weight, v.z, z.z), fmaf(weight, v.w, z.w)));
                        }
                    }
                    const float over = inverse_of(total);
#pragma unroll 4
                    for (int c = 0; c < D / 4; ++c) {
                        float4 y = get_sum(c);
                        y = total == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(y.x * over, y.y * over, y.z * over, y.w * over);
                        put_out(c, y);
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
                    if (warp * 32 + row < rows) *reinterpret_cast<float4*>(to + 4 * c) = v;
                }
            }
            tcgen05_fence_before();
            if (kStaged) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_empty[q_slot]);
            }
        }
    } else if (warp < kMmaWarp) {
        // ------------------------------- the items, their rows, codes to fp16
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
        const int cw = warp - 4;
        const int page = 1 << g.shift;
        const uint32_t page_pieces = (static_cast<uint32_t>(g.cache.kv_heads) << g.shift) * (D / 16);  // 16-byte pieces of a page

        // Items: row tiles x kv heads, those of a request that see most keys first.
        // Request s may have row tiles floor(token_offsets[s] * group / 128) + s and
        // on: enough of them.  A block's first item is its own number; warp 4 takes
        // the next ones from a counter that all blocks share, while the last tile of
        // the item before is on its way, and tells the other three.
        const uint32_t total = static_cast<uint32_t>(row_tiles) * g.cache.kv_heads * splits;
        bool first_take = true;
        const auto advance = [&](int it) {
            TileItem next = {};
#pragma unroll 1
            while (true) {
                uint32_t id = blockIdx.x;
                if (!first_take) {
                    if (lane == 0) id = gridDim.x + atomicAdd(taken, 1u);
                    id = __shfl_sync(~0u, id, 0);
                }
                first_take = false;
                next.tiles = -1;
                if (id >= total) break;
                const uint32_t whole = kParts ? id / static_cast<uint32_t>(splits) : id, group_of = whole / static_cast<uint32_t>(g.cache.kv_heads);
                if (kParts) {
                    next.part = static_cast<int>(id - whole * splits);
                    next.place = static_cast<int>(whole * splits);
                }
                const int index = row_tiles - 1 - static_cast<int>(group_of);
                next.head = static_cast<int>(whole - group_of * g.cache.kv_heads);
                int s = 0;
#pragma unroll 1
                for (int left = g.step.requests; left > 1;) {
                    const int step = (left + 31) >> 5, at = s + lane * step;
                    const bool below = lane * step < left && (g.step.token_offsets[at] * g.group >> 7) + at <= index;
                    const int hit = max(__popc(__ballot_sync(~0u, below)) - 1, 0);
                    s += hit * step;
                    left = min(step, left - hit * step);
                }
                const int begin = max(0, g.step.token_offsets[s]), end = min(g.step.token_offsets[s + 1], static_cast<int>(g.step.tokens));
                const int new_rows = max(0, end - begin) * g.group;
                const int tile_index = index - ((begin * g.group >> 7) + s);
                if (tile_index < 0 || tile_index * C::kRows >= new_rows) continue;
                next.row0 = begin;
                next.first_row = tile_index * C::kRows;
                next.rows = min(C::kRows, new_rows - next.first_row);
                next.context = g.step.context[s];
                next.request = s;
                const int held = min(g.step.page_offsets[s + 1] - g.step.page_offsets[s], static_cast<int>(g.step.max_pages));
                const int seen = next.context + token_of(next.first_row + next.rows - 1) + 1;  // by the last row
                next.keys = max(0, min(min(held << g.shift, g.step.lengths[s]), seen));
                // (Without keys, a tile that is all hidden.)
                const int tiles = max(1, (next.keys + C::kKeys - 1) / C::kKeys);
                next.tiles = tiles;
                if (kParts) {
                    next.parts = min(splits, max(1, tiles / kPartTiles));
                    if (next.part >= next.parts) continue;
                    next.tile0 = tiles * next.part / next.parts;
                    next.tiles = tiles * (next.part + 1) / next.parts - next.tile0;
                }
                break;
            }
            if (lane == 0) {
                items[it % C::kItems] = next;
                mbar_arrive(&found_full[it % C::kItems]);
            }
            __syncwarp();
        };
        // Lanes of a row: D / 8, eight values each (a rotation pair's quarters).
        constexpr int kLanes = D / 8;  // 4, 8, 12, 16
        constexpr int kAtOnce = 32 / kLanes, kPass = 4 * kAtOnce;
        constexpr int kTurns = (C::kRows + kPass - 1) / kPass;
        const int sub = lane / kLanes, part = lane - sub * kLanes;
        const int half = g.rotary >> 1;
        const bool turned = 4 * part < half;
        const int at = turned ? 4 * part : 2 * half + 4 * (part - half / 4);
        const int to = turned ? at + half : at + ((D - 2 * half) >> 1);
        // Loads run two turns ahead; rotated, scaled by the row's power of two, split,
        // stored swizzled.
        const int step_t = kPass / g.group, step_h = kPass - step_t * g.group;
        const auto put_rows = [&](const TileItem& next, uint8_t* q_hi, uint8_t* powers) {
            float4 a, b, cs, sn, a1, b1, cs1, sn1;  // this turn's, the next one's
            a = b = cs = sn = a1 = b1 = cs1 = sn1 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int r0 = next.first_row + cw * kAtOnce + sub;
            int t = token_of(r0), hq = r0 - t * g.group;  // of the row two turns ahead
#pragma unroll 1
            for (int i = -2; i < kTurns; ++i) {
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
                if (sub < kAtOnce && (i + 2) * kPass + cw * kAtOnce + sub < next.rows) {
                    const float* src = g.q + ((int64_t)next.row0 + t) * g.q_stride + (int64_t)(next.head * g.group + hq) * D;
                    a1 = load_now(reinterpret_cast<const float4*>(src + at));
                    b1 = load_now(reinterpret_cast<const float4*>(src + to));
                    if (turned) {
                        int64_t pos = (int64_t)next.context + t;
                        if (pos < 0 || pos >= g.table_rows) {
                            if (part == 0) report(watch, kSiteKv8Range);
                            pos = 0;
                        }
                        cs1 = load_now(reinterpret_cast<const float4*>(g.cos_table + pos * half + at));
                        sn1 = load_now(reinterpret_cast<const float4*>(g.sin_table + pos * half + at));
                    }
                }
                t += step_t;
                hq += step_h;
                if (hq >= g.group) {
                    hq -= g.group;
                    ++t;
                }
                if (i < 0) continue;
                const int r = i * kPass + cw * kAtOnce + sub;
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
                if (sub < kAtOnce && r < C::kRows) {
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
                        const int offset = (d >> 6) * (C::kRows * 128) + r * 128 + ((((d & 63) >> 3) ^ (r & 7)) << 4) + (d & 4) * 2;
                        *reinterpret_cast<uint2*>(q_hi + offset) = make_uint2(hi[0], hi[1]);
                        *reinterpret_cast<uint2*>(q_hi + C::kQBytes + offset) = make_uint2(lo[0], lo[1]);
                    }
                }
            }
        };
        // Warps 4 and 5 convert K, 6 and 7 V, by the same code.
        const bool is_k = cw < 2;
        const int ct = tid & 63, stages = is_k ? C::kKStages : C::kVStages;
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
        // (Every piece of work stands once: the roles' code shares the instruction
        // cache.  Turn -1 only finds the first item.)
        for (int it = -1;; ++it) {
            TileItem now = {};
            const int q_slot = it % C::kQSlots;
            if (it >= 0) {
                ok = __all_sync(~0u, tile_wait(watch, &found_full[it % C::kItems], it / C::kItems & 1));
                if (!ok) break;
                now = items[it % C::kItems];
                if (it >= C::kQSlots) ok = __all_sync(~0u, tile_wait(watch, &q_empty[q_slot], (it / C::kQSlots - 1) & 1));
                if (!ok) break;
            }
            const int keys = now.keys, tiles = now.tiles;
            if (tiles < 0) {
                if (lane == 0) mbar_arrive(&q_full[q_slot]);
                break;
            }
            const int32_t* table = g.step.table + (int64_t)now.request * g.step.max_pages;
            const uint32_t head_pieces = (static_cast<uint32_t>(now.head) << g.shift) * (D / 16);
            // Loads are asked for where they stand: the page numbers of a tile two
            // tiles ahead, its codes and scales one.
            int32_t ids[C::kPieces], group_id = 0;  // pages of the pieces; of 16-key group ct in the first lanes
            uint4 w[C::kPieces];
            float ks = 0.0f, vs = -1.0f;            // the group's scales; -1: not there
            const auto page_of = [&](int j, int row) {  // of key row `row` of tile j; past the keys: some page
                const int key = min(((kParts ? now.tile0 : 0) + j) * C::kKeys + row, keys - 1);
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
                    const int key = ((kParts ? now.tile0 : 0) + j) * C::kKeys + row_of(i);
                    w[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (key < keys && static_cast<uint32_t>(ids[i]) < static_cast<uint32_t>(g.cache.pages))
                        w[i] = load_now(codes + (ids[i] * page_pieces + (head_pieces + (key & (page - 1)) * (D / 16) + piece_of(i))));
                }
                ks = 0.0f;
                vs = -1.0f;
                if (is_k && ct < C::kGroups && ((kParts ? now.tile0 : 0) + j) * C::kKeys + 16 * ct < keys) {
                    if (static_cast<uint32_t>(group_id) < static_cast<uint32_t>(g.cache.pages)) {
                        const int64_t from = (int64_t)group_id * g.cache.kv_heads + now.head;
                        ks = load_now(g.cache.k_scales + from);
                        vs = load_now(g.cache.v_scales + from);
                    } else {
                        report(watch, kSiteKv8Range);
                    }
                }
            };
            if (it >= 0) ask_pages(0);
            if (it >= 0) {
                put_rows(now, q_rows + q_slot * 2 * C::kQBytes, power + q_slot * C::kRows);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[q_slot]);
                fetch(0);
                ask_pages(1);
            }
#pragma unroll 1
            for (int j = it >= 0 ? 0 : -1; j < tiles || j < 0; ++j) {
                if (cw == 0 && j == tiles - 1) advance(it + 1);
                if (j < 0) break;
                const int tile = n + j, stage = tile % stages;
                if (tile >= stages) ok = __all_sync(~0u, tile_wait(watch, &empty[stage], (tile / stages - 1) & 1));
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
        // ------------------------------------------------------ MMA issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
        // The whole warp keeps the loop, so that addresses stay in uniform registers;
        // one lane issues.
        const bool leader = elect_one_sync();
        constexpr uint32_t s_desc = umma_idesc_f16(C::kRows, C::kKeys, false), o_desc = umma_idesc_f16(C::kRows, C::kOutCols, true);
        const uint64_t qh = umma_desc_k_sw128(smem_u32(q_rows)), ql = qh + (C::kQBytes >> 4),
                       kt = umma_desc_k_sw128(smem_u32(k_tiles)), vt = umma_desc_mn_sw128(smem_u32(v_tiles), C::kKeys * 128);
        const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, tile_wait(watch, bar, parity)); };
        const auto commit = [&](uint64_t* bar) {
            if (leader) umma_commit(bar);
        };
        // S of tile n, into the buffer that PV of tile n - 2 reads: MMAs of
        // unlike accumulators keep no order, so that one is waited for (an
        // item's first: PV of tile n - 1, which has been issued before).
        const auto scores = [&](int n, bool first, int q_at) {
            const int stage = n % C::kKStages;
            if (!wait(&k_full[stage], (n / C::kKStages) & 1)) return false;
            if (n >= (first ? 1 : 2) && !wait(o_done, (first ? n - 1 : n) & 1)) return false;
            tcgen05_fence_after();
            const uint64_t k = kt + stage * (C::kKvBytes >> 4);
            const uint32_t s_tmem = tmem + (n & 1) * C::kKeys;
            if (leader) {
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        umma_f16(s_tmem, (part == 0 ? ql : qh) + q_at + ((i >> 2) * (C::kRows * 128 >> 4) + 2 * (i & 3)),
                                 k + ((i >> 2) * (C::kKeys * 128 >> 4) + 2 * (i & 3)), s_desc, part > 0 || i > 0);
            }
            __syncwarp();
            commit(&k_empty[stage]);
            commit(&s_full[n & 1]);
            return true;
        };
        int n = 0;
        bool ok = true;
        for (int it = 0; ok; ++it) {
            const int q_slot = it % C::kQSlots, q_at = q_slot * (2 * C::kQBytes >> 4);
            if (!wait(&q_full[q_slot], it / C::kQSlots & 1)) break;
            const int tiles = items[it % C::kItems].tiles;
            if (tiles < 0) break;
#pragma unroll 1
            for (int j = -1; j < tiles && ok; ++j) {
                if (j + 1 < tiles) {
                    ok = scores(n + (j >= 0), j < 0, q_at);
                    if (j + 2 == tiles) commit(&q_empty[q_slot]);
                }
                if (j < 0) continue;
                const int stage = n % C::kVStages;
                ok = ok && wait(&v_full[stage], (n / C::kVStages) & 1) && wait(&p_full[n & 1], (n >> 1) & 1);
                if (!ok) break;
                tcgen05_fence_after();
                const uint64_t v = vt + stage * (C::kKvBytes >> 4);
                const uint32_t p_tmem = tmem + (n & 1) * C::kKeys, more = j % C::kSpan > 0;
                if (leader) {
#pragma unroll
                    for (int i = 0; i < C::kKeys / 16; ++i)
#pragma unroll
                        for (int part = 0; part < 2; ++part)
                            umma_f16_ta(o_tmem, p_tmem + (i >> 1) * 32 + part * 16 + (i & 1) * 8, v + i * (2048 >> 4), o_desc,
                                        i > 0 || part > 0 ? 1u : more);
                }
                __syncwarp();
                commit(&v_empty[stage]);
                commit(o_done);
                ++n;
            }
            commit(item_done);
        }
        commit(drained);  // whatever was issued has completed before the block ends
        wait(drained, 0);
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
    // The last block leaves the counters at zero, those of the parts also where a wait has
    // run out and some have not arrived.  (By one thread: with all of them, behind a
    // barrier, 256 rows over 8,000 keys took 110 us instead of 104.)
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(taken + 1, 1u) == gridDim.x - 1) {
            taken[0] = taken[1] = 0;
            if (kParts)
                for (int i = 0; i < row_tiles * g.cache.kv_heads; ++i) reinterpret_cast<uint4*>(arrivals)[i] = make_uint4(0, 0, 0, 0);
        }
    }
}

template <int D, bool kParts>
int start_tile(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, int64_t row_tiles, int splits, bool pdl);

template <int D>
int run_tile(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl) {
    const int64_t row_tiles = (g.step.tokens * g.group >> 7) + g.step.requests;
    if (g.cache.pages > UINT32_MAX / (((int64_t)g.cache.kv_heads << g.shift) * (D / 16))) {
        set_error("leafq_kv8_attention: code pools of 64 GiB and more are not supported for prompts");
        return LEAFQ_ERR_UNSUPPORTED;
    }
    if (row_tiles * g.cache.kv_heads > INT_MAX || g.step.tokens * g.group > INT_MAX) {
        set_error("leafq_kv8_attention: too many rows");
        return LEAFQ_ERR_INVALID;
    }
    const int splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMostParts, kTileBlocks / (row_tiles * g.cache.kv_heads))));
    return splits > 1 ? start_tile<D, true>(s, g, workspace, row_tiles, splits, pdl)
                      : start_tile<D, false>(s, g, workspace, row_tiles, 1, pdl);
}

template <int D, bool kParts>
int start_tile(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, int64_t row_tiles, int splits, bool pdl) {
    DeviceWatch watch;
    int st = device_watch(&watch);
    if (st) return st;
    const void* kernel = reinterpret_cast<const void*>(kv8_attend_tile_kernel<D, kParts>);
    static const int registers = [kernel] {
        cudaFuncAttributes a;
        return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers != TileShape<D>::kLaunchRegs) {  // setmaxnreg would wait for registers that the launch does not have
        set_error("leafq_kv8_attention: the tile kernel was built with " + std::to_string(registers) + " registers a thread, not " +
                  std::to_string(TileShape<D>::kLaunchRegs));
        return LEAFQ_ERR_CUDA;
    }
    st = allow_smem(kernel, TileShape<D>::kSmem, "leafq_kv8_attention");
    if (st) return st;
    const int64_t blocks = std::min<int64_t>(row_tiles * g.cache.kv_heads * splits, 2 * (int64_t)sm_count());
    uint32_t* counters = static_cast<uint32_t*>(workspace) + kTileCounters;
    return launch(kv8_attend_tile_kernel<D, kParts>, dim3(static_cast<unsigned>(blocks)),
                  dim3(TileShape<D>::kThreads), TileShape<D>::kSmem, s, pdl, "leafq_kv8_attention", g, watch,
                  counters, counters + 4, reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes),
                  static_cast<int>(row_tiles), splits);
}

}  // namespace

size_t kv8_tile_part_bytes(int dim) { return sizeof(float) * kTileBlocks * 128 * (dim + 2); }

int launch_kv8_tiles(cudaStream_t s, const Kv8AttendArgs& g, void* workspace, bool pdl) {
    switch (g.cache.dim) {
        case 32: return run_tile<32>(s, g, workspace, pdl);
        case 64: return run_tile<64>(s, g, workspace, pdl);
        case 96: return run_tile<96>(s, g, workspace, pdl);
        default: return run_tile<128>(s, g, workspace, pdl);
    }
}

}  // namespace leafq
