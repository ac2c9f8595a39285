// Attention over the paged INT8 cache, many query rows (prompts, long chunks).
//
// Compiled as a whole program (build.py): setmaxnreg is ignored in relocatable
// device code.
#define LEAFQ_WHOLE_PROGRAM
#include <type_traits>

#include "kv8_attention.cuh"

namespace leafq {
namespace {

// A block owns 128 query
// rows of one kv head of a request (rows r = token * group + head-in-group),
// walks the keys in tiles, and two blocks share an SM, so that one's MMAs run
// under the other's softmax.  Roles:
//   warps 0-3  softmax: one row per thread (its TMEM lane), a tile's scores in
//              registers
//   warps 4-6  codes to fp16: 16-byte global loads a tile ahead, byte
//              permutes, 128-byte-swizzled shared memory
//   warp 7     MMA issue (kind::f16, fp32 accumulators in TMEM)
// The softmax warps take registers that the others leave (setmaxnreg).  S has
// two buffers: the next tile's scores are computed under this tile's softmax.
// The arithmetic is the split form's: codes exact in fp16, fp32 operands as
// hi + lo halves, the V scale in the exponent.
//   S [128][keys] = Qhi K^T + Qlo K^T   Q and K K-major in shared memory
//   O [128][D]   += Phi V + Plo V       P from TMEM, V as stored (MN-major)
// Each 32 columns of S are replaced in place by 16 columns of P's hi pairs and
// 16 of its lo pairs.  O is rescaled only when a row's maximum grows by more
// than 2^kSlack since its reference was taken: weights then stay below
// 2^(kTileLift + kSlack) < 65504, fp16's largest.  The MMA's additions truncate,
// which adds up over long sums (8192 keys: 5.5e-6 of the result), so every
// kSpan keys O is added to a rounded sum (in local memory) and starts anew
// -- and the lo halves of Q go first, while S is small.
constexpr float kTileLift = 6.0f, kSlack = 8.0f;

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
    static constexpr int kKvBytes = kBlocks * kKeys * 128;
    static constexpr int kSpan = 512 / kKeys;            // tiles between O's additions to the rounded sum
    static constexpr int kThreads = 256;
    static constexpr int kSoftmaxRegs = 168, kOtherRegs = 88;
    static constexpr int kConverters = 96;
    static constexpr int kAllPieces = kKeys * D / 16;    // 16-byte pieces of a K (or V) tile
    static constexpr int kPieces = (kAllPieces + kConverters - 1) / kConverters;
    static constexpr int kOutCols = kBlocks * 64;        // O columns (those past D are not read)
    static constexpr uint32_t kTmemCols = 256;
    static constexpr bool kSumInSmem = D <= 64;          // else in local memory
    static constexpr int kSumBytes = kSumInSmem ? kRows * D * 4 : kRows * 4;  // (it also takes the rows' factors first)
    static constexpr size_t kSmem = 2 * kQBytes + (kKStages + kVStages) * kKvBytes + kSumBytes + kInfo * kGroups * 16 +
                                    (2 * kKStages + 2 * kVStages + 7) * 8 + 8;
    static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two blocks share the SM's shared memory");
    static_assert(2 * kKeys + kOutCols <= 256, "two blocks share the SM's 512 TMEM columns");
    static_assert(2 * kQBytes >= kRows * D * 4, "the output leaves through Q's shared memory");
    static_assert(128 * (kSoftmaxRegs + kOtherRegs) == kThreads * 128, "the split of what the launch gives (128 a thread)");
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
    for (uint32_t spins = 1;; ++spins) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spins & 255u) == 0u && global_timer_ns() - start > *static_cast<volatile const unsigned long long*>(w.limit_ns)) {
            report(w, kSiteKv8Tile);
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

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int D>
__global__ void __launch_bounds__(TileShape<D>::kThreads, 2) kv8_attend_tile_kernel(const Kv8AttendArgs g, const DeviceWatch watch, int row_tiles) {
    using C = TileShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* q_hi = smem;
    uint8_t* q_lo = q_hi + C::kQBytes;
    uint8_t* k_tiles = q_lo + C::kQBytes;
    uint8_t* v_tiles = k_tiles + C::kKStages * C::kKvBytes;
    float4* sum_s = reinterpret_cast<float4*>(v_tiles + C::kVStages * C::kKvBytes);  // [D / 4][128]
    float* factor_s = reinterpret_cast<float*>(sum_s);                              // [128], before the first sum
    float4* info = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(sum_s) + C::kSumBytes);  // [kInfo][kGroups]: ks, log2 vs, 1 / vs
    uint64_t* k_full = reinterpret_cast<uint64_t*>(info + C::kInfo * C::kGroups);
    uint64_t* k_empty = k_full + C::kKStages;
    uint64_t* v_full = k_empty + C::kKStages;
    uint64_t* v_empty = v_full + C::kVStages;
    uint64_t* s_full = v_empty + C::kVStages;  // by S buffer, as p_full
    uint64_t* p_full = s_full + 2;
    uint64_t* o_done = p_full + 2;             // PV of a tile has completed
    uint64_t* drained = o_done + 1;
    uint64_t* q_full = drained + 1;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(q_full + 1);
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

    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it; dynamic shared memory starts there
        if (tid == 0) report(watch, kSiteKv8Tile);
        return;
    }
    if (warp == 7) {
        if (lane == 0) {
            for (int i = 0; i < C::kKStages; ++i) {
                mbar_init(&k_full[i], 3);
                mbar_init(&k_empty[i], 1);
            }
            for (int i = 0; i < C::kVStages; ++i) {
                mbar_init(&v_full[i], 3);
                mbar_init(&v_empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&s_full[i], 1);
                mbar_init(&p_full[i], 4);
            }
            mbar_init(o_done, 1);
            mbar_init(drained, 1);
            mbar_init(q_full, 4);
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

    if (warp < 4) {
        // ------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
        {
            // The warp's 32 rows: D / 8 lanes per row, eight values each, all asked
            // for before the first is used, rotated, scaled by the row's power of
            // two, split, stored swizzled.
            constexpr int kLanes = D / 8;  // 4, 8, 12, 16
            constexpr int kAtOnce = 32 / kLanes, kTurns = 32 / kAtOnce, kBatch = kTurns < 4 ? kTurns : 4;
            const int sub = lane / kLanes, i = lane - sub * kLanes;
            const int half = g.rotary >> 1;
            const bool turned = 4 * i < half;
            const int at = turned ? 4 * i : 2 * half + 4 * (i - half / 4);
            const int to = turned ? at + half : at + ((D - 2 * half) >> 1);
#pragma unroll 1
            for (int first = 0; first < kTurns; first += kBatch) {
                float4 a[kBatch], b[kBatch], cs[kBatch], sn[kBatch];
#pragma unroll
                for (int n = 0; n < kBatch; ++n) {
                    const int r = warp * 32 + (first + n) * kAtOnce + sub;
                    a[n] = b[n] = sn[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    cs[n] = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
                    if (sub < kAtOnce && r < rows) {
                        const int t = (first_row + r) / g.group, hq = (first_row + r) - t * g.group;
                        const float* src = g.q + (row0 + t) * g.q_stride + (int64_t)(h * g.group + hq) * D;
                        a[n] = load_now(reinterpret_cast<const float4*>(src + at));
                        b[n] = load_now(reinterpret_cast<const float4*>(src + to));
                        if (turned) {
                            int64_t pos = (int64_t)context + t;
                            if (pos < 0 || pos >= g.table_rows) {
                                if (i == 0) report(watch, kSiteKv8Range);
                                pos = 0;
                            }
                            cs[n] = load_now(reinterpret_cast<const float4*>(g.cos_table + pos * half + at));
                            sn[n] = load_now(reinterpret_cast<const float4*>(g.sin_table + pos * half + at));
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < kBatch; ++n) {
                    const int r = warp * 32 + (first + n) * kAtOnce + sub;
                    if (turned) turn(a[n], b[n], cs[n], sn[n]);
                    const float v[8] = {a[n].x, a[n].y, a[n].z, a[n].w, b[n].x, b[n].y, b[n].z, b[n].w};
                    uint32_t largest = 0;
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
                    if (sub < kAtOnce && r < warp * 32 + 32) {
                        if (i == 0) factor_s[r] = down * g.scale * kLog2e;
#pragma unroll
                        for (int part = 0; part < 2; ++part) {
                            const int d = part == 0 ? at : to;
                            const float x0 = v[4 * part] * up, x1 = v[4 * part + 1] * up, x2 = v[4 * part + 2] * up, x3 = v[4 * part + 3] * up;
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
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const int r = tid;
        const int64_t pos = (int64_t)context + (first_row + r) / g.group;
        const bool seen = r < rows && pos >= 0 && (g.rotary == 0 || pos < g.table_rows);
        const int limit = seen ? static_cast<int>(min64(keys, pos + 1)) : 0;
        const float factor = factor_s[r];
        __syncwarp();  // its place is free
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        float m = -INFINITY, l = 0.0f, m_sum = -INFINITY;
        __align__(16) float o_sum[C::kSumInSmem ? 4 : D];  // the rounded sum, relative to m_sum
        const uint32_t o_local = local_address(o_sum);
        const auto get_sum = [&](int c) { return C::kSumInSmem ? sum_s[c * C::kRows + r] : load_local(o_local + 16 * c); };
        const auto put_sum = [&](int c, float4 v) {
            if (C::kSumInSmem) sum_s[c * C::kRows + r] = v;
            else store_local(o_local + 16 * c, v);
        };
        // Adds O, complete up to the tile before, to it.
        const auto add_o = [&](bool first) {
            const float old = first || m_sum == -INFINITY ? 0.0f : ex2(m_sum - m);
            m_sum = m;
            constexpr int kBatch = 64;  // elements asked for at a time
#pragma unroll
            for (int base = 0; base < D; base += kBatch) {
                float4 z[kBatch / 4];
#pragma unroll
                for (int c = 0; c < kBatch / 4; ++c)
                    z[c] = first || base + 4 * c >= D ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : get_sum(base / 4 + c);
#pragma unroll
                for (int part = 0; part < kBatch && base + part < D; part += 32) {
                    uint32_t y[32];
                    tmem_ld_32x32b_x32(o_tmem + lanes + base + part, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float4 s4 = z[part / 4 + c];
                        put_sum((base + part) / 4 + c,
                                make_float4(fmaf(s4.x, old, __uint_as_float(y[4 * c])), fmaf(s4.y, old, __uint_as_float(y[4 * c + 1])),
                                            fmaf(s4.z, old, __uint_as_float(y[4 * c + 2])), fmaf(s4.w, old, __uint_as_float(y[4 * c + 3]))));
                    }
                }
            }
        };
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const uint32_t s_tmem = tmem + (j & 1) * C::kKeys;
            ok = __all_sync(~0u, tile_wait(watch, &s_full[j & 1], (j >> 1) & 1));
            if (!ok) break;
            tcgen05_fence_after();
            const bool anew = j % C::kSpan == 0;
            // This tile's S means that PV of tile j - 2 is done: o_done is waited for
            // one phase on at most, here and below.
            if (anew && j > 0) {
                ok = __all_sync(~0u, tile_wait(watch, o_done, (j - 1) & 1));
                if (!ok) break;
                tcgen05_fence_after();
                add_o(j == C::kSpan);
            }
            uint32_t x[C::kKeys];
#pragma unroll
            for (int c = 0; c < C::kKeys / 32; ++c)
                tmem_ld_32x32b_x32(s_tmem + lanes + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(x + 32 * c));
            const float4* scales = info + (j % C::kInfo) * C::kGroups;
            const int visible = limit - j * C::kKeys;  // columns of this tile that the row sees
            const bool whole = __all_sync(~0u, visible >= C::kKeys);
            tmem_wait_ld();
            if (!whole) {
#pragma unroll
                for (int e = 0; e < C::kKeys; ++e)
                    if (e >= visible) x[e] = 0xff800000u;
            }
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < C::kGroups; ++n) {
                const float* at = reinterpret_cast<const float*>(x) + 16 * n;
                float most = fmaxf(at[0], at[1]);
#pragma unroll
                for (int e = 2; e < 16; e += 2) most = max3(most, at[e], at[e + 1]);
                const float4 scale = scales[n];
                // A column that is not seen stays -inf whatever the scale.
                const float value = fmaf(most, scale.x * factor, scale.y);
                top = fmaxf(top, most == -INFINITY ? most : value);
            }
            if (anew) {
                // O starts anew with this tile: only L has a reference to keep.
                const float grown = fmaxf(m, top);
                l *= m == -INFINITY ? 0.0f : ex2(m - grown);
                m = grown;
            } else if (__any_sync(~0u, top > m + kSlack)) {
                ok = __all_sync(~0u, tile_wait(watch, o_done, (j - 1) & 1));
                if (!ok) break;
                tcgen05_fence_after();
                const float grown = top > m + kSlack ? top : m;
                const float old = m == -INFINITY ? 0.0f : ex2(m - grown);
                m = grown;
                l *= old;
#pragma unroll 1
                for (int c = 0; c < C::kOutCols / 32; ++c) {
                    uint32_t y[32];
                    tmem_ld_32x32b_x32(o_tmem + lanes + 32 * c, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * old);
                    tmem_st_32x32b_x32(o_tmem + lanes + 32 * c, y);
                }
            }
            const float shift = m == -INFINITY ? 0.0f : m - kTileLift;
            const auto weigh = [&](auto masked) {
#pragma unroll
                for (int c = 0; c < C::kKeys / 32; ++c) {
                    uint32_t p[32];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float4 scale = scales[2 * c + half];
                        const unsigned long long a = pack2(scale.x * factor, scale.x * factor);
                        const unsigned long long b = pack2(scale.y - shift, scale.y - shift);
                        unsigned long long sum = 0;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const int at = 32 * c + 16 * half + e;
                            const float2 y = unpack2(fma2(pack2(__uint_as_float(x[at]), __uint_as_float(x[at + 1])), a, b));
                            float w0 = ex2(y.x), w1 = ex2(y.y);
                            if constexpr (decltype(masked)::value) {  // -inf times a scale of zero is no number
                                w0 = at >= visible ? 0.0f : w0;
                                w1 = at + 1 >= visible ? 0.0f : w1;
                            }
                            const unsigned long long w = pack2(w0, w1);
                            sum = add2(sum, w);
                            const float h0 = __uint_as_float(__float_as_uint(w0) & 0xffffe000u);
                            const float h1 = __uint_as_float(__float_as_uint(w1) & 0xffffe000u);
                            const float2 low = unpack2(sub2(w, pack2(h0, h1)));
                            p[8 * half + e / 2] = half2_bits(h0, h1);
                            p[16 + 8 * half + e / 2] = half2_bits(low.x, low.y);
                        }
                        const float2 both = unpack2(sum);
                        l = fmaf(both.x + both.y, scale.z, l);
                    }
                    tmem_st_32x32b_x32(s_tmem + lanes + 32 * c, p);
                }
            };
            if (whole) weigh(std::false_type{});
            else weigh(std::true_type{});
            tmem_wait_st();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[j & 1]);
        }
        // Not o_done, which may be two phases back here.
        if (ok && tiles > 0) tile_wait(watch, drained, 0);
        __syncwarp();
        tcgen05_fence_after();
        const bool summed = tiles > C::kSpan;
        const float old = !summed || m_sum == -INFINITY ? 0.0f : ex2(m_sum - m);
        // Out through shared memory (Q's, no longer read): whole rows per store.
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* stage = smem + warp * (32 * D * 4);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            uint32_t x[32];
            if (tiles > 0) {
                tmem_ld_32x32b_x32(o_tmem + lanes + 32 * c, x);
                tmem_wait_ld();
                if (summed) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 z = get_sum(8 * c + e / 4);
                        x[e] = __float_as_uint(fmaf(z.x, old, __uint_as_float(x[e])));
                        x[e + 1] = __float_as_uint(fmaf(z.y, old, __uint_as_float(x[e + 1])));
                        x[e + 2] = __float_as_uint(fmaf(z.z, old, __uint_as_float(x[e + 2])));
                        x[e + 3] = __float_as_uint(fmaf(z.w, old, __uint_as_float(x[e + 3])));
                    }
                }
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
    } else if (warp < 7) {
        // ---------------------------------------------- codes to fp16
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
        const int ct = tid - 128;
        constexpr int kRowPieces = D / 16;
        const int32_t* table = g.step.table + (int64_t)s * g.step.max_pages;
        const int page = 1 << g.shift;
        const int64_t page_bytes = ((int64_t)g.cache.kv_heads << g.shift) * D, head_bytes = ((int64_t)h << g.shift) * D;
        // Loads are asked for where they stand: the page numbers of a tile two
        // tiles ahead, its codes and scales one.
        const auto page_of = [&](int j, int row) {  // of key row `row` of tile j; past the keys: some page
            const int key = min(j * C::kKeys + row, keys - 1);
            return load_now(table + (key >> g.shift));
        };
        // Four pieces a row and 64-element block at a time: eight lanes then store
        // to eight different bank groups.
        const auto row_of = [&](int n) {
            const int q = n * C::kConverters + ct;
            return kRowPieces % 4 == 0 ? (q >> 2) % C::kKeys : q / kRowPieces;
        };
        const auto piece_of = [&](int n) {
            const int q = n * C::kConverters + ct;
            return kRowPieces % 4 == 0 ? (q & 3) + 4 * (q / (4 * C::kKeys)) : q % kRowPieces;
        };
        const auto mine = [&](int n) { return C::kAllPieces % C::kConverters == 0 || n * C::kConverters + ct < C::kAllPieces; };
        // The pieces of tile j, whose pages are ids; zeros where there is no key.
        const auto fetch = [&](const int8_t* codes, int j, const int32_t (&ids)[C::kPieces], uint4 (&w)[C::kPieces]) {
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) {
                const int key = j * C::kKeys + row_of(n);
                const int inside = (key & (page - 1)) * D + piece_of(n) * 16;
                w[n] = make_uint4(0u, 0u, 0u, 0u);
                if (mine(n) && key < keys && static_cast<uint32_t>(ids[n]) < static_cast<uint32_t>(g.cache.pages))
                    w[n] = load_now(reinterpret_cast<const uint4*>(codes + (ids[n] * page_bytes + (head_bytes + inside))));
            }
        };
        const auto convert = [&](const uint4 (&w)[C::kPieces], uint8_t* tile) {
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) {
                if (!mine(n)) continue;
                const int row = row_of(n), cc = piece_of(n);
                const uint32_t b[4] = {w[n].x ^ 0x80808080u, w[n].y ^ 0x80808080u, w[n].z ^ 0x80808080u, w[n].w ^ 0x80808080u};
                uint8_t* line = tile + (cc >> 2) * (C::kKeys * 128) + row * 128;
                const int chunk = (cc & 3) * 2;
                *reinterpret_cast<uint4*>(line + ((chunk ^ (row & 7)) << 4)) =
                    make_uint4(codes_half2(b[0], 0x4140u), codes_half2(b[0], 0x4342u), codes_half2(b[1], 0x4140u), codes_half2(b[1], 0x4342u));
                *reinterpret_cast<uint4*>(line + (((chunk + 1) ^ (row & 7)) << 4)) =
                    make_uint4(codes_half2(b[2], 0x4140u), codes_half2(b[2], 0x4342u), codes_half2(b[3], 0x4140u), codes_half2(b[3], 0x4342u));
            }
        };
        int32_t ids[C::kPieces], later[C::kPieces], group_id = 0;  // pages of the pieces of two tiles; of 16-key group ct in the first lanes
        uint4 k[C::kPieces], v[C::kPieces];
        float ks = 0.0f, vs = -1.0f;  // the group's scales; -1: not there
        const auto ask_pages = [&](int j, int32_t (&into)[C::kPieces]) {
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) into[n] = page_of(j, min(row_of(n), C::kKeys - 1));
            if (ct < C::kGroups) group_id = page_of(j, 16 * ct);
        };
        const auto ask_scales = [&](int j) {
            ks = 0.0f;
            vs = -1.0f;
            if (ct < C::kGroups && j * C::kKeys + 16 * ct < keys) {
                if (static_cast<uint32_t>(group_id) < static_cast<uint32_t>(g.cache.pages)) {
                    const int64_t at = (int64_t)group_id * g.cache.kv_heads + h;
                    ks = load_now(g.cache.k_scales + at);
                    vs = load_now(g.cache.v_scales + at);
                } else {
                    report(watch, kSiteKv8Range);
                }
            }
        };
        const auto put_k = [&](int j) {  // k and the scales, into K of tile j
            convert(k, k_tiles + (j % C::kKStages) * C::kKvBytes);
            if (ct < C::kGroups) {
                float4 f = make_float4(0.0f, -INFINITY, 0.0f, 0.0f);  // hides the group
                // A page of zeros counts in the sum as any other.
                if (!(vs < 0.0f)) f = vs == 0.0f ? make_float4(ks, -126.0f, 0x1p126f, 0.0f) : make_float4(ks, log2f(vs), 1.0f / vs, 0.0f);
                info[(j % C::kInfo) * C::kGroups + ct] = f;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[j % C::kKStages]);
        };
        if (tiles > 0) {
            ask_pages(0, ids);
            fetch(g.cache.k_codes, 0, ids, k);
            ask_scales(0);
            fetch(g.cache.v_codes, 0, ids, v);
            ask_pages(1, ids);
            put_k(0);
            fetch(g.cache.k_codes, 1, ids, k);
            ask_scales(1);
            ask_pages(2, later);
        }
        bool ok = true;
        // K of tile j + 1 before V of tile j: its scores are computed first.
        for (int j = 0; j < tiles; ++j) {
            if (j + 1 < tiles) {
                if (j + 1 >= C::kKStages) ok = __all_sync(~0u, tile_wait(watch, &k_empty[(j + 1) % C::kKStages], ((j + 1) / C::kKStages - 1) & 1));
                if (!ok) break;
                put_k(j + 1);
                fetch(g.cache.k_codes, j + 2, later, k);
                ask_scales(j + 2);
            }
            const int stage = j % C::kVStages;
            if (j >= C::kVStages) ok = __all_sync(~0u, tile_wait(watch, &v_empty[stage], (j / C::kVStages - 1) & 1));
            if (!ok) break;
            convert(v, v_tiles + stage * C::kKvBytes);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[stage]);
            fetch(g.cache.v_codes, j + 1, ids, v);
#pragma unroll
            for (int n = 0; n < C::kPieces; ++n) ids[n] = later[n];
            ask_pages(j + 3, later);
        }
    } else {
        // ------------------------------------------------------ MMA issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
        if (tiles > 0 && lane == 0) {
            constexpr uint32_t s_desc = umma_idesc_f16(C::kRows, C::kKeys, false), o_desc = umma_idesc_f16(C::kRows, C::kOutCols, true);
            const uint32_t qh = smem_u32(q_hi), ql = smem_u32(q_lo), kt = smem_u32(k_tiles), vt = smem_u32(v_tiles);
            // S of tile j, into the buffer that PV of tile j - 2 reads: MMAs of
            // unlike accumulators keep no order, so that one is waited for.
            const auto scores = [&](int j) {
                const int stage = j % C::kKStages;
                if (!tile_wait(watch, &k_full[stage], (j / C::kKStages) & 1)) return false;
                if (j >= 2 && !tile_wait(watch, o_done, j & 1)) return false;
                tcgen05_fence_after();
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        umma_f16(tmem + (j & 1) * C::kKeys,
                                 umma_desc_k_sw128((part == 0 ? ql : qh) + (i >> 2) * (C::kRows * 128)) + 2 * (i & 3),
                                 umma_desc_k_sw128(kt + stage * C::kKvBytes + (i >> 2) * (C::kKeys * 128)) + 2 * (i & 3), s_desc,
                                 part > 0 || i > 0);
                umma_commit(&k_empty[stage]);
                umma_commit(&s_full[j & 1]);
                return true;
            };
            bool ok = tile_wait(watch, q_full, 0) && scores(0);
            for (int j = 0; j < tiles && ok; ++j) {
                if (j + 1 < tiles) ok = scores(j + 1);
                const int stage = j % C::kVStages;
                if (!ok || !tile_wait(watch, &v_full[stage], (j / C::kVStages) & 1) ||
                    !tile_wait(watch, &p_full[j & 1], (j >> 1) & 1))
                    break;
                tcgen05_fence_after();
#pragma unroll
                for (int i = 0; i < C::kKeys / 16; ++i)
#pragma unroll
                    for (int part = 0; part < 2; ++part)
                        umma_f16_ta(o_tmem, tmem + (j & 1) * C::kKeys + (i >> 1) * 32 + part * 16 + (i & 1) * 8,
                                    umma_desc_mn_sw128(vt + stage * C::kKvBytes + i * 2048, C::kKeys * 128), o_desc,
                                    j % C::kSpan > 0 || i > 0 || part > 0);
                umma_commit(&v_empty[stage]);
                umma_commit(o_done);
            }
            umma_commit(drained);  // all that was issued has completed: the output may be read, the block may end
            tile_wait(watch, drained, 0);
        }
    }
    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 7) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

template <int D>
int run_tile(cudaStream_t s, const Kv8AttendArgs& g, bool pdl) {
    DeviceWatch watch;
    int st = device_watch(&watch);
    if (st) return st;
    const int64_t row_tiles = (g.step.tokens * g.group >> 7) + g.step.requests;
    if (row_tiles * g.cache.kv_heads > INT_MAX) {
        set_error("leafq_kv8_attention: too many rows");
        return LEAFQ_ERR_INVALID;
    }
    const void* kernel = reinterpret_cast<const void*>(kv8_attend_tile_kernel<D>);
    static const int registers = [kernel] {
        cudaFuncAttributes a;
        return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers != 128) {  // setmaxnreg would wait for registers that the launch does not have
        set_error("leafq_kv8_attention: the tile kernel was built with " + std::to_string(registers) + " registers a thread, not 128");
        return LEAFQ_ERR_CUDA;
    }
    st = allow_smem(kernel, TileShape<D>::kSmem, "leafq_kv8_attention");
    if (st) return st;
    return launch(kv8_attend_tile_kernel<D>, dim3(static_cast<unsigned>(row_tiles * g.cache.kv_heads)),
                  dim3(TileShape<D>::kThreads), TileShape<D>::kSmem, s, pdl, "leafq_kv8_attention", g, watch,
                  static_cast<int>(row_tiles));
}

}  // namespace

int launch_kv8_tiles(cudaStream_t s, const Kv8AttendArgs& g, bool pdl) {
    switch (g.cache.dim) {
        case 32: return run_tile<32>(s, g, pdl);
        case 64: return run_tile<64>(s, g, pdl);
        case 96: return run_tile<96>(s, g, pdl);
        default: return run_tile<128>(s, g, pdl);
    }
}

}  // namespace leafq
