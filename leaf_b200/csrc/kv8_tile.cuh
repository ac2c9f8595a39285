// Shared by the two kernels that give 128 query rows to the tensor cores (kv8_tile.cu for
// prompts, kv8_tree_tile.cu for trees of drafts).  Both are compiled as whole programs.
#pragma once

#define LEAFQ_WHOLE_PROGRAM
#include <cfloat>

#include "kv8_attention.cuh"

namespace leafq {
namespace {

// Weights and the pages that need no test: kv8_tile.cu says how these are used.
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

}  // namespace
}  // namespace leafq
