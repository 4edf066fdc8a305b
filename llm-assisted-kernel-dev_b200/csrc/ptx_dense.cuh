// Inline-PTX wrappers of the 16-bit and 8-bit floating-point GEMMs: two-dimensional TMA copies,
// tcgen05.mma kind::f16 / kind::f8f6f4 on one CTA or a CTA pair, their descriptors, e4m3 conversion.
#pragma once

#include <cuda_bf16.h>

#include "ptx_sm100.cuh"

namespace b200 {

// ---------------------------------------------------------------------------
// TMA, two dimensions.  c0 is the innermost coordinate in elements; every caller keeps
// c0 * element size a multiple of 16 bytes.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d_elect(uint32_t smem_dst, const void* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n\t"
        "}\n" ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
// Load into this CTA's shared memory whose bytes are counted on a barrier of either CTA of the
// pair (`cluster_bar` from map_to_cta): the MMA issuer then waits on one barrier for both CTAs' operands.
__device__ __forceinline__ void tma_load_2d_pair_elect(uint32_t smem_dst, const void* map, uint32_t cluster_bar, int c0,
                                                       int c1) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];\n\t"
        "}\n" ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_bar), "r"(c0), "r"(c1)
        : "memory");
}
// Whole box shared memory -> global, clipped at the map's extents; joins the thread's bulk group.
__device__ __forceinline__ void tma_store_2d(const void* map, uint32_t smem_src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_src), "r"(c0), "r"(c1)
                 : "memory");
}

// ---------------------------------------------------------------------------
// Descriptors
// ---------------------------------------------------------------------------
// Both operand layouts use the 128-byte swizzle.  The low word of a shared-memory descriptor holds the
// start address and the leading byte offset, the high word the stride byte offset, version and layout.
//   K-major   128-byte rows along k; 8-row groups 1024 bytes apart (leading offset unused)
//   MN-major  boxes of 64 elements along m (or n) x 64 rows of k, 8 KiB each: 8-row groups of k are 1024
//             bytes apart (stride), the next 64 elements along m are 8192 bytes away (leading)
constexpr uint32_t kLboMnMajor = (8192u >> 4) << 16;
template <bool kMnMajor> __device__ __forceinline__ uint32_t dense_desc_lo(uint32_t smem_addr) {
    return ((smem_addr & 0x3FFFFu) >> 4) | (kMnMajor ? kLboMnMajor : (1u << 16));
}
// What 16 elements of k (32 bytes of a K-major row, 16 rows of an MN-major box) advance the start address by.
template <bool kMnMajor> constexpr uint32_t kDescStepK16 = kMnMajor ? (2048u >> 4) : (32u >> 4);

// Instruction descriptors, fp32 accumulation:
//   [4,6) D format (1 = f32)   [7,10) A format   [10,13) B format   [15] A is MN-major   [16] B is MN-major
//   [17,23) N >> 3   [24,29) M >> 4
// kind::f16: 0 = fp16, 1 = bf16.  kind::f8f6f4: 0 = e4m3.
__host__ __device__ constexpr uint32_t idesc_dense(int m, int n, uint32_t format, bool a_mn, bool b_mn) {
    return (1u << 4) | (format << 7) | (format << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// ---------------------------------------------------------------------------
// MMA: one elected lane of a converged warp issues; operands by descriptor low words.
// ---------------------------------------------------------------------------
#define B200_DENSE_MMA(name, group, kind)                                                                              \
    __device__ __forceinline__ void name(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,                \
                                         uint32_t accumulate) {                                                        \
        asm volatile(                                                                                                  \
            "{\n\t"                                                                                                    \
            ".reg .pred p, e;\n\t"                                                                                     \
            ".reg .b64 da, db;\n\t"                                                                                    \
            "mov.b64 da, {%1, %5};\n\t"                                                                                \
            "mov.b64 db, {%2, %5};\n\t"                                                                                \
            "setp.ne.b32 p, %4, 0;\n\t"                                                                                \
            "elect.sync _|e, 0xffffffff;\n\t"                                                                          \
            "@e tcgen05.mma.cta_group::" group ".kind::" kind " [%0], da, db, %3, p;\n\t"                              \
            "}\n" ::"r"(tmem_d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128)                  \
            : "memory");                                                                                               \
    }
B200_DENSE_MMA(tc_mma_f16_pair, "2", "f16")
B200_DENSE_MMA(tc_mma_f8_pair, "2", "f8f6f4")
B200_DENSE_MMA(tc_mma_f16_one, "1", "f16")
B200_DENSE_MMA(tc_mma_f8_one, "1", "f8f6f4")
#undef B200_DENSE_MMA

__device__ __forceinline__ void tc_commit_elect(uint32_t bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "}\n" ::"r"(bar)
        : "memory");
}

// Arrive (no release ordering, see mbar_arrive_cluster_relaxed) by one elected lane of a converged warp.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed_elect(uint32_t cluster_addr) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t"
        "}\n" ::"r"(cluster_addr)
        : "memory");
}

// Arrive on a barrier of this CTA (release) by one elected lane of a converged warp.
__device__ __forceinline__ void mbar_arrive_elect(uint32_t bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
        "}\n" ::"r"(bar)
        : "memory");
}

// Bounded wait of a converged warp in lock step: every lane tries, one vote decides, so a barrier that is already
// complete costs no divergent branch (about 40 clocks against 350 when one lane polls inside an `if`).
__device__ __forceinline__ bool mbar_wait_converged_slow(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                      uint32_t* status, uint32_t code) {
    const long long t0 = clock64();
#pragma unroll 1
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (__all_sync(0xffffffffu, mbar_try_wait_parked(bar, parity, 20000u))) return true;
        if (__any_sync(0xffffffffu, *abort_flag != 0u || clock64() - t0 > kWaitTimeoutCycles)) {
            if (*abort_flag == 0u) atomicOr(status, code);
            *abort_flag = 1u;
            return false;
        }
    }
}
__device__ __forceinline__ bool mbar_wait_converged(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag,
                                                    uint32_t* status, uint32_t code) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return mbar_wait_converged_slow(bar, parity, abort_flag, status, code);
}

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// TMEM -> registers, 32 consecutive columns of the warp's own lane quadrant.
__device__ __forceinline__ void tc_ld_x32(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
        "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

// ---------------------------------------------------------------------------
// 16-bit and 8-bit conversions
// ---------------------------------------------------------------------------
template <bool kBf16> __device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
    if constexpr (kBf16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        return pack_half2(lo, hi);
    }
}
template <bool kBf16> __device__ __forceinline__ float2 unpack_16(uint32_t v) {
    if constexpr (kBf16) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    } else {
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    }
}
// Two e4m3 codes, `lo` in the low byte; round to nearest even, beyond 448 -> 448, NaN -> NaN.
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16);
}
__device__ __forceinline__ float2 unpack_e4m3x2(uint32_t v) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(v)));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Packed fp32 pair: acc = x * s + acc.
__device__ __forceinline__ void fma_f32x2(uint64_t& acc, uint64_t x, uint64_t s) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(s));
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t pack_f32x2(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

}  // namespace b200
