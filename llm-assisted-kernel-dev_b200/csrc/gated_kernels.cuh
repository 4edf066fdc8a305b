// Gated feed-forward block in 16-bit floating point, forward and backward, on CTA pairs (tcgen05 cta_group::2,
// kind::f16, fp32 accumulators in tensor memory).
//
//   g = x W1^T, u = x W2^T, h = act(g) * u                              x [m, k], W1, W2 [n, k], h [m, n]
//   dg = dh * u * act'(g), du = dh * act(g)
//   dx = dg W1 + du W2,  dW1 = dg^T x,  dW2 = du^T x
//
// act(z) = z * sigma(c(z)): c(z) = z for SiLU, 2 sqrt(2/pi) (z + 0.044715 z^3) for the tanh form of GELU
// (0.5 (1 + tanh t) = sigma(2t)), so both share act' = sigma + z sigma (1 - sigma) c'.
//
// One kernel template, four uses:
//   Forward     256 x 128 tiles of g and u side by side (merged B: W1 rows in the first CTA, W2 rows in the
//               second); the epilogue forms h.  ff_forward_keep also makes the 8-bit copies of g and u
//   GradHidden  the same products again; the epilogue reads dh and writes dg and du
//   GradInput   256 x 256 tiles of dx, k range = dg W1 then du W2 into the same accumulators; W as stored is
//               MN-major for this product, which the MMA descriptor takes as it is: nothing is transposed
//   GradWeight  256 x 256 tiles of dW1 and dW2 (two batches of one launch); both operands MN-major
//
// Bound by the tensor cores.  A 256 x 256 x 64 step of a pair takes 512 clocks of MMA at 4096 multiply-adds
// per clock and SM; per SM it reads 32 KB by TMA (64 B/clk; this GPU feeds ~98) and 32 KB by MMA.  m=4096 n=14336
// k=4096 takes 871,000 clocks forward, 915,000 for dg and du, 957,000 for dx and 883,000 for the weights, where the
// MMAs of 25 rounds of tiles alone take 819,000; the clock settles at 1.3 to 1.45 GHz under the power cap (1.39 to
// 1.43 PFLOP/s sustained, cuBLAS 1.31 to 1.36 on one plain product).
// Ten warps: 0-7 epilogue (quadrant w % 4, one half of the columns each), 8 MMA issuer (first CTA), 9 TMA producer.
#pragma once

#include "dense_tiles.cuh"

namespace b200 {

enum class FfMode { Forward, GradHidden, GradInput, GradWeight };

struct FfProblem {
    CUtensorMap a[2], b[2];      // operands (see the modes above)
    CUtensorMap out[2];          // h | dg, du | dx | dW1, dW2
    CUtensorMap kept[2];         // ff_forward_keep: 8-bit copies of g and u
    const uint16_t* dh;          // GradHidden
    long long ld_dh;
    float* sf[2];                // scales of the 8-bit copies, [row * sf_row + block * sf_col]
    long long sf_row, sf_col;
    int rows, cols;              // of the outputs
    int k_tiles, segments;       // 64-wide steps per segment; segments share the accumulators
    int m_tiles, n_tiles, batches;
    int gelu;
    uint32_t* status;
};

// Shapes of one pair's tile: the merged B has kN rows, half of them in each CTA.  256 is the full-rate shape.  128 (outputs of
// 256 x 64 or 256 x 128) takes 0.65 of its time instead of half (the loads bound it), and is taken where 256 leaves pairs idle.
template <int kN> struct FfShape {
    static constexpr uint32_t kABytes = 128u * 128u;             // 128 rows x 64 k (K-major) or 2 boxes of 64 x 64 (MN-major)
    static constexpr uint32_t kBBytes = kN / 2 * 128u;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = kN == 256 ? 5 : 6;
};
constexpr uint32_t kFfStagingBytes = 8u * 8192u;                 // per epilogue warp two boxes of 32 rows x 128 bytes
constexpr int kFfThreads = 320;

struct FfControl {
    uint64_t full[6], empty[6];
    uint64_t acc_full[2], acc_release[2], done;
    uint32_t tmem_base, abort_flag;
};
template <int kN> constexpr uint32_t ff_smem_bytes() {
    return 1024u + FfShape<kN>::kStages * FfShape<kN>::kStageBytes + kFfStagingBytes + sizeof(FfControl);
}
static_assert(ff_smem_bytes<256>() <= 227u * 1024u && ff_smem_bytes<128>() <= 227u * 1024u, "shared memory budget");

// act(z) and, where asked for, act'(z).  sigma saturates to 0 and 1 without a NaN for finite z.
struct GateValue { float value, slope; };
template <bool kSlope> __device__ __forceinline__ GateValue gate(float z, int gelu) {
    constexpr float kA = 1.5957691216057308f;    // 2 sqrt(2 / pi)
    constexpr float kB = 0.044715f;
    const float zz = z * z;
    const float c = gelu ? kA * z * fmaf(kB, zz, 1.0f) : z;
    const float s = __fdividef(1.0f, 1.0f + __expf(-c));
    GateValue r;
    r.value = z * s;
    if constexpr (kSlope) {
        const float dc = gelu ? kA * fmaf(3.0f * kB, zz, 1.0f) : 1.0f;
        r.slope = fmaf(r.value * (1.0f - s), dc, s);
    } else {
        r.slope = 0.0f;
    }
    return r;
}

// h = act(g) u of 32 rows x 64 columns (`acc` and `col`: this warp's half).
template <bool kBf16, int kUp>      // u lies kUp columns behind g
__device__ __forceinline__ void ff_epilogue_forward(const FfProblem& p, uint32_t acc, BoxWriter& w, int row, int col) {
    const uint32_t box = w.acquire();
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
        uint32_t g[32], u[32];
        tc_ld_x32(acc + c * 32, g);
        tc_ld_x32(acc + kUp + c * 32, u);
        tc_wait_ld();
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = gate<false>(__uint_as_float(g[i]), p.gelu).value * __uint_as_float(u[i]);
        put_chunk<kBf16>(w, box, c * 4, f);
    }
    w.send(box, &p.out[0], col, row, row < p.rows && col < p.cols);
}

// dg and du of 32 rows x 64 columns from the accumulators and dh (`acc` and `col`: this warp's half).
__device__ __forceinline__ void ff_load_dh(const FfProblem& p, int row, int col, int lane, uint4 (&d)[8]) {
    const int r = row + lane;
    const uint16_t* dh = p.dh + r * p.ld_dh + col;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        d[j] = (r < p.rows && col + 8 * j < p.cols) ? *reinterpret_cast<const uint4*>(dh + 8 * j) : make_uint4(0, 0, 0, 0);
}
template <bool kBf16, int kUp>
__device__ __forceinline__ void ff_epilogue_grad_hidden(const FfProblem& p, uint32_t acc, BoxWriter& w, int row, int col,
                                                        const uint4 (&d)[8]) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const uint32_t box = w.acquire();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t g[16], u[16];
            tc_ld_x16(acc + c * 16, g);
            if (which == 0) tc_ld_x16(acc + kUp + c * 16, u);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float e[8], f[8];
                to_float8<kBf16>(d[c * 2 + j], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = 8 * j + i;
                    if (which == 0)
                        f[i] = e[i] * __uint_as_float(u[at]) * gate<true>(__uint_as_float(g[at]), p.gelu).slope;
                    else
                        f[i] = e[i] * gate<false>(__uint_as_float(g[at]), p.gelu).value;
                }
                w.put(box, c * 2 + j, pack_16<kBf16>(f[0], f[1]), pack_16<kBf16>(f[2], f[3]), pack_16<kBf16>(f[4], f[5]),
                      pack_16<kBf16>(f[6], f[7]));
            }
        }
        w.send(box, &p.out[which], col, row, row < p.rows && col < p.cols);
    }
}

// 32 rows x 64 kParts columns of a plain product.
template <bool kBf16, int kParts>
__device__ __forceinline__ void ff_epilogue_plain(const FfProblem& p, const CUtensorMap* map, uint32_t acc, BoxWriter& w,
                                                  int row, int col) {
#pragma unroll 1
    for (int part = 0; part < kParts; ++part) {
        const uint32_t box = w.acquire();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            tc_ld_x32(acc + part * 64 + c * 32, v);
            tc_wait_ld();
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
            put_chunk<kBf16>(w, box, c * 4, f);
        }
        w.send(box, map, col + part * 64, row, row < p.rows && col + part * 64 < p.cols);
    }
}

// Producer warp: this CTA's rows of A and its half of B, step after step.
template <FfMode kMode, int kN>
__device__ __forceinline__ void ff_produce(const FfProblem& p, FfControl* ctl, uint32_t smem_base, uint32_t rank, int pair, int pairs) {
    using S = FfShape<kN>;
    constexpr bool kDual = kMode == FfMode::Forward || kMode == FfMode::GradHidden;
    constexpr bool kAMn = kMode == FfMode::GradWeight, kBMn = kAMn || kMode == FfMode::GradInput;
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    const int steps = p.k_tiles * p.segments;
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, p.batches); ok && t.valid(); t.next()) {
        const int a_row = t.m * 256 + static_cast<int>(rank) * 128;
        const int b_row = kDual ? t.n * (kN / 2) : t.n * kN + static_cast<int>(rank) * (kN / 2);
        for (int i = 0; i < steps; ++i) {
            const int seg = i >= p.k_tiles ? 1 : 0;
            const int k0 = (i - seg * p.k_tiles) * 64;
            ok = mbar_wait_converged(smem_u32(&ctl->empty[s]), ph ^ 1u, abort_flag, p.status, kStatusDense);
            if (!ok) break;
            const uint32_t a_dst = smem_base + s * S::kStageBytes, b_dst = a_dst + S::kABytes;
            const uint32_t bar = map_to_cta(smem_u32(&ctl->full[s]), 0);
            if (rank == 0) mbar_arrive_expect_tx_elect(smem_u32(&ctl->full[s]), 2 * S::kStageBytes);   // both CTAs' bytes
            const CUtensorMap* ma = &p.a[kMode == FfMode::GradWeight ? t.batch : seg];
            const CUtensorMap* mb = &p.b[kDual ? rank : (kMode == FfMode::GradInput ? seg : 0)];
            if constexpr (kAMn) {
                tma_load_2d_pair_elect(a_dst, ma, bar, a_row, k0);
                tma_load_2d_pair_elect(a_dst + 8192, ma, bar, a_row + 64, k0);
            } else {
                tma_load_2d_pair_elect(a_dst, ma, bar, k0, a_row);
            }
            if constexpr (kBMn) {
                tma_load_2d_pair_elect(b_dst, mb, bar, b_row, k0);
                if constexpr (kN == 256) tma_load_2d_pair_elect(b_dst + 8192, mb, bar, b_row + 64, k0);
            } else {
                tma_load_2d_pair_elect(b_dst, mb, bar, k0, b_row);
            }
            if (++s == S::kStages) { s = 0; ph ^= 1u; }
        }
    }
    if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(2000);   // error path: let copies in flight land
    __syncwarp();
}

// MMA warp (the pair's first CTA issues): `chunk` steps go into one accumulator, then the other one is used.
template <FfMode kMode, bool kBf16, int kN>
__device__ __forceinline__ void ff_issue(const FfProblem& p, FfControl* ctl, uint32_t smem_base, uint32_t tmem_base, uint32_t rank,
                                         int pair, int pairs, int chunk) {
    using S = FfShape<kN>;
    constexpr bool kAMn = kMode == FfMode::GradWeight, kBMn = kAMn || kMode == FfMode::GradInput;
    constexpr uint32_t kIdesc = idesc_dense(256, kN, kBf16 ? 1u : 0u, kAMn, kBMn);
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    if (rank == 0) {
        const int steps = p.k_tiles * p.segments;
        uint32_t s = 0, ph = 0;
        int it = 0;
        bool ok = true;
        for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, p.batches); ok && t.valid(); t.next()) {
            for (int i0 = 0; ok && i0 < steps; i0 += chunk, ++it) {
                if (it >= 2)
                    ok = mbar_wait_converged(smem_u32(&ctl->acc_release[it & 1]), ((it >> 1) - 1) & 1, abort_flag, p.status, kStatusDense);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t acc = tmem_base + (it & 1) * 256;
                const int count = steps - i0 < chunk ? steps - i0 : chunk;
#pragma unroll 1
                for (int i = 0; i < count; ++i) {
                    ok = mbar_wait_converged(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, kStatusDense);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t a = dense_desc_lo<kAMn>(smem_base + s * S::kStageBytes);
                    const uint32_t b = dense_desc_lo<kBMn>(smem_base + s * S::kStageBytes + S::kABytes);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        tc_mma_f16_pair(acc, a + j * kDescStepK16<kAMn>, b + j * kDescStepK16<kBMn>, kIdesc, (i > 0 || j > 0) ? 1u : 0u);
                    tc_commit_pair_both_elect(smem_u32(&ctl->empty[s]), 3);
                    if (++s == S::kStages) { s = 0; ph ^= 1u; }
                }
                if (ok) tc_commit_pair_both_elect(smem_u32(&ctl->acc_full[it & 1]), 3);
            }
        }
        tc_commit_pair_elect(smem_u32(&ctl->done));
        mbar_wait<true>(smem_u32(&ctl->done), 0, abort_flag, p.status, kStatusDense);
    }
    __syncwarp();
}

// Barriers and tensor memory of a pair's CTA; returns the tensor memory's base.  `alloc_warp` allocates.
template <int kStages>
__device__ __forceinline__ uint32_t ff_setup(FfControl* ctl, int warp, int alloc_warp) {
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&ctl->acc_full[b]), 1);
            mbar_init(smem_u32(&ctl->acc_release[b]), 16);   // eight epilogue warps of each CTA; used in the first
        }
        mbar_init(smem_u32(&ctl->done), 1);
        ctl->abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == alloc_warp) {
        tmem_alloc_pair(smem_u32(&ctl->tmem_base), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    cluster_arrive();
    cluster_wait();            // both CTAs' barriers exist
    griddep_launch_dependents();   // after this CTA has its tensor memory: a CTA of the next kernel cannot take it away
    griddep_wait();
    return ctl->tmem_base;
}
// Nobody leaves while the partner may still signal its barriers or while MMAs run on this SM.
__device__ __forceinline__ void ff_leave(uint32_t tmem_base, int warp, int alloc_warp) {
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp == alloc_warp) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <FfMode kMode, bool kBf16, int kN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFfThreads, 1)
ff_gemm_pair(const __grid_constant__ FfProblem p) {
    using S = FfShape<kN>;
    constexpr int kStages = S::kStages;
    constexpr bool kDual = kMode == FfMode::Forward || kMode == FfMode::GradHidden;
    constexpr int kTileCols = kDual ? kN / 2 : kN;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t staging = smem_base + kStages * S::kStageBytes;
    FfControl* ctl = reinterpret_cast<FfControl*>(smem_raw + (staging - smem_u32(smem_raw)) + kFfStagingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    const uint32_t tmem_base = ff_setup<S::kStages>(ctl, warp, 8);
    if (warp == 9) ff_produce<kMode, kN>(p, ctl, smem_base, rank, pair, pairs);
    else if (warp == 8) ff_issue<kMode, kBf16, kN>(p, ctl, smem_base, tmem_base, rank, pair, pairs, p.k_tiles * p.segments);
    else {
        // ------------------------------ epilogue
        // a box is 64 columns: the 64 of a narrow dual tile are one warp's work per quadrant
        constexpr int kWarpCols = kTileCols / 2 < 64 ? 64 : kTileCols / 2;
        const int quad = warp & 3, half = warp >> 2;
        const bool works = half * kWarpCols < kTileCols;
        BoxWriter w{staging + static_cast<uint32_t>(warp) * 8192u, lane, 0};
        const uint32_t release = map_to_cta(smem_u32(&ctl->acc_release[0]), 0);
        int it = 0;
        for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, p.batches); t.valid(); t.next(), ++it) {
            const int row = t.m * 256 + static_cast<int>(rank) * 128 + quad * 32;
            const int col = t.n * kTileCols + half * kWarpCols;
            uint4 d[8];
            if constexpr (kMode == FfMode::GradHidden)
                if (works) ff_load_dh(p, row, col, lane, d);          // arrives while the products are formed
            if (!mbar_wait_converged(smem_u32(&ctl->acc_full[it & 1]), (it >> 1) & 1, abort_flag, p.status, kStatusDense)) break;
            tc_fence_after_sync();
            const uint32_t acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + (it & 1) * 256;
            if (works) {
                if constexpr (kMode == FfMode::Forward) {
                    ff_epilogue_forward<kBf16, kTileCols>(p, acc + half * kWarpCols, w, row, col);
                } else if constexpr (kMode == FfMode::GradHidden) {
                    ff_epilogue_grad_hidden<kBf16, kTileCols>(p, acc + half * kWarpCols, w, row, col, d);
                } else {
                    ff_epilogue_plain<kBf16, kWarpCols / 64>(p, &p.out[t.batch], acc + half * kWarpCols, w, row, col);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            mbar_arrive_cluster_relaxed_elect(release + 8 * (it & 1));
        }
        if (lane == 0) bulk_wait_group_read_all();
        __syncwarp();
    }
    ff_leave(tmem_base, warp, 8);
}

// The forward pass that also makes the 8-bit copies of g and u.  Tensor memory adds with truncation, one MMA after the other:
// summed there over k = 7168, one code in 3400 was a neighbour of the right one, 6 to 12 % away, and the weights' gradients were
// 1.53 times as far off as their own rounding makes them.  So the accumulators are emptied every kKeepChunk steps into fp32
// registers (the two accumulators take turns, the MMAs do not wait): one code in 64000, and the same time; with 4 steps one in 93000
// and 3 % more (m=2048 n=4096 k=7168: 162 us, 158 without the copies; fp32 products on the ordinary pipe: one in 35000).
// Each of the eight epilogue warps sums 32 rows x 64 columns of g and of u; the two warps of a quadrant agree on a row's largest
// magnitudes through shared memory.  Registers: 384 threads start with 168; the two epilogue warpgroups take 216, the third
// keeps 72 (256 * 216 + 128 * 72 = 384 * 168).
constexpr int kKeepThreads = 384, kKeepChunk = 8;
constexpr uint32_t kKeepSumRegs = 216, kKeepOtherRegs = 72;
static_assert(256 * kKeepSumRegs + 128 * kKeepOtherRegs <= kKeepThreads * 168, "register split");

// Barrier of the two warps of a quadrant; the second form also tells both whether both are well, so that neither waits for a
// partner that has given up.
__device__ __forceinline__ void quad_bar_sync(int quad) { asm volatile("bar.sync %0, 64;" ::"r"(quad + 1) : "memory"); }
__device__ __forceinline__ bool quad_bar_and(int quad, bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "bar.red.and.pred q, %1, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}\n"
        : "=r"(all)
        : "r"(quad + 1), "r"(static_cast<uint32_t>(ok))
        : "memory");
    return all != 0;
}

template <bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kKeepThreads, 1)
ff_forward_keep(const __grid_constant__ FfProblem p) {
    using S = FfShape<256>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t staging = smem_base + S::kStages * S::kStageBytes;
    FfControl* ctl = reinterpret_cast<FfControl*>(smem_raw + (staging - smem_u32(smem_raw)) + kFfStagingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    const uint32_t tmem_base = ff_setup<S::kStages>(ctl, warp, 8);
    if (warp >= 8) {
        warpgroup_reg_dec<kKeepOtherRegs>();
        if (warp == 9) ff_produce<FfMode::Forward, 256>(p, ctl, smem_base, rank, pair, pairs);
        else if (warp == 8) ff_issue<FfMode::Forward, kBf16, 256>(p, ctl, smem_base, tmem_base, rank, pair, pairs, kKeepChunk);
    } else {
        warpgroup_reg_inc<kKeepSumRegs>();
        const int quad = warp & 3, half = warp >> 2;
        // one box per warp for h; one for the codes of g and one for those of u per quadrant
        const uint32_t box_h = staging + static_cast<uint32_t>(warp) * 4096u;
        const uint32_t box_q = staging + 8u * 4096u + static_cast<uint32_t>(quad) * 8192u;
        const uint32_t release = map_to_cta(smem_u32(&ctl->acc_release[0]), 0);
        const uint32_t own = static_cast<uint32_t>(lane) * 128u, swz = static_cast<uint32_t>(lane & 7);
        const int chunks = (p.k_tiles + kKeepChunk - 1) / kKeepChunk;
        int it = 0;
        bool ok = true;
        for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, 1); ok && t.valid(); t.next()) {
            uint64_t g[32], u[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = u[i] = 0;
#pragma unroll 1
            for (int c = 0; c < chunks; ++c, ++it) {
                ok = mbar_wait_converged(smem_u32(&ctl->acc_full[it & 1]), (it >> 1) & 1, abort_flag, p.status, kStatusDense);
                if (!ok) break;
                tc_fence_after_sync();
                const uint32_t acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + (it & 1) * 256 + half * 64;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t v[16];
                    tc_ld_x16(acc + j * 16, v);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[j * 8 + i] = add_f32x2(g[j * 8 + i], pack_f32x2(v[2 * i], v[2 * i + 1]));
                    tc_ld_x16(acc + 128 + j * 16, v);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) u[j * 8 + i] = add_f32x2(u[j * 8 + i], pack_f32x2(v[2 * i], v[2 * i + 1]));
                }
                tc_fence_before_sync();
                mbar_arrive_cluster_relaxed_elect(release + 8 * (it & 1));
            }
            const int row = t.m * 256 + static_cast<int>(rank) * 128 + quad * 32, col = t.n * 128;
            // boxes and scratch are free once the previous tile's copies have been read
            if (lane == 0) bulk_wait_group_read_all();
            __syncwarp();
            ok = quad_bar_and(quad, ok);
            if (!ok) break;
            float mg = kAmaxFloor, mu = kAmaxFloor;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 a = unpack_f32x2(g[j * 4 + i]), b = unpack_f32x2(u[j * 4 + i]);
                    mg = fmaxf(mg, fmaxf(fabsf(a.x), fabsf(a.y)));
                    mu = fmaxf(mu, fmaxf(fabsf(b.x), fabsf(b.y)));
                    w[i] = pack_16<kBf16>(gate<false>(a.x, p.gelu).value * b.x, gate<false>(a.y, p.gelu).value * b.y);
                }
                st_shared_v4(box_h + own + ((static_cast<uint32_t>(j) ^ swz) << 4), w[0], w[1], w[2], w[3]);
            }
            // largest magnitudes of the whole 128-wide block: the partner warp has the other half
            const uint32_t scratch = box_q + static_cast<uint32_t>(lane) * 16u;
            st_shared_f32(scratch + half * 8, mg);
            st_shared_f32(scratch + half * 8 + 4, mu);
            quad_bar_sync(quad);
            uint32_t om, ou;
            ld_shared_v2(scratch + (half ^ 1) * 8, om, ou);
            mg = fmaxf(mg, __uint_as_float(om));
            mu = fmaxf(mu, __uint_as_float(ou));
            quad_bar_sync(quad);                     // read before the codes take its place
            const PowerScale sg(mg), su(mu);
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                const PowerScale& sc = which ? su : sg;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t q[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 a = unpack_f32x2((which ? u : g)[j * 8 + 2 * i]), b = unpack_f32x2((which ? u : g)[j * 8 + 2 * i + 1]);
                        q[i] = pack_e4m3x4(sc(a.x), sc(a.y), sc(b.x), sc(b.y));
                    }
                    st_shared_v4(box_q + which * 4096u + own + ((static_cast<uint32_t>(half * 4 + j) ^ swz) << 4), q[0], q[1], q[2], q[3]);
                }
            }
            if (half == 0 && row + lane < p.rows && col < p.cols) {
                const long long at = (row + lane) * p.sf_row + (col / kFp8Block) * p.sf_col;
                p.sf[0][at] = sg.scale;
                p.sf[1][at] = su.scale;
            }
            fence_proxy_async_smem();
            quad_bar_sync(quad);
            if (lane == 0) {
                const bool inside = row < p.rows;
                if (inside && col + half * 64 < p.cols) tma_store_2d(&p.out[0], box_h, col + half * 64, row);
                if (inside && col < p.cols) tma_store_2d(&p.kept[half], box_q + half * 4096u, col, row);
                bulk_commit_group();
            }
        }
        if (lane == 0) bulk_wait_group_read_all();
        __syncwarp();
    }
    ff_leave(tmem_base, warp, 8);
}

// dg and du from the 8-bit copies of g and u: a streaming pass, 2 bytes of codes, 2 of dh and 4 of results per
// element.  A thread takes 16 columns of kKeptRows rows, all loaded before the first is used.  Bound by memory: m=2048 n=4096
// (67 MB) 17 us, m=8192 n=14336 (940 MB) 187 us = 5.0 TB/s (250 with one block for each two rows).
__device__ __forceinline__ uint4 load_codes16(const uint8_t* p, bool all) {
    if (all) return *reinterpret_cast<const uint4*>(p);
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_uint4(v.x, v.y, 0, 0);
}
constexpr int kKeptRows = 2, kKeptThreads = 128;
constexpr unsigned kKeptBlocksPerSm = 14;     // resident twice over: the blocks walk down the rows
constexpr int kKeptCols = kKeptThreads * 16;
template <bool kBf16>
__global__ void __launch_bounds__(kKeptThreads)
gated_grad_kept(const uint8_t* __restrict__ qg, const uint8_t* __restrict__ qu, long long ldq, const float* __restrict__ sg,
                const float* __restrict__ su, long long sf_row, long long sf_col, const uint16_t* __restrict__ dh,
                long long ld_dh, uint16_t* __restrict__ dg, uint16_t* __restrict__ du, long long ld_out, int rows, int n,
                int gelu) {
    griddep_launch_dependents();
    griddep_wait();
    const int col = blockIdx.x * kKeptCols + threadIdx.x * 16;
    if (col >= n) return;
    const bool upper = col + 8 < n;              // n is a multiple of 8: the thread's second half may be missing
    for (long long r0 = static_cast<long long>(blockIdx.y) * kKeptRows; r0 < rows; r0 += static_cast<long long>(gridDim.y) * kKeptRows) {
        uint4 a[kKeptRows], b[kKeptRows], d[kKeptRows][2];
        float s1[kKeptRows], s2[kKeptRows];
#pragma unroll
        for (int i = 0; i < kKeptRows; ++i) {
            const long long r = r0 + i;
            if (r >= rows) break;
            a[i] = load_codes16(qg + r * ldq + col, upper);
            b[i] = load_codes16(qu + r * ldq + col, upper);
            const uint4* dr = reinterpret_cast<const uint4*>(dh + r * ld_dh + col);
            d[i][0] = dr[0];
            d[i][1] = upper ? dr[1] : make_uint4(0, 0, 0, 0);
            s1[i] = sg[r * sf_row + (col / kFp8Block) * sf_col];
            s2[i] = su[r * sf_row + (col / kFp8Block) * sf_col];
        }
#pragma unroll
        for (int i = 0; i < kKeptRows; ++i) {
            const long long r = r0 + i;
            if (r >= rows) break;
            const uint32_t wa[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, wb[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                if (part == 1 && !upper) break;
                float e[8];
                to_float8<kBf16>(d[i][part], e);
                uint32_t og[4], ou[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 g = unpack_e4m3x2(wa[part * 2 + j / 2] >> (16 * (j & 1)));
                    const float2 v = unpack_e4m3x2(wb[part * 2 + j / 2] >> (16 * (j & 1)));
                    const GateValue g0 = gate<true>(g.x * s1[i], gelu), g1 = gate<true>(g.y * s1[i], gelu);
                    og[j] = pack_16<kBf16>(e[2 * j] * (v.x * s2[i]) * g0.slope, e[2 * j + 1] * (v.y * s2[i]) * g1.slope);
                    ou[j] = pack_16<kBf16>(e[2 * j] * g0.value, e[2 * j + 1] * g1.value);
                }
                *reinterpret_cast<uint4*>(dg + r * ld_out + col + part * 8) = make_uint4(og[0], og[1], og[2], og[3]);
                *reinterpret_cast<uint4*>(du + r * ld_out + col + part * 8) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
            }
        }
    }
}

}  // namespace b200
