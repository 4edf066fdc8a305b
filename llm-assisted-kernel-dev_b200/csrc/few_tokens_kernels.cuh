// The fp8 linear layer and the gated block's forward pass for few tokens (a decoding step, a short prompt).
//
// With m of a few dozen rows these products read each weight once and do little with it: the floor is the weight's
// bytes at memory bandwidth, and 256-row tiles would leave most SMs idle (n / 256 tiles).  So the operands change
// places - C^T = W A^T: 128 rows of W are the MMA's M, 16 to 128 tokens its N - and the k range of a tile is cut
// over a cluster of up to eight CTAs, so that every SM streams weights.  The partial sums meet through distributed
// shared memory, added in rank order: no workspace, no atomics, the same bits on every run.
//
//   Few8      fp8: fp32 sums of one 128-wide block in tensor memory, scaled and added up in registers (one weight
//             row per lane, one column per token), as in fp8_gemm_pair
//             With kFuse the tokens come as 16-bit rows and four more warps quantise them on their way into shared
//             memory (up to 16 tokens: every tile of W repeats that work, and a launch of its own costs more)
//   FewGated  16-bit: g and u of the same rows and tokens side by side in tensor memory, h formed after the exchange
//
// Bound by memory for few tokens: gated m=1 n=14336 k=4096 38.6 us (6.1 TB/s).  A small weight pays a fixed 4 us: 1 us of
// set-up, 2 us until the first block is there, 1 us for the exchange (fp8 m=1 n=4096 k=7168: 8.4 us, 4.5 of them the weight's
// bytes).  With 128 tokens the adding up counts (fp8 m=256 n=4096 k=7168 16.0 us; it was 19.4 with scales copied per
// block and multiplied by every lane).
// Warps: four or eight for sums and results, then MMA issuer, weight loads, token loads, and one for scale products (Few8) or four
// that quantise (kFuse).
#pragma once

#include "dense_tiles.cuh"
#include "gated_kernels.cuh"

namespace b200 {

enum class FewOp { Few8, FewGated };

struct FewProblem {
    CUtensorMap w[2], x;
    const uint16_t* x16;         // kFuse: the tokens
    long long ldx;
    int k, vec;                  // vec: rows of x start on 16-byte boundaries
    const float* sfa;            // Few8: token scales, [token * sfa_row + block * sfa_col]
    const float* sfb;            // Few8: weight scales, [(row / 128) * sfb_row + block * sfb_col]
    long long sfa_row, sfa_col, sfb_row, sfb_col;
    uint16_t* c;
    long long ldc;
    int m, n, steps;             // steps: 128-byte pieces of k (128 e4m3, 64 16-bit)
    int gelu;
    int weights_early;           // the kernel before this one on the stream is known not to write the weights and to have waited
                                 // for all before it: weight loads need not wait for it
    uint32_t* status;
};

constexpr int kFewBatch = 8;             // blocks whose scales are handed over at a time

template <FewOp kOp, int kTokens, bool kFuse> struct FewShape {
    static constexpr bool kFp8 = kOp == FewOp::Few8;
    static constexpr uint32_t kWeightBytes = (kFp8 ? 1u : 2u) * 16384u;     // 128 rows x 128 bytes of each weight
    static constexpr uint32_t kTokenBytes = kTokens * 128u;
    static constexpr uint32_t kStageBytes = kWeightBytes + kTokenBytes;
    // warps that add up the blocks' sums: two for each quadrant of tensor memory with 128 tokens, half of them each
    static constexpr int kSumWarps = kFp8 && kTokens == 128 ? 8 : 4;
    static constexpr int kThreads = 32 * (kSumWarps + (kFuse ? 7 : kFp8 ? 4 : 3));
    // two CTAs on an SM up to 64 (fp8) or 32 tokens, one beyond: registers and stages
    static constexpr int kCtasPerSm = kTokens <= (kFp8 ? 64 : 32) ? 2 : 1;
    static constexpr int kStages = static_cast<int>((kCtasPerSm == 2 ? 108u * 1024u : 200u * 1024u) / kStageBytes);
    static constexpr int kBuffers = kFp8 ? 4 : 1;                           // accumulators that take turns
    static constexpr uint32_t kTmemCols = (kFp8 ? kBuffers : 2) * kTokens;  // these, or g and u
    static constexpr int kArrivals = kFuse ? 5 : 2;        // on a stage's barrier: weight loads; token loads or the quantising warps
    // scales: a slot for each stage (kFuse), or two batches of kFewBatch blocks
    static constexpr int kScaleRows = kFuse ? kStages : 2 * kFewBatch;
    // partial sums for the exchange take the place of the stages
    static_assert((kFp8 ? 1u : 2u) * kTokens * 512u <= kStages * kStageBytes, "exchange area");
    static_assert(kStageBytes % 1024 == 0, "stages keep the alignment of the swizzle");
};
template <FewOp kOp, int kTokens, bool kFuse> struct FewControl {
    using S = FewShape<kOp, kTokens, kFuse>;
    uint64_t full[S::kStages], empty[S::kStages];
    uint64_t scale_full[2], scale_free[S::kStages];      // batches; a slot of kFuse is full with its stage
    uint64_t acc_full[S::kBuffers], acc_release[S::kBuffers];
    uint32_t tmem_base, abort_flag;
    alignas(16) float scale[S::kScaleRows][kTokens];     // s_A, or s_A s_B
};
template <FewOp kOp, int kTokens, bool kFuse> constexpr uint32_t few_smem_bytes() {
    using S = FewShape<kOp, kTokens, kFuse>;
    return 1024u + S::kStages * S::kStageBytes + sizeof(FewControl<kOp, kTokens, kFuse>);
}

__device__ __forceinline__ float4 ld_cluster_v4f(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void add_v4f(float4& a, const float4& b) {
    a.x += b.x;
    a.y += b.y;
    a.z += b.z;
    a.w += b.w;
}
template <bool kBf16> __device__ __forceinline__ uint16_t to_16(float v) { return static_cast<uint16_t>(pack_16<kBf16>(v, 0.0f)); }

template <int kN> __device__ __forceinline__ void tc_ld_cols(uint32_t taddr, uint32_t (&v)[kN]) {
    static_assert(kN == 16 || kN == 32, "columns per load");
    if constexpr (kN == 16) tc_ld_x16(taddr, v);
    else tc_ld_x32(taddr, v);
}

// Results of the tokens that fall to this warp, from the sums of all ranks.  kGroup tokens of kMost loads each (two of them for
// the gated block) are in flight before the first is added: one remote load takes about 0.5 us.
template <FewOp kOp, int kTokens, bool kBf16, int kMost, int kGroup>
__device__ __forceinline__ void few_sum_ranks(const FewProblem& p, uint32_t area, int w_row, int token0, int tokens, uint32_t rank,
                                              uint32_t splits, int warp, int warps, int lane) {
    constexpr bool kFp8 = kOp == FewOp::Few8;
    const int col = w_row + lane * 4;        // four neighbouring columns of C; n is a multiple of four
    if (col >= p.n) return;
    const int step = static_cast<int>(splits) * warps;
#pragma unroll 1
    for (int t0 = static_cast<int>(rank + splits * warp); t0 < tokens; t0 += step * kGroup) {
        float4 g[kGroup][kMost], u[kGroup][kFp8 ? 1 : kMost];
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            const uint32_t mine = area + (t0 + j * step) * 512 + lane * 16;
#pragma unroll
            for (uint32_t r = 0; r < kMost; ++r)
                if (t0 + j * step < tokens && r < splits) {
                    g[j][r] = ld_cluster_v4f(map_to_cta(mine, r));
                    if constexpr (!kFp8) u[j][r] = ld_cluster_v4f(map_to_cta(mine + kTokens * 512, r));
                }
        }
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            if (t0 + j * step >= tokens) break;
            float4 y = g[j][0];
#pragma unroll
            for (uint32_t r = 1; r < kMost; ++r)
                if (r < splits) add_v4f(y, g[j][r]);
            if constexpr (!kFp8) {
                float4 z = u[j][0];
#pragma unroll
                for (uint32_t r = 1; r < kMost; ++r)
                    if (r < splits) add_v4f(z, u[j][r]);
                y.x = gate<false>(y.x, p.gelu).value * z.x;
                y.y = gate<false>(y.y, p.gelu).value * z.y;
                y.z = gate<false>(y.z, p.gelu).value * z.z;
                y.w = gate<false>(y.w, p.gelu).value * z.w;
            }
            uint16_t* dst = p.c + (token0 + t0 + j * step) * p.ldc + col;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_16<kBf16>(y.x, y.y), pack_16<kBf16>(y.z, y.w));
        }
    }
}

template <FewOp kOp, int kTokens, bool kBf16, bool kFuse = false>
__global__ void __launch_bounds__(FewShape<kOp, kTokens, kFuse>::kThreads, FewShape<kOp, kTokens, kFuse>::kCtasPerSm)
few_tokens_gemm(const __grid_constant__ FewProblem p) {
    using S = FewShape<kOp, kTokens, kFuse>;
    constexpr bool kFp8 = S::kFp8;
    constexpr int kStages = S::kStages;
    constexpr int kSumWarps = S::kSumWarps, kMma = kSumWarps, kLoadW = kSumWarps + 1, kLoadX = kSumWarps + 2, kScale = kSumWarps + 3;
    constexpr int kMine = kTokens * 4 / kSumWarps;        // tokens of one summing warp
    constexpr int kChunk = kMine < 32 ? kMine : 32;
    constexpr int kFuseAhead = 4;                         // blocks of k whose tokens a quantising half-warp loads at a time
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    auto* ctl = reinterpret_cast<FewControl<kOp, kTokens, kFuse>*>(smem_raw + (smem_base - smem_u32(smem_raw)) + kStages * S::kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t splits;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
    const uint32_t rank = cluster_cta_rank();
    const int w_row = static_cast<int>(blockIdx.x / splits) * 128;
    const int token0 = blockIdx.y * kTokens;
    const int begin = static_cast<int>(static_cast<long long>(p.steps) * rank / splits);
    const int count = static_cast<int>(static_cast<long long>(p.steps) * (rank + 1) / splits) - begin;
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), S::kArrivals);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
            mbar_init(smem_u32(&ctl->scale_free[s]), kSumWarps);
        }
        for (int b = 0; b < 2; ++b) mbar_init(smem_u32(&ctl->scale_full[b]), 32);    // every lane of the scale warp
        for (int b = 0; b < S::kBuffers; ++b) {
            mbar_init(smem_u32(&ctl->acc_full[b]), 1);
            mbar_init(smem_u32(&ctl->acc_release[b]), kSumWarps);
        }
        ctl->abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == kMma) {
        tmem_alloc(smem_u32(&ctl->tmem_base), S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = ctl->tmem_base;
    griddep_launch_dependents();   // after this CTA has its tensor memory: a CTA of the next kernel cannot take it away
    if (!(warp == kLoadW && p.weights_early)) griddep_wait();

    float sum[kFp8 ? kMine : 1];        // Few8: this lane's weight row, this warp's tokens
    bool ok = true;
    if (kFuse && warp >= kLoadX) {
        // ------------------------------ tokens: quantised here (a half-warp holds one token's block of 128)
        if (warp > kLoadX) {
            const int half = (warp - kLoadX - 1) * 2 + (lane >> 4), l = lane & 15;
            uint32_t s = 0, ph = 0;
            for (int i0 = 0; ok && i0 < count; i0 += kFuseAhead) {
                uint4 v[kFuseAhead][kTokens / 8];
#pragma unroll
                for (int a = 0; a < kFuseAhead; ++a)
#pragma unroll
                    for (int t = 0; t < kTokens / 8; ++t) {
                        const int token = token0 + t * 8 + half, col = (begin + i0 + a) * kFp8Block + l * 8;
                        const int valid = token < p.m && i0 + a < count ? p.k - col : 0;
                        const uint16_t* src = p.x16 + token * p.ldx + col;
                        v[a][t] = p.vec ? load_8x16<true>(src, valid) : load_8x16<false>(src, valid);
                    }
#pragma unroll
                for (int a = 0; a < kFuseAhead; ++a) {
                    if (i0 + a >= count) break;
                    ok = mbar_wait_converged(smem_u32(&ctl->empty[s]), ph ^ 1u, abort_flag, p.status, kStatusDense) &&
                         mbar_wait_converged(smem_u32(&ctl->scale_free[s]), ph ^ 1u, abort_flag, p.status, kStatusDense);
                    if (!ok) break;
                    const uint32_t tile = smem_base + s * S::kStageBytes + S::kWeightBytes;
#pragma unroll
                    for (int t = 0; t < kTokens / 8; ++t) {
                        const int row = t * 8 + half;       // rows past the last token stay as they are: nobody reads their sums
                        float f[8];
                        to_float8<kBf16>(v[a][t], f);
                        float m = amax8(f);
#pragma unroll
                        for (int d = 8; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
                        const LinearScale c(fmaxf(m, kAmaxFloor));
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] = c(f[j]);
                        if (token0 + row < p.m) {
                            const uint32_t at = tile + row * 128 + (static_cast<uint32_t>((l >> 1) ^ (row & 7)) << 4) + (l & 1) * 8;
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(pack_e4m3x4(f[0], f[1], f[2], f[3])),
                                         "r"(pack_e4m3x4(f[4], f[5], f[6], f[7]))
                                         : "memory");
                            if (l == 0) ctl->scale[s][row] = c.scale;
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    mbar_arrive_elect(smem_u32(&ctl->full[s]));
                    if (++s == kStages) { s = 0; ph ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == kLoadW || warp == kLoadX) {
        // ------------------------------ loads
        uint32_t s = 0, ph = 0;
        for (int i = 0; i < count; ++i) {
            ok = mbar_wait_converged(smem_u32(&ctl->empty[s]), ph ^ 1u, abort_flag, p.status, kStatusDense);
            if (!ok) break;
            const uint32_t dst = smem_base + s * S::kStageBytes;
            const int k0 = (begin + i) * (kFp8 ? 128 : 64);
            if (warp == kLoadW) {
                const uint32_t bar = smem_u32(&ctl->full[s]);
                mbar_arrive_expect_tx_elect(bar, S::kWeightBytes);
                tma_load_2d_elect(dst, &p.w[0], bar, k0, w_row);
                if constexpr (!kFp8) tma_load_2d_elect(dst + 16384, &p.w[1], bar, k0, w_row);
            } else {
                const uint32_t bar = smem_u32(&ctl->full[s]);
                mbar_arrive_expect_tx_elect(bar, S::kTokenBytes);
                tma_load_2d_elect(dst + S::kWeightBytes, &p.x, bar, k0, token0);
            }
            if (++s == kStages) { s = 0; ph ^= 1u; }
        }
        if (!ok)
            for (int i = 0; i < 64; ++i) __nanosleep(2000);   // error path: let copies in flight land
        __syncwarp();
    } else if (kFp8 && !kFuse && warp == kScale) {
        // ------------------------------ scales: products s_A s_B, a batch of blocks at a time
        constexpr int kPer = kTokens / 32 < 1 ? 1 : kTokens / 32;
        const float* sb = p.sfb + (w_row / kFp8Block) * p.sfb_row + begin * p.sfb_col;
        const float* sa[kPer];
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
            const int token = token0 + r * 32 + lane;           // tokens past the last get scales that exist; nobody reads their sums
            sa[r] = p.sfa + (token < p.m ? token : 0) * p.sfa_row + begin * p.sfa_col;
        }
        uint32_t batch = 0;
        for (int i0 = 0; i0 < count; i0 += kFewBatch, ++batch) {
            ok = mbar_wait_converged(smem_u32(&ctl->scale_free[batch & 1]), ((batch >> 1) & 1) ^ 1u, abort_flag, p.status, kStatusDense);
            if (!ok) break;
            float a[kFewBatch][kPer], b[kFewBatch];
#pragma unroll
            for (int j = 0; j < kFewBatch; ++j) {
                const int at = i0 + j < count ? i0 + j : count - 1;
#pragma unroll
                for (int r = 0; r < kPer; ++r) a[j][r] = sa[r][at * p.sfa_col];
                b[j] = sb[at * p.sfb_col];
            }
#pragma unroll
            for (int j = 0; j < kFewBatch; ++j)
#pragma unroll
                for (int r = 0; r < kPer; ++r)
                    if (kTokens >= 32 || lane < kTokens) ctl->scale[(batch & 1) * kFewBatch + j][r * 32 + lane] = a[j][r] * b[j];
            mbar_arrive(smem_u32(&ctl->scale_full[batch & 1]));
        }
        __syncwarp();
    } else if (warp == kMma) {
        // ------------------------------ MMA issuer
        constexpr uint32_t kIdesc = idesc_dense(128, kTokens, kFp8 ? 0u : (kBf16 ? 1u : 0u), false, false);
        uint32_t s = 0, ph = 0;
        for (int i = 0; i < count; ++i) {
            const int buf = i % S::kBuffers;
            ok = mbar_wait_converged(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, kStatusDense);
            if (kFp8 && ok && i >= S::kBuffers)
                ok = mbar_wait_converged(smem_u32(&ctl->acc_release[buf]), (i / S::kBuffers - 1) & 1, abort_flag, p.status, kStatusDense);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t w = dense_desc_lo<false>(smem_base + s * S::kStageBytes);
            const uint32_t t = w + (S::kWeightBytes >> 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (kFp8) {
                    tc_mma_f8_one(tmem_base + buf * kTokens, w + 2 * j, t + 2 * j, kIdesc, j > 0 ? 1u : 0u);
                } else {
                    const uint32_t more = (i > 0 || j > 0) ? 1u : 0u;
                    tc_mma_f16_one(tmem_base, w + 2 * j, t + 2 * j, kIdesc, more);
                    tc_mma_f16_one(tmem_base + kTokens, w + (16384u >> 4) + 2 * j, t + 2 * j, kIdesc, more);
                }
            }
            if constexpr (kFp8) tc_commit_elect(smem_u32(&ctl->acc_full[buf]));
            tc_commit_elect(smem_u32(&ctl->empty[s]));
            if (++s == kStages) { s = 0; ph ^= 1u; }
        }
        if constexpr (!kFp8)
            if (ok) tc_commit_elect(smem_u32(&ctl->acc_full[0]));
        __syncwarp();
    } else if constexpr (kFp8) {
        // ------------------------------ sums of the blocks
        uint64_t acc[kMine / 2];
#pragma unroll
        for (int j = 0; j < kMine / 2; ++j) acc[j] = 0;
        const float* sb = p.sfb + (w_row / kFp8Block) * p.sfb_row + begin * p.sfb_col;
        float b_next = kFuse && count > 0 ? sb[0] : 0.0f;
        const uint32_t lanes = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + (warp >> 2) * kMine;
        uint32_t s = 0, ph = 0;
        for (int i = 0; i < count; ++i) {
            const uint64_t b2 = pack_f32x2(__float_as_uint(b_next), __float_as_uint(b_next));
            if (kFuse && i + 1 < count) b_next = sb[(i + 1) * p.sfb_col];
            // the scales: with their stage, or with their batch; then the sums
            const int buf = i % S::kBuffers, batch = i / kFewBatch;
            if constexpr (kFuse)
                ok = mbar_wait_converged(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, kStatusDense);
            else if (i % kFewBatch == 0)
                ok = mbar_wait_converged(smem_u32(&ctl->scale_full[batch & 1]), (batch >> 1) & 1, abort_flag, p.status, kStatusDense);
            ok = ok && mbar_wait_converged(smem_u32(&ctl->acc_full[buf]), (i / S::kBuffers) & 1, abort_flag, p.status, kStatusDense);
            if (!ok) break;
            tc_fence_after_sync();
            const int slot = kFuse ? static_cast<int>(s) : (batch & 1) * kFewBatch + i % kFewBatch;
            const uint32_t scales = smem_u32(&ctl->scale[slot][(warp >> 2) * kMine]);
#pragma unroll
            for (int c = 0; c < kMine / kChunk; ++c) {
                uint32_t v[kChunk];
                tc_ld_cols<kChunk>(lanes + buf * kTokens + c * kChunk, v);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < kChunk / 4; ++j) {
                    uint32_t f0, f1, f2, f3;
                    ld_shared_v4(scales + (c * kChunk + 4 * j) * 4, f0, f1, f2, f3);
                    uint64_t lo = pack_f32x2(f0, f1), hi = pack_f32x2(f2, f3);
                    if constexpr (kFuse) {
                        lo = mul_f32x2(lo, b2);
                        hi = mul_f32x2(hi, b2);
                    }
                    fma_f32x2(acc[c * (kChunk / 2) + 2 * j], pack_f32x2(v[4 * j], v[4 * j + 1]), lo);
                    fma_f32x2(acc[c * (kChunk / 2) + 2 * j + 1], pack_f32x2(v[4 * j + 2], v[4 * j + 3]), hi);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            mbar_arrive_elect(smem_u32(&ctl->acc_release[buf]));
            if (kFuse || i % kFewBatch == kFewBatch - 1)
                mbar_arrive_elect(smem_u32(&ctl->scale_free[kFuse ? static_cast<int>(s) : batch & 1]));
            if (++s == kStages) { s = 0; ph ^= 1u; }
        }
#pragma unroll
        for (int j = 0; j < kMine / 2; ++j) {
            const float2 two = unpack_f32x2(acc[j]);
            sum[2 * j] = two.x;
            sum[2 * j + 1] = two.y;
        }
    } else {
        ok = __all_sync(0xffffffffu, mbar_wait<true>(smem_u32(&ctl->acc_full[0]), 0, abort_flag, p.status, kStatusDense));
        tc_fence_after_sync();
    }

    // ------------------------------ results
    const int tokens = p.m - token0 < kTokens ? p.m - token0 : kTokens;
    const int row = w_row + (warp & 3) * 32 + lane;                 // summing warps: this lane's weight row = column of C
    const int first = (warp >> 2) * kMine;                          // and first token
    const uint32_t area = smem_base + ((warp & 3) * 32 + lane) * 4; // exchange: [g | u][token][128 rows]
    uint16_t* out = p.c + token0 * p.ldc + row;
    if (splits == 1) {
        if (warp < kSumWarps && ok) {
            if constexpr (kFp8) {
#pragma unroll
                for (int t = 0; t < kMine; ++t)
                    if (first + t < tokens && row < p.n) out[(first + t) * p.ldc] = to_16<kBf16>(sum[t]);
            } else {
                const uint32_t acc = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
#pragma unroll 1
                for (int c = 0; c < kTokens / 16; ++c) {
                    uint32_t g[16], u[16];
                    tc_ld_x16(acc + c * 16, g);
                    tc_ld_x16(acc + kTokens + c * 16, u);
                    tc_wait_ld();
#pragma unroll
                    for (int t = 0; t < 16; ++t)
                        if (c * 16 + t < tokens && row < p.n)
                            out[(c * 16 + t) * p.ldc] =
                                to_16<kBf16>(gate<false>(__uint_as_float(g[t]), p.gelu).value * __uint_as_float(u[t]));
                }
            }
        }
    } else {
        // every stage has been consumed (the last accumulator is complete): its memory now holds the partial sums
        if (warp < kSumWarps && ok) {
            if constexpr (kFp8) {
#pragma unroll
                for (int t = 0; t < kMine; ++t)
                    if (first + t < tokens) st_shared_f32(area + (first + t) * 512, sum[t]);
            } else {
                const uint32_t acc = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
#pragma unroll 1
                for (int c = 0; c < kTokens / 16; ++c) {
                    uint32_t g[16], u[16];
                    tc_ld_x16(acc + c * 16, g);
                    tc_ld_x16(acc + kTokens + c * 16, u);
                    tc_wait_ld();
#pragma unroll
                    for (int t = 0; t < 16; ++t)
                        if (c * 16 + t < tokens) {
                            st_shared_f32(area + (c * 16 + t) * 512, __uint_as_float(g[t]));
                            st_shared_f32(area + (kTokens + c * 16 + t) * 512, __uint_as_float(u[t]));
                        }
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        // token t is summed by rank t % splits, in rank order
        if (warp < kSumWarps) {
            // tokens at a time: what the registers of one or two CTAs per SM hold
            constexpr int kFull = (S::kCtasPerSm == 1 ? 2 : 1) * (kFp8 ? 2 : 1);
            if (splits <= 2) few_sum_ranks<kOp, kTokens, kBf16, 2, 2 * kFull>(p, smem_base, w_row, token0, tokens, rank, splits, warp, kSumWarps, lane);
            else few_sum_ranks<kOp, kTokens, kBf16, 8, kFull / 2 < 1 ? 1 : kFull / 2>(p, smem_base, w_row, token0, tokens, rank, splits, warp, kSumWarps, lane);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();            // nobody leaves while its sums are read
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kMma) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, S::kTmemCols);
    }
}

}  // namespace b200
