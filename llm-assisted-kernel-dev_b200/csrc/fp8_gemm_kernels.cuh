// C = (A . s_A) (B . s_B)^T for e4m3 operands in the block format of fp8_blocks.cuh: A [m, k] with one fp32
// scale for each row and 128 columns, B [n, k] with one for each 128 x 128 block, C 16-bit.
//
//   C[i, j] = sum_b s_A[i, b] s_B[j / 128, b] sum_{c in block b} A[i, c] B[j, c]
//
// The inner sums run on the tensor cores (tcgen05 kind::f8f6f4, fp32 accumulation in tensor memory) and are
// fresh for every block; the outer sum is kept in fp32 registers: scales of the block format are arbitrary
// fp32 numbers, which the block-scaled MMA kinds (8-bit exponents) cannot take.
//
// CTA pairs, 256 x 256 tiles (or 256 x 128).  One 128-wide block of k is 512 clocks of MMA per pair (8192 multiply-adds per
// clock and SM); meanwhile the eight promotion warps of each SM read the 128 x 256 sums of the block before
// (tensor memory, two buffers of 256 columns) and add them, scaled, to 128 registers per thread with packed
// fp32 pairs.  That is what bounds the kernel: the 64 fma.f32x2 per thread and block alone take 328 clocks, with the
// tensor-memory loads and MMAs running beside them 460, and with the hand-overs of the two buffers about 700.
// Measured for it (clocks per block, this loop without loads): 32 columns at a time 585, 16 warps of 64 columns 623, a
// test of the next buffer ahead of time 670, one lane polling 850.  In the whole kernel: scales fetched by the promotion
// warps 1000, tiles found by divisions 600 more per tile, C stored from registers (32 bytes per lane) 1200 more per
// tile than through boxes.  m=8192 n=14336 k=4096: 414 us in a burst (2.32 PFLOP/s), 470 to 515 under the power cap;
// the library's product with one scale for each whole matrix 399 there.
// Twelve warps: 0-7 promotion and epilogue (quadrant w % 4, columns 128 (w / 4) ..), 8 MMA issuer, 9 TMA producer,
// 10 scale products.
#pragma once

#include "dense_tiles.cuh"

namespace b200 {

struct Fp8Problem {
    CUtensorMap a, b, c;
    const float* sfa;            // [row * sfa_row + block * sfa_col]
    const float* sfb;            // [(column / 128) * sfb_row + block * sfb_col]
    long long sfa_row, sfa_col, sfb_row, sfb_col;
    int m, n, k_tiles;           // k_tiles: 128-wide blocks
    int m_tiles, n_tiles;        // of 256 x kN
    uint32_t* status;
};

constexpr int kFp8Batch = 8;             // blocks whose scales are handed over at a time
constexpr uint32_t kFp8OperandBytes = 128u * 128u;
constexpr uint32_t kFp8StagingBytes = 8u * 8192u;            // per promotion warp two boxes of 32 rows x 128 bytes
constexpr int kFp8Threads = 384;     // warp 11 only completes the third warpgroup's register hand-back
// Registers: 384 threads start with 168 each; two promotion warpgroups take 216, the third keeps 72 (256 * 216 + 128 * 72 =
// 384 * 168).
constexpr uint32_t kFp8PromoteRegs = 216, kFp8OtherRegs = 72;
static_assert(256 * kFp8PromoteRegs + 128 * kFp8OtherRegs <= 384 * 168, "register split");

// Tiles of 256 x kN.  256 is the full-rate shape; 128 takes 0.62 to 0.68 of its time and is taken where 256 leaves pairs idle.
template <int kN> struct Fp8Shape {
    static constexpr uint32_t kStageBytes = kFp8OperandBytes + kN / 2 * 128u;
    static constexpr int kStages = kN == 256 ? 4 : 5;
    static constexpr int kBuffers = 512 / kN;                    // accumulators that take turns
    // scale products: two batches of kFp8Batch blocks x [128-wide column block][128 rows]
    static constexpr uint32_t kBlockBytes = kN / 128 * 512u;
    static constexpr uint32_t kBatchBytes = kFp8Batch * kBlockBytes;
    static constexpr uint32_t kRingAt = kStages * kStageBytes + kFp8StagingBytes;
    static constexpr uint32_t kControlAt = kRingAt + 2u * kBatchBytes;
};
struct Fp8Control {
    uint64_t full[5], empty[5];
    uint64_t acc_full[4], acc_release[4], scale_full[2], scale_free[2], done;
    uint32_t tmem_base, abort_flag;
    int2 place[4];               // row and column of the tiles whose scales are in the ring
};
template <int kN> constexpr uint32_t fp8_smem_bytes() { return 1024u + Fp8Shape<kN>::kControlAt + sizeof(Fp8Control); }
static_assert(fp8_smem_bytes<256>() <= 227u * 1024u && fp8_smem_bytes<128>() <= 227u * 1024u, "shared memory budget");

template <bool kBf16, int kN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFp8Threads, 1)
fp8_gemm_pair(const __grid_constant__ Fp8Problem p) {
    using S = Fp8Shape<kN>;
    constexpr int kStages = S::kStages, kBuffers = S::kBuffers;
    constexpr int kWarpCols = kN / 2;        // columns of one promotion warp
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    Fp8Control* ctl = reinterpret_cast<Fp8Control*>(smem_raw + (smem_base - smem_u32(smem_raw)) + S::kControlAt);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        for (int b = 0; b < kBuffers; ++b) {
            mbar_init(smem_u32(&ctl->acc_full[b]), 1);
            mbar_init(smem_u32(&ctl->acc_release[b]), 16);   // eight promotion warps of each CTA; used in the first
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&ctl->scale_full[b]), 32);    // every lane of the scale warp
            mbar_init(smem_u32(&ctl->scale_free[b]), 8);     // the promotion warps
        }
        mbar_init(smem_u32(&ctl->done), 1);
        ctl->abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == 8) {
        tmem_alloc_pair(smem_u32(&ctl->tmem_base), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    cluster_arrive();
    cluster_wait();            // both CTAs' barriers exist
    const uint32_t tmem_base = ctl->tmem_base;
    griddep_launch_dependents();   // after this CTA has its tensor memory: a CTA of the next kernel cannot take it away
    griddep_wait();

    if (warp >= 8) {
        warpgroup_reg_dec<kFp8OtherRegs>();
        if (warp == 9) {
            // ------------------------------ producer: this CTA's 128 rows of A and of B
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, 1); ok && t.valid(); t.next()) {
                const int a_row = t.m * 256 + static_cast<int>(rank) * 128, b_row = t.n * kN + static_cast<int>(rank) * (kN / 2);
                for (int i = 0; i < p.k_tiles; ++i) {
                    if (!__all_sync(0xffffffffu, mbar_wait<true>(smem_u32(&ctl->empty[s]), ph ^ 1u, abort_flag, p.status, kStatusDense))) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = smem_base + s * S::kStageBytes;
                    const uint32_t bar = map_to_cta(smem_u32(&ctl->full[s]), 0);
                    if (rank == 0) mbar_arrive_expect_tx_elect(smem_u32(&ctl->full[s]), 2 * S::kStageBytes);   // both CTAs' bytes
                    tma_load_2d_pair_elect(dst, &p.a, bar, i * 128, a_row);
                    tma_load_2d_pair_elect(dst + kFp8OperandBytes, &p.b, bar, i * 128, b_row);
                    if (++s == kStages) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok)
                for (int i = 0; i < 64; ++i) __nanosleep(2000);   // error path: let copies in flight land
            __syncwarp();
        } else if (warp == 10) {
            // ------------------------------ scales: products s_A s_B of this CTA's 128 rows and both column halves
            const uint32_t ring = smem_base + S::kRingAt;
            uint32_t batch = 0, nth = 0;
            bool ok = true;
            for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, 1); ok && t.valid(); t.next(), ++nth) {
                const int row0 = t.m * 256 + static_cast<int>(rank) * 128, col = t.n * kN;
                // rows and columns past the matrix get scales that exist; what they scale is never stored
                const float* sa[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) sa[r] = p.sfa + (row0 + r * 32 + lane < p.m ? row0 + r * 32 + lane : 0) * p.sfa_row;
                const float* sb = p.sfb + (col / kFp8Block) * p.sfb_row;
                const long long next_half = col + 128 < p.n ? p.sfb_row : 0;
                for (int i0 = 0; i0 < p.k_tiles; i0 += kFp8Batch, ++batch) {
                    ok = mbar_wait_converged(smem_u32(&ctl->scale_free[batch & 1]), ((batch >> 1) & 1) ^ 1u, abort_flag, p.status, kStatusDense);
                    if (!ok) break;
                    if (i0 == 0 && lane == 0) ctl->place[nth & 3] = make_int2(row0, col);
                    const uint32_t dst = ring + (batch & 1) * S::kBatchBytes + lane * 4;
#pragma unroll
                    for (int part = 0; part < kFp8Batch; part += 4) {
                        float a[4][4], b[4][kN / 128];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int at = i0 + part + j < p.k_tiles ? i0 + part + j : p.k_tiles - 1;
#pragma unroll
                            for (int r = 0; r < 4; ++r) a[j][r] = sa[r][at * p.sfa_col];
                            b[j][0] = sb[at * p.sfb_col];
                            if constexpr (kN == 256) b[j][1] = sb[at * p.sfb_col + next_half];
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                st_shared_f32(dst + (part + j) * S::kBlockBytes + r * 128, a[j][r] * b[j][0]);
                                if constexpr (kN == 256) st_shared_f32(dst + (part + j) * S::kBlockBytes + 512 + r * 128, a[j][r] * b[j][1]);
                            }
                    }
                    mbar_arrive(smem_u32(&ctl->scale_full[batch & 1]));
                }
            }
            __syncwarp();
        } else if (warp == 8) {
            // ------------------------------ MMA issuer
            if (rank == 0) {
                constexpr uint32_t kIdesc = idesc_dense(256, kN, 0u, false, false);
                uint32_t s = 0, ph = 0, cnt = 0;
                bool ok = true;
                for (TileWalk t(pair, pairs, p.m_tiles, p.n_tiles, 1); ok && t.valid(); t.next()) {
#pragma unroll 1
                    for (int i = 0; i < p.k_tiles; ++i, ++cnt) {
                        ok = mbar_wait_converged(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, kStatusDense);
                        const uint32_t buf = cnt % kBuffers;
                        if (ok && cnt >= kBuffers)
                            ok = mbar_wait_converged(smem_u32(&ctl->acc_release[buf]), (cnt / kBuffers - 1) & 1, abort_flag, p.status,
                                                     kStatusDense);
                        if (!ok) break;
                        tc_fence_after_sync();
                        const uint32_t a = dense_desc_lo<false>(smem_base + s * S::kStageBytes);
                        const uint32_t acc = tmem_base + buf * kN;
#pragma unroll
                        for (int j = 0; j < 4; ++j)     // 32 e4m3 elements of k = 32 bytes each
                            tc_mma_f8_pair(acc, a + 2 * j, a + (kFp8OperandBytes >> 4) + 2 * j, kIdesc, j > 0 ? 1u : 0u);
                        tc_commit_pair_both_elect(smem_u32(&ctl->acc_full[buf]), 3);
                        tc_commit_pair_both_elect(smem_u32(&ctl->empty[s]), 3);
                        if (++s == kStages) { s = 0; ph ^= 1u; }
                    }
                }
                tc_commit_pair_elect(smem_u32(&ctl->done));
                mbar_wait<true>(smem_u32(&ctl->done), 0, abort_flag, p.status, kStatusDense);
            }
            __syncwarp();
        }
    } else {
        warpgroup_reg_inc<kFp8PromoteRegs>();
        // ------------------------------ promotion and epilogue: 32 rows x kN / 2 columns per warp, one row per lane
        const int quad = warp & 3, half = warp >> 2;
        BoxWriter w{smem_base + kStages * S::kStageBytes + static_cast<uint32_t>(warp) * 8192u, lane, 0};
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * kWarpCols;
        const uint32_t ring = smem_base + S::kRingAt + (kN == 256 ? half * 512 : 0) + (quad * 32 + lane) * 4;
        const uint32_t scale_full = smem_u32(&ctl->scale_full[0]), scale_free = smem_u32(&ctl->scale_free[0]);
        const uint32_t acc_full = smem_u32(&ctl->acc_full[0]), release = map_to_cta(smem_u32(&ctl->acc_release[0]), 0);
        uint32_t cnt = 0, batch = 0;
        bool ok = true;
        // where a tile lies is only needed at its end: the scale warp, which walks the tiles, hands it over with the scales
        const int mine = (p.m_tiles * p.n_tiles - pair + pairs - 1) / pairs;
        for (int nth = 0; ok && nth < mine; ++nth) {
            // the scale of block i, read while the block before is being added
            auto next_scale = [&](int i) {
                if (i % kFp8Batch == 0) {
                    if (i > 0) mbar_arrive_elect(scale_free + 8 * (batch++ & 1));
                    ok = mbar_wait_converged(scale_full + 8 * (batch & 1), (batch >> 1) & 1, abort_flag, p.status, kStatusDense);
                }
                const uint32_t f = ld_shared_u32(ring + (batch & 1) * S::kBatchBytes + (i % kFp8Batch) * S::kBlockBytes);
                return pack_f32x2(f, f);
            };
            uint64_t acc[kWarpCols / 2];
#pragma unroll
            for (int i = 0; i < kWarpCols / 2; ++i) acc[i] = 0;
            uint64_t scale = next_scale(0);
#pragma unroll 1
            for (int i = 0; ok && i < p.k_tiles; ++i) {
                const uint32_t buf = cnt % kBuffers;
                if (!mbar_wait_converged(acc_full + 8 * buf, (cnt / kBuffers) & 1, abort_flag, p.status, kStatusDense)) {
                    ok = false;
                    break;
                }
                ++cnt;
                tc_fence_after_sync();
                const uint32_t src = lane_base + buf * kN;
                uint64_t scale_next = scale;
#pragma unroll
                for (int c = 0; c < kWarpCols / 32; ++c) {
                    uint32_t v[32];
                    tc_ld_x32(src + c * 32, v);
                    tc_wait_ld();
                    if (c == kWarpCols / 32 - 1) {       // everything read: the buffer goes back
                        tc_fence_before_sync();
                        mbar_arrive_cluster_relaxed_elect(release + 8 * buf);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) fma_f32x2(acc[c * 16 + j], pack_f32x2(v[2 * j], v[2 * j + 1]), scale);
                    if (c == kWarpCols / 64 - 1 && i + 1 < p.k_tiles) scale_next = next_scale(i + 1);
                }
                scale = scale_next;
            }
            if (!ok) break;
            const int2 at = ctl->place[nth & 3];
            const int row = at.x + quad * 32, col = at.y + half * kWarpCols;
            __syncwarp();
            mbar_arrive_elect(scale_free + 8 * (batch++ & 1));
#pragma unroll
            for (int part = 0; part < kWarpCols / 64; ++part) {
                const uint32_t box = w.acquire();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 two = unpack_f32x2(acc[part * 32 + c * 16 + j]);
                        f[2 * j] = two.x;
                        f[2 * j + 1] = two.y;
                    }
                    put_chunk<kBf16>(w, box, c * 4, f);
                }
                w.send(box, &p.c, col + part * 64, row, row < p.m && col + part * 64 < p.n);
            }
        }
        if (lane == 0) bulk_wait_group_read_all();
        __syncwarp();
    }
    // Nobody leaves while the partner may still signal its barriers or while MMAs run on this SM.
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp == 8) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

}  // namespace b200
