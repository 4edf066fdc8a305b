// C = (A . s_A) (B . s_B)^T for e4m3 operands in the block format of fp8_blocks.cuh: A [m, k] with one fp32
// scale for each row and 128 columns, B [n, k] with one for each 128 x 128 block, C 16-bit.
//
//   C[i, j] = sum_b s_A[i, b] s_B[j / 128, b] sum_{c in block b} A[i, c] B[j, c]
//
// The inner sums run on the tensor cores (tcgen05 kind::f8f6f4, fp32 accumulation in tensor memory) and are
// fresh for every block; the outer sum is kept in fp32 registers: scales of the block format are arbitrary
// fp32 numbers, which the block-scaled MMA kinds (8-bit exponents) cannot take.
//
// CTA pairs, 256 x 256 tiles.  One 128-wide block of k is 512 clocks of MMA per pair (8192 multiply-adds per
// clock and SM); meanwhile the eight promotion warps of each SM read the 128 x 256 sums of the block before
// (tensor memory, two buffers of 256 columns) and add them, scaled, to 128 registers per thread with packed
// fp32 pairs: 64 fma.f32x2 per thread and block, 128 issue slots per scheduler.
// Ten warps: 0-7 promotion and epilogue (quadrant w % 4, columns 128 (w / 4) ..), 8 MMA issuer, 9 TMA producer.
#pragma once

#include "dense_tiles.cuh"

namespace b200 {

struct Fp8Problem {
    CUtensorMap a, b, c;
    const float* sfa;            // [row * sfa_row + block * sfa_col]
    const float* sfb;            // [(column / 128) * sfb_row + block * sfb_col]
    long long sfa_row, sfa_col, sfb_row, sfb_col;
    int m, n, k_tiles;           // k_tiles: 128-wide blocks
    int m_tiles, n_tiles;        // 256 x 256
    uint32_t* status;
};

constexpr int kFp8Stages = 6;
constexpr uint32_t kFp8OperandBytes = 128u * 128u;
constexpr uint32_t kFp8StageBytes = 2u * kFp8OperandBytes;
constexpr uint32_t kFp8StagingBytes = 8u * 4096u;
constexpr int kFp8Threads = 384;     // warps 10 and 11 only complete the third warpgroup's register hand-back
// Registers: 384 threads start with 168 each; two promotion warpgroups take 216, the third keeps 72 (256 * 216 + 128 * 72 =
// 384 * 168).
constexpr uint32_t kFp8PromoteRegs = 216, kFp8OtherRegs = 72;
static_assert(256 * kFp8PromoteRegs + 128 * kFp8OtherRegs <= 384 * 168, "register split");

struct Fp8Control {
    uint64_t full[kFp8Stages], empty[kFp8Stages];
    uint64_t acc_full[2], acc_release[2], done;
    uint32_t tmem_base, abort_flag;
};
constexpr uint32_t kFp8SmemBytes = 1024u + kFp8Stages * kFp8StageBytes + kFp8StagingBytes + sizeof(Fp8Control);
static_assert(kFp8SmemBytes <= 227u * 1024u, "shared memory budget");

template <bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFp8Threads, 1)
fp8_gemm_pair(const __grid_constant__ Fp8Problem p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    Fp8Control* ctl = reinterpret_cast<Fp8Control*>(smem_raw + (smem_base - smem_u32(smem_raw)) +
                                                    kFp8Stages * kFp8StageBytes + kFp8StagingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles = p.m_tiles * p.n_tiles;
    volatile uint32_t* abort_flag = &ctl->abort_flag;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kFp8Stages; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&ctl->acc_full[b]), 1);
            mbar_init(smem_u32(&ctl->acc_release[b]), 16);   // eight promotion warps of each CTA; used in the first
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
        for (int tile = pair; ok && tile < tiles; tile += pairs) {
            const TileAt t = banded_tile(tile, p.m_tiles, p.n_tiles);
            const int a_row = t.m * 256 + static_cast<int>(rank) * 128, b_row = t.n * 256 + static_cast<int>(rank) * 128;
            for (int i = 0; i < p.k_tiles; ++i) {
                if (!__all_sync(0xffffffffu, mbar_wait<true>(smem_u32(&ctl->empty[s]), ph ^ 1u, abort_flag, p.status, kStatusDense))) {
                    ok = false;
                    break;
                }
                const uint32_t dst = smem_base + s * kFp8StageBytes;
                const uint32_t bar = map_to_cta(smem_u32(&ctl->full[s]), 0);
                if (rank == 0) mbar_arrive_expect_tx_elect(smem_u32(&ctl->full[s]), 2 * kFp8StageBytes);   // both CTAs' bytes
                tma_load_2d_pair_elect(dst, &p.a, bar, i * 128, a_row);
                tma_load_2d_pair_elect(dst + kFp8OperandBytes, &p.b, bar, i * 128, b_row);
                if (++s == kFp8Stages) { s = 0; ph ^= 1u; }
            }
        }
        if (!ok)
            for (int i = 0; i < 64; ++i) __nanosleep(2000);   // error path: let copies in flight land
        __syncwarp();
      } else if (warp == 8) {
        // ------------------------------ MMA issuer
        if (rank == 0) {
            constexpr uint32_t kIdesc = idesc_dense(256, 256, 0u, false, false);
            uint32_t s = 0, ph = 0, cnt = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < tiles; tile += pairs) {
#pragma unroll 1
                for (int i = 0; i < p.k_tiles; ++i, ++cnt) {
                    ok = mbar_wait<true>(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, kStatusDense);
                    if (ok && cnt >= 2)
                        ok = mbar_wait<true>(smem_u32(&ctl->acc_release[cnt & 1]), ((cnt >> 1) - 1) & 1, abort_flag, p.status, kStatusDense);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t a = dense_desc_lo<false>(smem_base + s * kFp8StageBytes);
                    const uint32_t acc = tmem_base + (cnt & 1) * 256;
#pragma unroll
                    for (int j = 0; j < 4; ++j)     // 32 e4m3 elements of k = 32 bytes each
                        tc_mma_f8_pair(acc, a + 2 * j, a + (kFp8OperandBytes >> 4) + 2 * j, kIdesc, j > 0 ? 1u : 0u);
                    tc_commit_pair_both_elect(smem_u32(&ctl->acc_full[cnt & 1]), 3);
                    tc_commit_pair_both_elect(smem_u32(&ctl->empty[s]), 3);
                    if (++s == kFp8Stages) { s = 0; ph ^= 1u; }
                }
            }
            tc_commit_pair_elect(smem_u32(&ctl->done));
            mbar_wait<true>(smem_u32(&ctl->done), 0, abort_flag, p.status, kStatusDense);
        }
        __syncwarp();
      }
    } else {
        warpgroup_reg_inc<kFp8PromoteRegs>();
        // ------------------------------ promotion and epilogue: 32 rows x 128 columns per warp, one row per lane
        const int quad = warp & 3, half = warp >> 2;
        BoxWriter<1> w{smem_base + kFp8Stages * kFp8StageBytes + static_cast<uint32_t>(warp) * 4096u, lane, 0};
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * 128;
        uint32_t cnt = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < tiles; tile += pairs) {
            const TileAt t = banded_tile(tile, p.m_tiles, p.n_tiles);
            const int row = t.m * 256 + static_cast<int>(rank) * 128 + quad * 32, col = t.n * 256 + half * 128;
            const bool exists = row + lane < p.m && col < p.n;
            const float* sa = p.sfa + (row + lane) * p.sfa_row;
            const float* sb = p.sfb + (col / kFp8Block) * p.sfb_row;
            float a_next = exists ? sa[0] : 0.0f, b_next = exists ? sb[0] : 0.0f;
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
#pragma unroll 1
            for (int i = 0; i < p.k_tiles; ++i, ++cnt) {
                const float f = a_next * b_next;
                const uint64_t scale = pack_f32x2(__float_as_uint(f), __float_as_uint(f));
                if (exists && i + 1 < p.k_tiles) {       // a block ahead: arrives while this one is worked on
                    a_next = sa[(i + 1) * p.sfa_col];
                    b_next = sb[(i + 1) * p.sfb_col];
                }
                if (!mbar_wait_warp(smem_u32(&ctl->acc_full[cnt & 1]), (cnt >> 1) & 1, lane, abort_flag, p.status, kStatusDense)) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                // the next 32 columns are on their way while these are added
                const uint32_t src = lane_base + (cnt & 1) * 256;
                uint32_t v[2][32];
                tc_ld_x32(src, v[0]);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c < 3) {
                        tc_ld_x32(src + (c + 1) * 32, v[(c + 1) & 1]);
                    } else {                             // everything read: the buffer goes back
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&ctl->acc_release[cnt & 1]), 0));
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        fma_f32x2(acc[c * 16 + j], pack_f32x2(v[c & 1][2 * j], v[c & 1][2 * j + 1]), scale);
                    if (c < 3) tc_wait_ld();
                }
            }
            if (!ok) break;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const uint32_t box = w.acquire();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        f[2 * j] = __uint_as_float(static_cast<uint32_t>(acc[part * 32 + c * 16 + j]));
                        f[2 * j + 1] = __uint_as_float(static_cast<uint32_t>(acc[part * 32 + c * 16 + j] >> 32));
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
