// What the 16-bit and 8-bit floating-point GEMMs on CTA pairs share: the order in which tiles are walked and the
// way a tile leaves the SM.
#pragma once

#include "fp8_blocks.cuh"

namespace b200 {

constexpr uint32_t kStatusDense = 0x100;   // a wait of these kernels ran out

// Tiles are walked in bands of eight row tiles, rows fastest inside a band: the pairs that run at the same
// time then share about 8 row tiles and 9 column tiles, whose operands stay in L2 along the k range.
constexpr int kTileBand = 8;
struct TileAt { int m, n, batch; };
__device__ __forceinline__ TileAt banded_tile(int tile, int m_tiles, int n_tiles) {
    TileAt t;
    const int per_batch = m_tiles * n_tiles;
    t.batch = tile / per_batch;
    tile -= t.batch * per_batch;
    const int band = tile / (kTileBand * n_tiles);
    const int left = m_tiles - band * kTileBand;
    const int height = left < kTileBand ? left : kTileBand;
    tile -= band * kTileBand * n_tiles;
    t.n = tile / height;
    t.m = band * kTileBand + tile - t.n * height;
    return t;
}

// One epilogue warp's way out: 32 rows x 128 bytes at a time through its swizzled boxes (4 KiB each) and the
// TMA unit, which clips rows and columns past the matrix.
template <int kBoxes> struct BoxWriter {
    static_assert(kBoxes == 1 || kBoxes == 2, "one box, or two in turn");
    uint32_t base;      // this warp's boxes
    int lane;
    uint32_t turn;
    __device__ uint32_t acquire() {      // box to fill next; the copy that last read it is done
        if (lane == 0) {
            if constexpr (kBoxes == 2) bulk_wait_group_read_1();
            else bulk_wait_group_read_all();
        }
        __syncwarp();
        return base + (kBoxes == 2 ? (turn & 1u) * 4096u : 0u);
    }
    // 16-byte unit `u` of this lane's row
    __device__ void put(uint32_t box, int u, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
        st_shared_v4(box + lane * 128 + (static_cast<uint32_t>(u ^ (lane & 7)) << 4), a, b, c, d);
    }
    __device__ void send(uint32_t box, const void* map, int col, int row, bool inside) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (inside) tma_store_2d(map, box, col, row);
            bulk_commit_group();
        }
        ++turn;
    }
};

template <bool kBf16, int kBoxes>
__device__ __forceinline__ void put_chunk(BoxWriter<kBoxes>& w, uint32_t box, int unit0, const float (&f)[32]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w.put(box, unit0 + j, pack_16<kBf16>(f[8 * j], f[8 * j + 1]), pack_16<kBf16>(f[8 * j + 2], f[8 * j + 3]),
              pack_16<kBf16>(f[8 * j + 4], f[8 * j + 5]), pack_16<kBf16>(f[8 * j + 6], f[8 * j + 7]));
}

}  // namespace b200
