// What the 16-bit and 8-bit floating-point GEMMs on CTA pairs share: the order in which tiles are walked and the
// way a tile leaves the SM.
#pragma once

#include "fp8_blocks.cuh"

namespace b200 {

constexpr uint32_t kStatusDense = 0x100;   // a wait of these kernels ran out

// Tiles are walked in bands of eight row tiles, rows fastest inside a band: the pairs that run at the same
// time then share about 8 row tiles and 9 column tiles, whose operands stay in L2 along the k range.
constexpr int kTileBand = 8;
struct TileWalk {
    int m, n, batch;             // the tile
    int tile, tiles, step;
    __device__ TileWalk(int first, int step_, int m_tiles_, int n_tiles, int batches)
        : tile(first), tiles(m_tiles_ * n_tiles * batches), step(step_), m_tiles(m_tiles_), band_tiles(kTileBand * n_tiles),
          per_batch(m_tiles_ * n_tiles) {
        batch = first / per_batch;
        const int in_batch = first - batch * per_batch;
        band = in_batch / band_tiles;
        at = in_batch - band * band_tiles;
        place();
    }
    __device__ bool valid() const { return tile < tiles; }
    // The following tile of this pair.  Subtractions instead of divisions: three of those cost 600 clocks, which the
    // fp8 kernel's promotion warps do not have between two tiles.
    __device__ void next() {
        tile += step;
        at += step;
        while (true) {
            const int here = min(kTileBand, m_tiles - band * kTileBand) * (band_tiles / kTileBand);
            if (at < here) break;
            at -= here;
            if (++band * kTileBand >= m_tiles) {
                band = 0;
                ++batch;
                if (tile >= tiles) break;
            }
        }
        place();
    }

private:
    int m_tiles, band_tiles, per_batch, band, at;
    __device__ void place() {
        const int height = min(kTileBand, m_tiles - band * kTileBand);
        n = height == kTileBand ? at / kTileBand : at / height;
        m = band * kTileBand + at - n * height;
    }
};

// One epilogue warp's way out: 32 rows x 128 bytes at a time through two swizzled boxes (4 KiB each) and the
// TMA unit, which clips rows and columns past the matrix.
struct BoxWriter {
    uint32_t base;      // this warp's two boxes
    int lane;
    uint32_t turn;
    __device__ uint32_t acquire() {      // box to fill next; the copy that last read it is done
        if (lane == 0) bulk_wait_group_read_1();
        __syncwarp();
        return base + (turn & 1u) * 4096u;
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

template <bool kBf16>
__device__ __forceinline__ void put_chunk(BoxWriter& w, uint32_t box, int unit0, const float (&f)[32]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w.put(box, unit0 + j, pack_16<kBf16>(f[8 * j], f[8 * j + 1]), pack_16<kBf16>(f[8 * j + 2], f[8 * j + 3]),
              pack_16<kBf16>(f[8 * j + 4], f[8 * j + 5]), pack_16<kBf16>(f[8 * j + 6], f[8 * j + 7]));
}

}  // namespace b200
