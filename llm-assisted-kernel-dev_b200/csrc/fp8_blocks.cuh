// The 8-bit block format and the streaming kernels on it.
//
// A row of a matrix is cut into blocks of 128 columns (the last one may be shorter); a block holds one
// fp32 scale s and an e4m3 code for each element, value = code * s.  With a = max(|x|, 2^-100) over the
// block:
//   linear layers        s = a / 448 (rounded once), code = e4m3(448 x / a)
//   kept activations     s = the smallest power of two with a <= 448 s, code = e4m3(x / s): the value is then
//                        a 16-bit number again, bit for bit, and can be an operand of a 16-bit product
// Weights have one scale for each 128 x 128 block, by the first rule.
#pragma once

#include "ptx_dense.cuh"

namespace b200 {

constexpr int kFp8Block = 128;
constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;   // 2^-100: what a block of zeros gets for its largest magnitude

// 448 x / a for |x| <= a.  0.875 x and a / 512 are exact for 16-bit x; the quotient's remainder is exact in
// a fused multiply-add, so one Newton correction makes every quotient that fits fp32 exact.  That is what
// counts: a quotient half way between two codes has five significant bits and is met exactly, and any other
// 16-bit x and a leave it more than 2^-18 away from a half-way point, far more than the rounding errors here.
struct LinearScale {
    float scale, den, inv;
    __device__ explicit LinearScale(float amax) {
        scale = __fdiv_rn(amax, kE4m3Max);
        den = amax * (1.0f / 512.0f);
        inv = __frcp_rn(den);
    }
    __device__ float operator()(float x) const {
        const float num = 0.875f * x;
        const float y = num * inv;
        return fmaf(fmaf(-den, y, num), inv, y);
    }
};
// The smallest power of two s with a <= 448 s = 1.75 * 2^8 s.  Exact for every finite a >= 2^-100; an infinity
// is kept as one (its code saturates and 448 * 2^120 overflows again).
struct PowerScale {
    float scale, inv;
    __device__ explicit PowerScale(float amax) {
        const uint32_t bits = __float_as_uint(amax);
        const uint32_t e = (bits >> 23) - 8u + ((bits & 0x7FFFFFu) > 0x600000u ? 1u : 0u);   // biased exponent of s
        scale = __uint_as_float(e << 23);
        inv = __uint_as_float((254u - e) << 23);
    }
    __device__ float operator()(float x) const { return x * inv; }
};

// Eight 16-bit elements starting at p, of which `valid` exist (the others read as zero).
template <bool kVec> __device__ __forceinline__ uint4 load_8x16(const uint16_t* p, int valid) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (kVec && valid >= 8) {
        v = *reinterpret_cast<const uint4*>(p);
    } else {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < valid ? p[i] : 0u;
        v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
    }
    return v;
}
template <bool kBf16> __device__ __forceinline__ void to_float8(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = unpack_16<kBf16>(w[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ float amax8(const float (&f)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
    return m;
}
// Eight codes at q, of which `valid` are stored.  q is 8-byte aligned (16-byte row pitch, columns in eights).
__device__ __forceinline__ void store_codes(uint8_t* q, const float (&y)[8], int valid) {
    const uint32_t lo = pack_e4m3x4(y[0], y[1], y[2], y[3]), hi = pack_e4m3x4(y[4], y[5], y[6], y[7]);
    if (valid >= 8) {
        *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
    } else {
        for (int i = 0; i < valid; ++i) q[i] = static_cast<uint8_t>((i < 4 ? lo >> (8 * i) : hi >> (8 * (i - 4))));
    }
}

// Sixteen codes at q (16-byte aligned), of which `valid` are stored.
__device__ __forceinline__ void store_codes16(uint8_t* q, const float (&lo)[8], const float (&hi)[8], int valid) {
    if (valid >= 16) {
        *reinterpret_cast<uint4*>(q) = make_uint4(pack_e4m3x4(lo[0], lo[1], lo[2], lo[3]), pack_e4m3x4(lo[4], lo[5], lo[6], lo[7]),
                                                  pack_e4m3x4(hi[0], hi[1], hi[2], hi[3]), pack_e4m3x4(hi[4], hi[5], hi[6], hi[7]));
    } else {
        store_codes(q, lo, valid);
        store_codes(q + 8, hi, valid - 8);
    }
}

// Rows: eight lanes hold one block of 128 columns in registers (two 16-byte loads each), agree on its largest
// magnitude with three shuffles and write sixteen codes each; x is read once.  kRowUnits blocks per eight lanes are
// loaded before the first is reduced.  3 bytes + 1/32 per element; the divisions of a block's scale are the lanes' own,
// so with eight elements per lane they, not memory, bounded it (m=8192 k=4096, 101 MB: 24.3 us, 16 elements 20.5).
constexpr int kRowUnits = 4;
constexpr int kRowThreads = 256;
constexpr int kRowLanes = 8;
template <bool kBf16, bool kPow2, bool kVec>
__global__ void __launch_bounds__(kRowThreads)
fp8_quantize_rows(const uint16_t* __restrict__ x, long long ldx, int rows, int k, uint8_t* __restrict__ q, long long ldq,
                  float* __restrict__ sf, long long sf_row, long long sf_col) {
    griddep_wait();
    griddep_launch_dependents();   // in this order: whoever starts from here on finds all work before this kernel complete
    constexpr unsigned kGroups = kRowThreads / kRowLanes;
    const unsigned blocks_k = (k + kFp8Block - 1) / kFp8Block;
    const unsigned units = static_cast<unsigned>(rows) * blocks_k;       // below 2^32 (checked on the host)
    const int l = threadIdx.x & (kRowLanes - 1);
    const unsigned first = blockIdx.x * (kGroups * kRowUnits) + threadIdx.x / kRowLanes;
    uint4 v[kRowUnits][2];
    unsigned row[kRowUnits], blk[kRowUnits];
#pragma unroll
    for (int i = 0; i < kRowUnits; ++i) {
        const unsigned u = first + i * kGroups;
        row[i] = u / blocks_k;
        blk[i] = u - row[i] * blocks_k;
        const int col = blk[i] * kFp8Block + l * 16;
        const int valid = u < units ? k - col : 0;
        const uint16_t* src = x + row[i] * ldx + col;
        v[i][0] = load_8x16<kVec>(src, valid);
        v[i][1] = load_8x16<kVec>(src + 8, valid - 8);
    }
#pragma unroll
    for (int i = 0; i < kRowUnits; ++i) {
        const int col = blk[i] * kFp8Block + l * 16;
        float f[2][8];
        to_float8<kBf16>(v[i][0], f[0]);
        to_float8<kBf16>(v[i][1], f[1]);
        float m = fmaxf(amax8(f[0]), amax8(f[1]));
#pragma unroll
        for (int s = kRowLanes / 2; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        if (first + i * kGroups >= units) continue;
        m = fmaxf(m, kAmaxFloor);
        float scale;
        if constexpr (kPow2) {
            const PowerScale c(m);
            scale = c.scale;
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j / 8][j % 8] = c(f[j / 8][j % 8]);
        } else {
            const LinearScale c(m);
            scale = c.scale;
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j / 8][j % 8] = c(f[j / 8][j % 8]);
        }
        store_codes16(q + row[i] * ldq + col, f[0], f[1], k - col);
        if (l == 0) sf[row[i] * sf_row + blk[i] * sf_col] = scale;
    }
}

// 128 x 128 blocks (weights): one thread block each, 64 elements per thread kept in registers.
template <bool kBf16, bool kVec>
__global__ void __launch_bounds__(256)
fp8_quantize_blocks(const uint16_t* __restrict__ w, long long ldw, int n, int k, uint8_t* __restrict__ q, long long ldq,
                    float* __restrict__ sf, long long sf_row, long long sf_col) {
    __shared__ float part[8];
    const int row0 = blockIdx.y * kFp8Block + (threadIdx.x >> 4);
    const int col = blockIdx.x * kFp8Block + (threadIdx.x & 15) * 8;
    uint4 v[8];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = row0 + 16 * i;
        v[i] = load_8x16<kVec>(w + r * ldw + col, r < n ? k - col : 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float f[8];
        to_float8<kBf16>(v[i], f);
        m = fmaxf(m, amax8(f));
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = kAmaxFloor;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i]);
    const LinearScale c(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = row0 + 16 * i;
        if (r >= n) break;
        float f[8];
        to_float8<kBf16>(v[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = c(f[j]);
        store_codes(q + r * ldq + col, f, k - col);
    }
    if (threadIdx.x == 0) sf[blockIdx.y * sf_row + blockIdx.x * sf_col] = c.scale;
}

// Values of a quantised matrix as 16-bit numbers (exact for power-of-two scales).  Sixteen columns per thread.
template <bool kBf16>
__global__ void __launch_bounds__(256)
fp8_dequantize_rows(const uint8_t* __restrict__ q, long long ldq, const float* __restrict__ sf, long long sf_row,
                    long long sf_col, int rows, int k, uint16_t* __restrict__ out, long long ldo) {
    griddep_launch_dependents();
    griddep_wait();
    const unsigned per_row = (k + 15) / 16;
    const unsigned u = blockIdx.x * 256u + threadIdx.x;                 // rows * per_row < 2^32 (checked on the host)
    const unsigned r = u / per_row;
    if (r >= static_cast<unsigned>(rows)) return;
    const int col = (u - r * per_row) * 16;
    const float s = sf[r * sf_row + (col / kFp8Block) * sf_col];
    const int valid = k - col;
    const uint8_t* src = q + r * ldq + col;
    uint16_t* dst = out + r * ldo + col;
    uint32_t c[4] = {0, 0, 0, 0};
    if (valid >= 16) {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        c[0] = v.x;
        c[1] = v.y;
        c[2] = v.z;
        c[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < valid) c[i / 4] |= static_cast<uint32_t>(src[i]) << (8 * (i & 3));
    }
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 t = unpack_e4m3x2(c[i / 2] >> (16 * (i & 1)));
        o[i] = pack_16<kBf16>(t.x * s, t.y * s);
    }
    const bool vec = (ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const uint32_t* w = o + part * 4;
        if (vec && valid >= part * 8 + 8) {
            *reinterpret_cast<uint4*>(dst + part * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (part * 8 + i < valid) dst[part * 8 + i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

}  // namespace b200
