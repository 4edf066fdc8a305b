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

// Rows: sixteen lanes hold one block of 128 columns in registers (one 16-byte load each), agree on its
// largest magnitude with four shuffles and write eight codes each; x is read once.  kRowUnits blocks per
// half-warp are loaded before the first is reduced.  Bound by memory: 3 bytes + 1/32 per element.
constexpr int kRowUnits = 4;
constexpr int kRowThreads = 256;
template <bool kBf16, bool kPow2, bool kVec>
__global__ void __launch_bounds__(kRowThreads)
fp8_quantize_rows(const uint16_t* __restrict__ x, long long ldx, int rows, int k, uint8_t* __restrict__ q, long long ldq,
                  float* __restrict__ sf, long long sf_row, long long sf_col) {
    griddep_wait();
    griddep_launch_dependents();   // in this order: whoever starts from here on finds all work before this kernel complete
    const unsigned blocks_k = (k + kFp8Block - 1) / kFp8Block;
    const unsigned units = static_cast<unsigned>(rows) * blocks_k;       // below 2^32 (checked on the host)
    const int half = threadIdx.x >> 4, l = threadIdx.x & 15;
    const unsigned first = blockIdx.x * (kRowThreads / 16 * kRowUnits) + half;
    uint4 v[kRowUnits];
    unsigned row[kRowUnits], blk[kRowUnits];
#pragma unroll
    for (int i = 0; i < kRowUnits; ++i) {
        const unsigned u = first + i * (kRowThreads / 16);
        row[i] = u / blocks_k;
        blk[i] = u - row[i] * blocks_k;
        const int col = blk[i] * kFp8Block + l * 8;
        v[i] = load_8x16<kVec>(x + row[i] * ldx + col, u < units ? k - col : 0);
    }
#pragma unroll
    for (int i = 0; i < kRowUnits; ++i) {
        const int col = blk[i] * kFp8Block + l * 8;
        float f[8];
        to_float8<kBf16>(v[i], f);
        float m = amax8(f);
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        if (first + i * (kRowThreads / 16) >= units) continue;
        m = fmaxf(m, kAmaxFloor);
        float scale;
        if constexpr (kPow2) {
            const PowerScale c(m);
            scale = c.scale;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = c(f[j]);
        } else {
            const LinearScale c(m);
            scale = c.scale;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = c(f[j]);
        }
        store_codes(q + row[i] * ldq + col, f, k - col);
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

// Values of a quantised matrix as 16-bit numbers (exact for power-of-two scales).  Eight columns per thread.
template <bool kBf16>
__global__ void __launch_bounds__(256)
fp8_dequantize_rows(const uint8_t* __restrict__ q, long long ldq, const float* __restrict__ sf, long long sf_row,
                    long long sf_col, int rows, int k, uint16_t* __restrict__ out, long long ldo) {
    griddep_launch_dependents();
    griddep_wait();
    const unsigned per_row = (k + 7) / 8;
    const unsigned u = blockIdx.x * 256u + threadIdx.x;                 // rows * per_row < 2^32 (checked on the host)
    const unsigned r = u / per_row;
    if (r >= static_cast<unsigned>(rows)) return;
    const int col = (u - r * per_row) * 8;
    const float s = sf[r * sf_row + (col / kFp8Block) * sf_col];
    const int valid = k - col;
    const uint8_t* src = q + r * ldq + col;
    uint16_t* dst = out + r * ldo + col;
    uint2 c = make_uint2(0, 0);
    if (valid >= 8) {
        c = *reinterpret_cast<const uint2*>(src);
    } else {
        for (int i = 0; i < valid; ++i) (i < 4 ? c.x : c.y) |= static_cast<uint32_t>(src[i]) << (8 * (i & 3));
    }
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = unpack_e4m3x2((i < 2 ? c.x : c.y) >> (16 * (i & 1)));
        o[i] = pack_16<kBf16>(t.x * s, t.y * s);
    }
    if (valid >= 8 && (ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
        for (int i = 0; i < 8 && i < valid; ++i) dst[i] = static_cast<uint16_t>(o[i >> 1] >> (16 * (i & 1)));
    }
}

}  // namespace b200
