// FP8 (e4m3) with a scale per block of 128: what the norm, the SwiGLU and the products share.
//   rows      q [R, K] e4m3 bytes, scale [R, ceil(K / 128)] FP32: value = q * scale of the row's 128-column block
//   matrices  q [N, K], scale [ceil(N / 128), ceil(K / 128)]: one scale per 128 x 128 block (the last ones may be partial)
#pragma once

#include "common.cuh"

namespace sb {

constexpr int kFp8Block = 128;
inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

#ifdef __CUDACC__
// |v| as an integer that orders like |v|, with every NaN above infinity: an integer maximum keeps a NaN that fmaxf would drop.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The scale of a block from its largest magnitude: 448 (the largest e4m3 value) stands for it. The floor 2^-100 gives a block of
// zeros a scale that divides and keeps the quotient away from the subnormals; a NaN stays one.
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
    const uint32_t floor_bits = 0x0D800000u;  // 2^-100
    return __uint_as_float(amax_bits < floor_bits ? floor_bits : amax_bits) / 448.0f;
}

// Two values in e4m3, round to nearest even, saturating at +-448 (NaN -> the NaN code); `lo` in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// 8 values of one block -> 8 e4m3 bytes of v / scale. An IEEE division, as the definition says: a reciprocal moves values that lie
// next to a rounding border.
__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8], float scale) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = e4m3x2(__fdiv_rn(v[2 * i], scale), __fdiv_rn(v[2 * i + 1], scale));
    return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// The largest abs_bits among the 16 lanes of a half warp (the 16 x 8 values of a block).
__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
        const uint32_t o = __shfl_xor_sync(0xffffffffu, v, off);
        v = o > v ? o : v;
    }
    return v;
}

// 8 consecutive activations, 16-byte (BF16) or 2 x 16-byte (FP32) accesses.
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const uint16_t *p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(uint16_t *p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f32_to_bf16_bits(v[2 * i]) | ((uint32_t)f32_to_bf16_bits(v[2 * i + 1]) << 16);
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
#endif  // __CUDACC__

}  // namespace sb
