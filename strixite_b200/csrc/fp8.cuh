// FP8 (e4m3) with a scale per block of 128: what the norm, the SwiGLU and the products share.
//   rows      q [R, K] e4m3 bytes, scale [R, ceil(K / 128)] FP32: value = q * scale of the row's 128-column block
//   matrices  q [N, K], scale [ceil(N / 128), ceil(K / 128)]: one scale per 128 x 128 block (the last ones may be partial)
#pragma once

#include "common.cuh"

namespace sb {

constexpr int kFp8Block = 128;
inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

#ifdef __CUDACC__
// The largest magnitude of a, v and w; a NaN in any stays one (fmaxf would drop it).
__device__ __forceinline__ float max_abs(float a, float v, float w) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(v), "f"(w));
    return r;
}
__device__ __forceinline__ float max_abs(float a, float v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(v)));
    return r;
}
__device__ __forceinline__ float max_abs8(const float (&v)[8]) {
    return max_abs(max_abs(v[0], v[1], v[2]), max_abs(v[3], v[4], v[5]), max_abs(v[6], v[7]));
}

// Two values in e4m3, round to nearest even, saturating at +-448 (NaN -> the NaN code); `lo` in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float fast_rcp(float d) {  // 1 ulp; 1 / d inside FP32's normal range
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}

// What the 8 values of a thread are to the block that they belong to: v = hi + lo unevaluated, so that a product's rounding does not reach
// the codes. An e4m3 code changes where the value crosses the middle between two neighbours; every FP32 rounding in front of it
// moves a value across with a chance of about 2^-21, and a matrix has tens of millions of them.
struct Block8 {
    float hi[8], lo[8];
};

// Two FP32 values in one register pair: an instruction for both, each half rounded as the scalar one rounds it.
using Pair2 = uint64_t;
__device__ __forceinline__ Pair2 two(float a, float b) {
    Pair2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair2 both(float a) { return two(a, a); }
__device__ __forceinline__ void halves(Pair2 p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ Pair2 mul2(Pair2 a, Pair2 b) {
    Pair2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair2 fma2(Pair2 a, Pair2 b, Pair2 c) {
    Pair2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// The 8 N values (times `unit`, a factor that the block shares) as e4m3 bytes of v / scale, scale = max(amax * unit, 2^-100) / 448: the largest
// magnitude gets the largest e4m3 value, and a block of zeros has a scale that divides. A NaN stays one. The quotient is taken against
// the block's largest in front of the scale's own rounding, in which the unit cancels: 448 / (amax + amax_lo) as two floats, three FMAs
// a value. Only the norm of FP32 rows passes the largest value's second part; the others leave amax_lo at 0, and a block whose largest
// was rounded has its codes at a scale that is off by up to 2^-24.
template <int N>
__device__ __forceinline__ void fp8_pack(const Block8 (&v)[N], float amax, float amax_lo, float unit, float &scale, uint2 (&codes)[N]) {
    const float top = amax * unit;
    if (top >= 0x1p-100f && amax > 0x1p-60f && amax < 0x1p60f) {
        const float s = top * (1.0f / 448.0f);
        scale = fmaf(fmaf(-s, 448.0f, top), 1.0f / 448.0f, s);
        float r = fast_rcp(amax);
        r = fmaf(fmaf(-r, amax, 1.0f), r, r);
        const float inv = 448.0f * r, rest = fmaf(-inv, amax_lo, fmaf(-inv, amax, 448.0f)) * r;  // 448 / (amax + amax_lo) = inv + rest
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Pair2 hi = two(v[n].hi[2 * i], v[n].hi[2 * i + 1]), lo = two(v[n].lo[2 * i], v[n].lo[2 * i + 1]);
                float a, b;
                halves(fma2(hi, both(inv), fma2(hi, both(rest), mul2(lo, both(inv)))), a, b);
                h[i] = e4m3x2(a, b);
            }
            codes[n] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        }
    } else {  // near FP32's ends, zero, infinite or NaN: word for word
        scale = __fdiv_rn(max_abs(0x1p-100f, top), 448.0f);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = e4m3x2(__fdiv_rn(v[n].hi[2 * i] * unit, scale), __fdiv_rn(v[n].hi[2 * i + 1] * unit, scale));
            codes[n] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
        }
    }
}

// silu(g) * u of 8 pairs. e^-g for |g| < 80 is 2^t with t = -g log2(e) in two parts (log2(e) = 1.44269502 + 1.93e-8), the second applied to
// first order: off by the 2^-22 of ex2.approx and two roundings. g / (1 + e) by the approximate reciprocal and one correction by the
// exact remainder (Markstein's step). Where a gate is near the ends of the exponential's range (or infinite, or NaN), as the definition
// says. In pairs, because the kernel is bound by the instructions that it issues.
__device__ __forceinline__ void swiglu8(const float (&g)[8], const float (&u)[8], Block8 &h) {
    if (max_abs8(g) < 80.0f) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const Pair2 gg = two(g[j], g[j + 1]), uu = two(u[j], u[j + 1]);
            const Pair2 t = mul2(gg, both(1.44269502f)), rest = fma2(gg, both(-1.92596299e-8f), fma2(gg, both(-1.44269502f), t));  // -t is 2's exponent
            float t0, t1, e0, e1, d0, d1;
            halves(t, t0, t1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(-t0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(-t1));
            Pair2 e = two(e0, e1);
            e = fma2(mul2(e, both(0.693147181f)), rest, e);
            const Pair2 minus_d = fma2(e, both(-1.0f), both(-1.0f));
            halves(minus_d, d0, d1);
            const Pair2 r = two(fast_rcp(-d0), fast_rcp(-d1)), q = mul2(gg, r), silu = fma2(fma2(q, minus_d, gg), r, q);
            const Pair2 hi = mul2(silu, uu);
            halves(hi, h.hi[j], h.hi[j + 1]);
            halves(fma2(silu, uu, mul2(hi, both(-1.0f))), h.lo[j], h.lo[j + 1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h.hi[j] = silu_f(g[j]) * u[j], h.lo[j] = 0.f;
    }
}

// Two values in BF16, round to nearest even; `lo` in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The largest of LANES neighbouring lanes (those that hold the 128 values of a block); NaN if one is.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) v = max_abs(v, __shfl_xor_sync(0xffffffffu, v, off));
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
    *reinterpret_cast<uint4 *>(p) = make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
}
// The values that a store8 followed by a load8 gives back, and the store.
__device__ __forceinline__ void store8_and_keep(float *p, float (&v)[8]) { store8(p, v); }
__device__ __forceinline__ void store8_and_keep(uint16_t *p, float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = bf16x2(v[2 * i], v[2 * i + 1]);
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
#endif  // __CUDACC__

}  // namespace sb
