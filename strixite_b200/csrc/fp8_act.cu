// The two places of a layer where activations become FP8 rows: the RMS norm in front of the FFN (with the residual's addition)
// and the SwiGLU between its two products.
#include "fp8.cuh"

#include "strixite_b200.h"

namespace {

using namespace sb;

constexpr int kNormMaxThreads = 256;
constexpr int kNormMaxVec = 8;  // 8-element pieces a thread can hold: d <= 256 * 8 * 8

// The warps' values (each the same in all lanes of a warp) folded in the order of the warps; what stood in `part` has been read by then.
template <typename F>
__device__ __forceinline__ float block_fold(float *part, float v, F f) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float all = part[0];
#pragma unroll 1
    for (int i = 1; i < (int)blockDim.x / 32; ++i) all = f(all, part[i]);
    return all;
}

// One block per row; a thread holds VEC pieces of 8 consecutive elements in registers, so a row is read once whatever its
// length: x' = x + y rounded to the activation type (what the residual stream keeps), r = 1 / sqrt(mean(x'^2) + eps) from the stored
// values, h = x' r g. 16 neighbouring threads hold one 128-column block: its largest magnitude is a half-warp reduction.
// Bound by memory: nothing is read twice, and the row's values never leave the registers (16384 x 2048 BF16 with residual and h: 53.2 us,
// 5.7 TB/s). A small batch of FP32 rows is bound by its blocks: 64 registers let 6 of 160 threads run on an SM, and the last 113 of 1001 rows
// of 2560 are a second wave (6.3 us).
template <typename T, int VEC>
__global__ void __launch_bounds__(kNormMaxThreads)
    rmsnorm_fp8_kernel(const T *x, const T *y, const float *w, float w_add, float eps, int d, float inv_d, T *x_out, T *h_out, uint8_t *q, float *scale,
                       int blocks) {
    let_next_begin();
    wait_for_previous();
    constexpr int kWarps = kNormMaxThreads / 32;
    constexpr bool kWide = sizeof(T) == 4;
    __shared__ alignas(16) float part[kWarps];
    const int64_t row = blockIdx.x, base = row * d;
    float v[VEC][8];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * 8;
        if (c < d) {
            load8(x + base + c, v[i]);
            if (y != nullptr) {
                float a[8];
                load8(y + base + c, a);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] += a[j];
                store8_and_keep(x_out + base + c, v[i]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(v[i][j], v[i][j], sq);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
    }
    sq = warp_sum(sq);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sq;
    __syncthreads();
    // every thread adds the warps' sums in the same order; a root of the mean by the approximate instruction and one Newton step
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) total += i < (int)blockDim.x / 32 ? part[i] : 0.f;
    const float mean = fmaf(total, inv_d, eps);
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(mean));
    if (mean > 0x1p-100f && mean < 0x1p100f) {
        r = fmaf(r * 0.5f, fmaf(-mean * r, r, 1.0f), r);
    } else {
        // The squares may have left FP32's range or lost their low bits below it; the norm itself is an ordinary number. Once more on the row
        // (and sqrt(eps)) times a power of two that brings the largest to 2^30, or as near as a float gets it: exact (but where h is
        // below 2^-150), and h stays. (Costs other rows 0.1 us at 1001 x 2560 FP32, nothing measurable at the large sizes.)
        float top = sqrtf(eps);
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max_abs(top, max_abs8(v[i]));
        top = block_fold(part, lanes_max<32>(top), [](float a, float b) { return max_abs(a, b); });
        if (top > 0.f && top < INFINITY) {
            const float s = __int_as_float((min(127, 157 - (__float_as_int(top) >> 23)) + 127) << 23);
            sq = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] *= s, sq = fmaf(v[i][j], v[i][j], sq);
            total = block_fold(part, warp_sum(sq), [](float a, float b) { return a + b; });
            r = 1.0f / sqrtf(fmaf(total, inv_d, eps * s * s));
        } else {
            r = 1.0f / sqrtf(mean);
        }
    }
    const bool plain = !(r > 0x1p-60f && r < 0x1p60f);  // a row with an infinity or a NaN, or of zeros with eps 0: h first, then its codes
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = (threadIdx.x + i * blockDim.x) * 8;
        float top = 0.f;
        Block8 part8[1], &p = part8[0];  // x' g in two parts (h / r), or h
        if (c < d) {
            float g[8], h[8];
            load8(w + c, g);
            if (!plain) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float gain = g[j] + w_add;
                    p.hi[j] = v[i][j] * gain;
                    p.lo[j] = fmaf(v[i][j], gain, -p.hi[j]);
                    h[j] = p.hi[j] * r;
                }
                if (kWide && w_add != 0.0f) {  // what the gain's sum rounded off (Knuth's two-sum)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float gain = g[j] + w_add, t = gain - g[j];
                        p.lo[j] = fmaf(v[i][j], (g[j] - (gain - t)) + (w_add - t), p.lo[j]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = p.hi[j] = v[i][j] * r * (g[j] + w_add), p.lo[j] = 0.f;
            }
            top = max_abs8(p.hi);
            if (h_out != nullptr) store8(h_out + base + c, h);
        }
        if (q != nullptr) {  // the same for the whole grid; the reduction runs on full warps
            top = lanes_max<16>(top);
            // FP32 rows: the second part of the block's largest as well (16384 x 2048 BF16 with it: 53 -> 69 us, 7 fewer codes of 34 M that differ from
            // 64 bits; 4096 x 4096 FP32: 46.3 -> 47.3).
            float low = 0.f;
            if constexpr (kWide) {
                low = -INFINITY;
                if (c < d) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (fabsf(p.hi[j]) == top) low = fmaxf(low, p.hi[j] < 0.f ? -p.lo[j] : p.lo[j]);
                }
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) low = fmaxf(low, __shfl_xor_sync(0xffffffffu, low, off));
            }
            if (c < d) {
                float s;
                uint2 codes[1];
                fp8_pack(part8, top, low, plain ? 1.0f : r, s, codes);
                *reinterpret_cast<uint2 *>(q + base + c) = codes[0];
                if ((c & (kFp8Block - 1)) == 0) scale[row * blocks + c / kFp8Block] = s;
            }
        }
    }
}

template <typename T>
cudaError_t launch_norm(const void *x, const void *y, const float *w, float w_add, float eps, int64_t M, int64_t d, void *x_out, void *h, uint8_t *q, float *scale,
                 cudaStream_t st) {
    const int pieces = (int)(d / 8);
    int vec = 1;
    while (vec < kNormMaxVec && pieces > vec * kNormMaxThreads) vec *= 2;
    const int threads = ((pieces + vec - 1) / vec + 31) / 32 * 32;
    const int blocks = (int)fp8_blocks(d);
#define SB_NORM(V) \
    launch_after(rmsnorm_fp8_kernel<T, V>, dim3((unsigned)M), dim3(threads), 0, st, 1, (const T *)x, (const T *)y, w, w_add, eps, (int)d, 1.0f / (float)d, \
                 (T *)x_out, (T *)h, q, scale, blocks)
    return vec == 1 ? SB_NORM(1) : vec == 2 ? SB_NORM(2) : vec == 4 ? SB_NORM(4) : SB_NORM(8);
#undef SB_NORM
}

// u / blocks for u < 2^31: (u * mul) >> shift with mul = ceil(2^shift / blocks), shift = 31 + ceil(log2 blocks) (the excess of mul * blocks
// over 2^shift is below blocks <= 2^(shift - 31), so u times it stays below 2^shift). mul = 0: by division.
struct RowOf {
    uint32_t mul;
    int shift;
};

// Eight lanes per (row, 128-column block) of h = silu(gate) * up, 16 elements a thread. Gate and up stay FP32 until the one rounding
// to e4m3. FP32 rows are bound by memory (40960 x 512: 28.5 us, 6.6 TB/s), BF16 rows by the instructions issued (19.5 us, 5.4 TB/s; with
// 8 elements a thread, whose index, maximum and scale cost as much as those of 16: 25.1 us, and with scalar arithmetic 26.5). Small
// blocks, as many as there is work: 256 threads and blocks that stay for several units: 21.9 us; with 8 blocks an SM for BF16: 20.0.
constexpr int kSwigluThreads = 128, kSwigluUnits = kSwigluThreads / 8;  // of a block
template <typename T>
__global__ void __launch_bounds__(kSwigluThreads, sizeof(T) == 2 ? 10 : 8) swiglu_fp8_kernel(const T *gu, uint8_t *q, float *scale, int64_t units, int I, int blocks, RowOf row_of) {
    let_next_begin();
    wait_for_previous();
    const int t = threadIdx.x & 7;
    const int64_t u = (int64_t)blockIdx.x * kSwigluUnits + threadIdx.x / 8;
    const int64_t row = row_of.mul != 0 ? (int64_t)((uint64_t)(uint32_t)u * row_of.mul >> row_of.shift) : u / blocks;
    const int b = (int)(u - row * blocks), c = b * kFp8Block + t * 16;
    const bool live = u < units && c < I;  // I % 16 == 0
    Block8 h[2];
    float top = 0.f;
    if (live) {
        const T *gate = gu + row * 2 * I + c, *up = gate + I;
        float g[2][8], v[2][8];
        load8(gate, g[0]), load8(gate + 8, g[1]);
        load8(up, v[0]), load8(up + 8, v[1]);
        swiglu8(g[0], v[0], h[0]), swiglu8(g[1], v[1], h[1]);
        top = max_abs(max_abs8(h[0].hi), max_abs8(h[1].hi));
    }
    top = lanes_max<8>(top);
    if (live) {
        float s;
        uint2 codes[2];
        fp8_pack(h, top, 0.f, 1.0f, s, codes);
        *reinterpret_cast<uint4 *>(q + row * I + c) = make_uint4(codes[0].x, codes[0].y, codes[1].x, codes[1].y);
        if (t == 0) scale[u] = s;
    }
}

}  // namespace

extern "C" {

int strix_residual_rmsnorm_fp8(const void *x, const void *y, const float *w, int centered, float eps, int64_t M, int64_t d, void *x_out, void *h,
                               uint8_t *q, float *scale, int act, void *stream) {
    const char *fn = "residual_rmsnorm_fp8";
    SB_CHECK(x != nullptr && w != nullptr, fn, ": null pointer (x=", x, ", w=", (const void *)w, ")");
    SB_CHECK((y == nullptr) == (x_out == nullptr), fn, ": y and x_out come together (y=", y, ", x_out=", x_out, ")");
    SB_CHECK((q == nullptr) == (scale == nullptr), fn, ": q and scale come together (q=", (const void *)q, ", scale=", (const void *)scale, ")");
    SB_CHECK(h != nullptr || q != nullptr, fn, ": neither h nor q is asked for");
    SB_CHECK(act_ok(act), fn, ": unsupported activation dtype ", act);
    SB_CHECK(M >= 1 && M <= 0x7fffffff, fn, ": M = ", M, " rows, expected 1..2^31-1");
    SB_CHECK(d >= 16 && d % 16 == 0 && d <= kNormMaxThreads * kNormMaxVec * 8, fn, ": d = ", d, ", expected a multiple of 16 up to ",
             kNormMaxThreads * kNormMaxVec * 8);
    SB_CHECK(eps >= 0.0f, fn, ": eps = ", eps, ", expected >= 0");
    SB_CHECK(aligned16(x) && aligned16(y) && aligned16(w) && aligned16(x_out) && aligned16(h) && aligned16(q) && reinterpret_cast<uintptr_t>(scale) % 4 == 0,
             fn, ": x, y, w, x_out, h and q must be 16-byte aligned, scale 4-byte");
    const int64_t xb = M * d * act_size(act), qb = M * d, sb_ = M * fp8_blocks(d) * 4, wb = d * 4;
    // a block of threads reads a whole row before it writes h and q, but other rows' blocks run at the same time: only exact aliases
    // of the same rows are harmless
    SB_CHECK(x_out == nullptr || ((x_out == x || apart(x_out, xb, x, xb)) && (x_out == y || apart(x_out, xb, y, xb))), fn,
             ": x_out partly overlaps x or y");
    const void *ins[3] = {x, y, w}, *outs[4] = {x_out, h, q, scale};
    const int64_t in_b[3] = {xb, xb, wb}, out_b[4] = {xb, xb, qb, sb_};
    for (int o = 0; o < 4; ++o) {
        if (outs[o] == nullptr) continue;
        for (int i = 0; i < 3; ++i)
            SB_CHECK(ins[i] == nullptr || (o == 0 && i < 2) || apart(outs[o], out_b[o], ins[i], in_b[i]), fn, ": output ", o, " [", outs[o], ", +", out_b[o],
                     " B) overlaps input ", i, " [", ins[i], ", +", in_b[i], " B)");
        for (int p = 0; p < o; ++p)
            SB_CHECK(outs[p] == nullptr || apart(outs[o], out_b[o], outs[p], out_b[p]), fn, ": outputs ", p, " and ", o, " overlap");
    }
    auto st = static_cast<cudaStream_t>(stream);
    const float w_add = centered ? 1.0f : 0.0f;
    SB_CUDA((act == kF32 ? launch_norm<float>(x, y, w, w_add, eps, M, d, x_out, h, q, scale, st)
                         : launch_norm<uint16_t>(x, y, w, w_add, eps, M, d, x_out, h, q, scale, st)),
            fn, " ", act_name(act), " M=", M, " d=", d);
    return 0;
}

int strix_swiglu_fp8(const void *gu, uint8_t *q, float *scale, int64_t rows, int64_t I, int act, void *stream) {
    const char *fn = "swiglu_fp8";
    SB_CHECK(gu != nullptr && q != nullptr && scale != nullptr, fn, ": null pointer (gu=", gu, ", q=", (const void *)q, ", scale=", (const void *)scale, ")");
    SB_CHECK(act_ok(act), fn, ": unsupported activation dtype ", act);
    SB_CHECK(rows >= 1 && I >= 16 && I % 16 == 0 && I <= (1 << 24), fn, ": rows = ", rows, ", I = ", I, " (I a multiple of 16 up to 2^24)");
    SB_CHECK(rows <= (1ll << 40) / I / 2, fn, ": rows * 2I = ", rows, " * ", 2 * I, " is too large (rows/I swapped?)");
    SB_CHECK(aligned16(gu) && aligned16(q) && reinterpret_cast<uintptr_t>(scale) % 4 == 0, fn, ": gu and q must be 16-byte aligned, scale 4-byte");
    const int64_t gb = rows * 2 * I * act_size(act), qb = rows * I, sb_ = rows * fp8_blocks(I) * 4;
    SB_CHECK(apart(q, qb, gu, gb) && apart(scale, sb_, gu, gb) && apart(q, qb, scale, sb_), fn, ": q [", (const void *)q, "], scale [", (const void *)scale,
             "] and gu [", gu, "] overlap");
    const int blocks = (int)fp8_blocks(I);
    const int64_t units = rows * blocks;  // at most 2^35
    const unsigned grid = (unsigned)((units + kSwigluUnits - 1) / kSwigluUnits);
    SB_CHECK((units + kSwigluUnits - 1) / kSwigluUnits <= 0x7fffffff, fn, ": ", rows, " rows of ", blocks, " blocks are too many");
    auto st = static_cast<cudaStream_t>(stream);
    RowOf row_of{0, 0};
    if (units + kSwigluUnits < (1ll << 31)) {
        int log = 0;
        while ((1 << log) < blocks) ++log;
        row_of.shift = 31 + log;
        row_of.mul = (uint32_t)(((1ull << row_of.shift) + blocks - 1) / blocks);
    }
    SB_CUDA((act == kF32 ? launch_after(swiglu_fp8_kernel<float>, dim3(grid), dim3(kSwigluThreads), 0, st, 1, (const float *)gu, q, scale, units, (int)I, blocks, row_of)
                         : launch_after(swiglu_fp8_kernel<uint16_t>, dim3(grid), dim3(kSwigluThreads), 0, st, 1, (const uint16_t *)gu, q, scale, units, (int)I, blocks, row_of)),
            fn, " ", act_name(act), " rows=", rows, " I=", I);
    return 0;
}

}  // extern "C"
