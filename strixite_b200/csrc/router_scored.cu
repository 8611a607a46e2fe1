// Score-based routing: softmax or sigmoid scores of the experts, a balance bias that takes part in the choice but not in the weights,
// expert groups of which a few stay open, top-k, renormalised weights.
//
//   s_e = softmax(l)_e or sigmoid(l_e);  c_e = s_e + bias_e
//   group g = experts [g * E/G, (g + 1) * E/G): value = the largest c of the group, or the sum of its two largest
//   the topk_group largest groups are open (ties: lower group); the k largest c of open groups are the picks (ties: lower expert)
//   coef = s_pick (/ the picks' sum) * route_scale
//
// The order is decided by the 64-bit values of c (without a bias: by the logits, which order the scores): two experts whose sums agree to
// 32 bits still have an order, and a token's experts do not depend on the last bit of an exponential. The kernel works in FP32 with a bound
// on its own error; a token in which two values that the choice tells apart lie closer than that bound is done again in 64 bits.
#include "common.cuh"

#include "strixite_b200.h"

#include <cfloat>
#include <climits>

namespace {

using namespace sb;

constexpr int kWarps = 2;        // tokens per block (16384 x 512 with 1, 2, 4, 8: 23.3, 22.5, 23.5, 23.2 us; 4097 x 160: 7.0, 5.3, 5.3, 9.8)
constexpr int kMaxCand = 256;    // candidates a token may have in the FP32 path
constexpr int64_t kMaxExperts = 1024, kMaxTopK = 32, kMaxGroups = 32;
enum Score : int { kSoftmax = 0, kSigmoid = 1 };

struct RouteArgs {
    int64_t ld, M;
    int E, k, score, G, topk_group, group_top, renorm;
    float route_scale;
    const float *bias;
    int64_t shared_ld;
    int32_t shared_id;
    int32_t *ids;
    float *coef;
    int A;
    int per, L, log_L;  // experts of a group; lanes of a group: 32 / (G rounded up to a power of two)
    uint32_t *err;
};

// Order-preserving maps to unsigned integers (no NaN; -0 and +0 are equal).
__device__ __forceinline__ uint32_t order_key(float f) {
    uint32_t u = __float_as_uint(f);
    if (u == 0x80000000u) u = 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ uint64_t order_key(double v) {
    uint64_t u = (uint64_t)__double_as_longlong(v);
    if (u == 0x8000000000000000ull) u = 0;
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}

// A score in 64 bits (softmax: top and sum of the token's exponentials).
__device__ __noinline__ double score_64(float l, float top, double sum, int kind) {
    const double e = exp(kind == kSigmoid ? -(double)l : (double)l - (double)top);
    return kind == kSigmoid ? 1.0 / (1.0 + e) : e / sum;
}
// sum of exp(l - top) over a token's experts, one warp.
template <typename T>
__device__ __noinline__ double softmax_sum_64(const T *row, int E, float top) {
    double sum = 0.0;
#pragma unroll 4
    for (int e = threadIdx.x & 31; e < E; e += 32) sum += exp((double)ld_act(row, e) - (double)top);
    return warp_sum_d(sum);
}

// A token in 64 bits from end to end, one warp, finite logits and bias: for what the FP32 path leaves (scores outside FP32's range, hundreds
// of candidates). Lane `sub` of group g holds the group's experts sub, sub + L, .. Seldom run, so its
// loops are not unrolled and its values live in local memory: it must not cost the FP32 path registers.
template <typename T>
__device__ __noinline__ void route_64(const T *row, const RouteArgs &a, int64_t m) {
    const unsigned full = 0xffffffffu;
    const int lane = threadIdx.x & 31, g = lane / a.L, sub = lane % a.L;
    const int n = g < a.G && sub < a.per ? (a.per - sub + a.L - 1) / a.L : 0;
    double c[64];  // of the lane's experts: what they are chosen by
    auto expert = [&](int j) { return g * a.per + sub + a.L * j; };
    float top = -INFINITY;
    double sum = 1.0;
    if (a.score == kSoftmax) {
#pragma unroll 1
        for (int j = 0; j < n; ++j) top = fmaxf(top, ld_act(row, expert(j)));
        top = warp_max(top);
        sum = softmax_sum_64(row, a.E, top);
    }
    auto score = [&](float l) { return score_64(l, top, sum, a.score); };
    const bool biased = a.bias != nullptr;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
        const float l = ld_act(row, expert(j));
        c[j] = biased ? score(l) + (double)a.bias[expert(j)] : (double)l;
    }
    if (a.topk_group < a.G) {
        double b1 = -INFINITY, b2 = -INFINITY;  // the two largest of the lane, then of the group
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            if (c[j] > b1) b2 = b1, b1 = c[j];
            else if (c[j] > b2) b2 = c[j];
        }
#pragma unroll 1
        for (int off = a.L / 2; off > 0; off >>= 1) {
            const double o1 = __shfl_xor_sync(full, b1, off), o2 = __shfl_xor_sync(full, b2, off);
            b2 = o1 > b1 ? fmax(b1, o2) : fmax(b2, o1);
            b1 = fmax(b1, o1);
        }
        double value = b1;
        if (a.group_top == 2 && a.per > 1) value = biased ? b1 + b2 : score((float)b1) + score((float)b2);
        int rank = 0;  // groups in front of this lane's
#pragma unroll 1
        for (int h = 0; h < a.G; ++h) {
            const double o = __shfl_sync(full, value, h * a.L);
            rank += o > value || (o == value && h < g);
        }
        if (g >= a.G || rank >= a.topk_group) {
#pragma unroll 1
            for (int j = 0; j < n; ++j) c[j] = -INFINITY;
        }
    }
    int my_i = -1;
#pragma unroll 1
    for (int r = 0; r < a.k; ++r) {
        double lv = -INFINITY;
        int li = INT_MAX, lj = 0;
#pragma unroll 1
        for (int j = 0; j < n; ++j)
            if (c[j] > lv) lv = c[j], li = expert(j), lj = j;  // ascending with strict >: the lower index survives a tie
        const uint64_t key = order_key(lv);
        const uint32_t hi = (uint32_t)(key >> 32), hmax = __reduce_max_sync(full, hi);
        const uint32_t lmax = __reduce_max_sync(full, hi == hmax ? (uint32_t)key : 0u);
        const unsigned pick = __reduce_min_sync(full, hi == hmax && (uint32_t)key == lmax ? (unsigned)li : UINT_MAX);
        if (lane == r) my_i = (int)pick;
        if ((unsigned)li == pick) c[lj] = -INFINITY;
    }
    const double p = lane < a.k ? score(ld_act(row, my_i)) : 0.0, of_picks = warp_sum_d(p);
    if (lane < a.k) {
        a.ids[m * a.A + lane] = my_i;
        // scores that all underflow to zero stay zero
        a.coef[m * a.A + lane] = (float)((a.renorm ? (of_picks > 0.0 ? p / of_picks : 0.0) : p) * (double)a.route_scale);
    }
}

// 4 neighbouring logits.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const uint16_t *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}

// One warp per token. The lanes are dealt to the groups (a group's L neighbouring lanes hold its experts, NV a lane, in runs of four where
// VEC), so a group's value is a reduction over L lanes and a closed group is a lane that drops out.
// The choice: the k-th largest lane maximum bounds the k-th largest value from below, what reaches it are the candidates (about 1.3 k of
// them), they meet in shared memory and each counts those in front of it: no k rounds of warp-wide maxima. Where neighbours in that
// order are closer than the error, the candidates are valued again in 64 bits (one token in a thousand).
// Bound by the instructions issued, 1046 a token: 16384 x 512 experts, 10 of 4 of 8 groups, 22.2 us, of which the loads are 4.9, scores 2.9,
// groups 3.5, candidates and their order 7, the last step 4. Groups that do not fill the vectors load element by element (16384 x 1008 in
// 16 groups: 78 us), and with as many picks as open lanes the bound is near the least lane maximum, so that most experts are
// candidates (32 of 256 in one group: 249 us).
//
// The FP32 errors that the choice allows for (documented bounds: expf 2 ulp; ex2.approx 2^-22, rcp.approx 2^-23 relative):
//   sigmoid  e = 2^(-l log2 e): the argument's roundings move e by 1.5 |l| 2^-24, so p by p (1 - p) (2^-22 + 1.5 |l| 2^-24) <= 0.7 * 2^-23; 1 + e
//            and the reciprocal by 1.5 * 2^-23: 2.2 * 2^-23, for two values 4.4 * 2^-23 < 2^-20
//            relative to p itself the factor 1 - p no longer helps where l is negative: (7 + 1.5 |l|) 2^-24 < 2^-20 + 2^-23 |l|; for
//            l > 0, (1 - p) l < 0.28: 7.5 * 2^-24 < 2^-20
//   softmax  e = expf(l - top): (2 + |x| / 2) 2^-23 of e; the sum of up to 64 a lane and 5 steps: 35 * 2^-23 and the terms' mean, at most
//            2 + ln(1024) / 2; p by at most 45 * 2^-23 of the largest p, for two values 90 * 2^-23 < 2^-16
//            relative to p itself: its exponential's error with |x| < 88 and the sum's, below 2^-16 p
//   c = p + bias one rounding each, 2^-24 |c|: 2^-22 (|c| + |c'|) is above both; 2^-120 is above what is lost where a score is flushed to zero
__device__ __forceinline__ float fast_sigmoid(float l) {
    float e, p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(l * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.0f + e));
    return p;
}

struct PerToken {
    union {
        struct {
            float2 cand[kMaxCand];   // value, expert (as bits)
            double exact[kMaxCand];  // of a close token: the candidates' values in 64 bits
        };
        float dealt[kMaxCand * 4];
    };
};

template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, NV <= 8 ? 14 : 0) router_scored_kernel(const T *logits, const T *shared, const RouteArgs a) {
    __shared__ PerToken tokens[kWarps];
    __shared__ float2 sorted[kWarps][40];
    const unsigned full = 0xffffffffu;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    PerToken &tok = tokens[warp];
    const int64_t m = (int64_t)blockIdx.x * kWarps + warp;
    let_next_begin();
    wait_for_previous();
    if (m >= a.M) return;  // whole warps leave together; no block-level barrier below
    const int L = a.L, g = lane >> a.log_L, sub = lane & (L - 1);
    const T *row = logits + m * a.ld;
    auto expert = [&](int j) { return VEC ? g * a.per + (j >> 2) * 4 * L + sub * 4 + (j & 3) : g * a.per + sub + L * j; };
    auto holds = [&](int j) { return g < a.G && (VEC ? (j >> 2) * 4 * L + sub * 4 : sub + L * j) < a.per; };

    float c[NV];  // the logits, then what the experts are chosen by
    float chk = 0.f;  // stays 0 while everything is finite: 0 * inf and 0 * NaN are NaN
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < NV; j += 4) {
            float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (holds(j)) {
                v = load4(row + expert(j));
                chk = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, chk))));
            }
            c[j] = v.x, c[j + 1] = v.y, c[j + 2] = v.z, c[j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            c[j] = -INFINITY;
            if (holds(j)) c[j] = ld_act(row, expert(j)), chk = fmaf(c[j], 0.f, chk);
        }
    }
    float sl = 0.f;
    if (shared != nullptr) sl = ld_act(shared, m * a.shared_ld), chk = fmaf(sl, 0.f, chk);

    const bool biased = a.bias != nullptr;
    float top = 0.f, sum = 1.f, base = 0.f;
    if (a.score == kSoftmax) {
        top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) top = fmaxf(top, c[j]);
        top = warp_max(top);
        if (biased || !a.renorm) {
            sum = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) sum += expf(c[j] - top);  // absent experts: exp(-inf) = 0
            sum = warp_sum(sum);
        }
    }
    if (biased) {
        const float inv = 1.0f / sum;
        base = a.score == kSigmoid ? 0x1p-20f : 0x1p-16f * inv;
        auto choose_by = [&](auto score) {
#pragma unroll
            for (int j = 0; j < NV; j += VEC ? 4 : 1) {
                if (!holds(j)) continue;
                if constexpr (VEC) {
                    const float4 v = load4(a.bias + expert(j));
                    chk = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, chk))));
                    c[j] = score(c[j]) + v.x, c[j + 1] = score(c[j + 1]) + v.y, c[j + 2] = score(c[j + 2]) + v.z, c[j + 3] = score(c[j + 3]) + v.w;
                } else {
                    const float v = a.bias[expert(j)];
                    chk = fmaf(v, 0.f, chk);
                    c[j] = score(c[j]) + v;
                }
            }
        };
        if (a.score == kSigmoid) choose_by([](float l) { return fast_sigmoid(l); });
        else choose_by([&](float l) { return expf(l - top) * inv; });
    }
    if (__any_sync(full, !(chk == 0.f))) {  // a non-finite logit or bias fails the token: ids -1, coefficients NaN
        unsigned bad = UINT_MAX;
        for (int e = lane; e < a.E; e += 32)
            if (!isfinite(ld_act(row, e)) || (biased && !isfinite(a.bias[e]))) bad = min(bad, (unsigned)e);
        if (!isfinite(sl)) bad = min(bad, (unsigned)a.E);
        bad = __reduce_min_sync(full, bad);
        if (lane == 0) raise_err(a.err, (uint32_t)m, bad);
        for (int i = lane; i < a.A; i += 32) a.ids[m * a.A + i] = -1, a.coef[m * a.A + i] = qnan();
        return;
    }

    double sum64 = 0.0;  // of the softmax, where something is done in 64 bits
    float lm = -INFINITY;  // the lane's largest; -inf in a closed group
    bool open = g < a.G;
    if (a.topk_group < a.G) {
        float b1 = -INFINITY, b2 = -INFINITY;  // the two largest of the lane, then of the group
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            b2 = fmaxf(b2, fminf(b1, c[j]));
            b1 = fmaxf(b1, c[j]);
        }
        lm = b1;
        for (int off = L / 2; off > 0; off >>= 1) {
            const float o1 = __shfl_xor_sync(full, b1, off), o2 = __shfl_xor_sync(full, b2, off);
            b2 = fmaxf(fmaxf(b2, o2), fminf(b1, o1));
            b1 = fmaxf(b1, o1);
        }
        float value = b1, tol = 0.f;
        if (a.group_top == 2 && a.per > 1) {
            if (biased) value = b1 + b2, tol = 2.f * base + 0x1p-21f * (fabsf(b1) + fabsf(b2));
            else if (a.score == kSigmoid) value = fast_sigmoid(b1) + fast_sigmoid(b2), tol = 0x1p-18f;
            else value = expf(b1 - top) + expf(b2 - top), tol = 0x1p-18f;
        } else if (biased) {
            tol = base + 0x1p-21f * fabsf(b1);
        }
        int rank = 0;  // groups in front of this lane's: a larger value, or the same and a lower group
        const uint32_t key = order_key(value);
#pragma unroll 4
        for (int h = 0; h < a.G; ++h) rank += __shfl_sync(full, key, h << a.log_L) + (h < g) > key;  // no value's key is the largest integer
        open = g < a.G && rank < a.topk_group;
        if (biased || (a.group_top == 2 && a.per > 1)) {  // else the values are exact
            const float worst = __uint_as_float(__reduce_max_sync(full, g < a.G ? __float_as_uint(tol) : 0u));
            const float least_open = key_value(__reduce_min_sync(full, open ? order_key(value) : UINT_MAX));
            const float most_shut = key_value(__reduce_max_sync(full, g < a.G && !open ? order_key(value) : order_key(-INFINITY)));
            if (!(least_open - most_shut > worst)) {
                // Too close to tell: the groups' values in 64 bits, from the experts that FP32 does not rule out as one of their largest.
                if (a.score == kSoftmax) sum64 = softmax_sum_64(row, a.E, top);
                const float least = a.group_top == 2 && a.per > 1 ? b2 : b1, reach = biased ? least - (base + 0x1p-21f * fabsf(least)) : least;
                uint64_t mask = 0;
#pragma unroll
                for (int j = 0; j < NV; ++j) mask |= (uint64_t)(c[j] >= reach && c[j] > -INFINITY) << j;
                double d1 = -INFINITY, d2 = -INFINITY;
#pragma unroll 1
                while (mask != 0) {
                    const int e = expert(__ffsll((long long)mask) - 1);
                    mask &= mask - 1;
                    const double v = score_64(ld_act(row, e), top, sum64, a.score) + (biased ? (double)a.bias[e] : 0.0);
                    d2 = fmax(d2, fmin(d1, v)), d1 = fmax(d1, v);
                }
                __syncwarp();
#pragma unroll 1
                for (int off = L / 2; off > 0; off >>= 1) {
                    const double o1 = __shfl_xor_sync(full, d1, off), o2 = __shfl_xor_sync(full, d2, off);
                    d2 = fmax(fmax(d2, o2), fmin(d1, o1)), d1 = fmax(d1, o1);
                }
                const double exact_value = a.group_top == 2 && a.per > 1 ? d1 + d2 : d1;
                rank = 0;
#pragma unroll 1
                for (int h = 0; h < a.G; ++h) {
                    const double o = __shfl_sync(full, exact_value, h * L);
                    rank += o > exact_value || (o == exact_value && h < g);
                }
                open = g < a.G && rank < a.topk_group;
            }
        }
        if (!open) lm = -INFINITY;
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) lm = fmaxf(lm, c[j]);
    }

    int n = 0;  // candidates
    {
        const unsigned lanes = __ballot_sync(full, open);
        const int many = __popc(lanes);
        if (many * 4 < a.k * 5 && many < 32 && a.topk_group * a.per > 32) {
            // Few lanes are open and hold the experts of all: these are dealt anew, to every lane its share, or the bound would let most of them
            // in (16384 tokens: 16 picks of 512 experts in 16 open lanes 68 -> 27 us, of 256 in 8 lanes 185 -> 46; below the rule, 6 of 64 in
            // 8 lanes, 17.1 -> 17.0, 10 of 256 in 16 lanes 23.4 -> 24.6 us).
            const int total = min(many * ((a.per + L - 1) >> a.log_L), kMaxCand * 4);  // what is not dealt only lowers the bound
            int at = __popc(lanes & ((1u << lane) - 1));
#pragma unroll
            for (int j = 0; j < NV; ++j, at += many)
                if (open && at < total) tok.dealt[at] = c[j];
            __syncwarp();
            lm = -INFINITY;
            for (int i = lane; i < total; i += 32) lm = fmaxf(lm, tok.dealt[i]);
            __syncwarp();
        }
        // the k-th largest lane maximum: k rounds of the warp's maximum (a hardware reduction of the ordered bits), the lane that held it out
        uint32_t key = order_key(lm), kth_key = 0;
        for (int r = 0; r < a.k; ++r) {
            kth_key = __reduce_max_sync(full, key);
            if (key == kth_key) key = 0;  // equal maxima go together: the bound is only lower
        }
        const float kth = kth_key == 0 ? -INFINITY : key_value(kth_key);
        // what lies below the k-th by no more than the error is a candidate too: nothing that is left out can belong to the picks.
        // -FLT_MAX: every finite value.
        const float bound = open ? fmaxf(biased ? kth - (base + 0x1p-21f * fabsf(kth)) : kth, -FLT_MAX) : INFINITY;
        int mine = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) mine += c[j] >= bound;
        int at = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(full, at, off);
            if (lane >= off) at += o;
        }
        n = __shfl_sync(full, at, 31);
        at -= mine;
        if (n <= kMaxCand) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const bool in = c[j] >= bound;
                if (in) tok.cand[at] = make_float2(c[j], __int_as_float(expert(j)));
                at += in;
            }
            __syncwarp();
            // in front: a larger value, then the lower expert; no two candidates are equal in both, so the ranks are 0 .. n - 1. Up to 32 (nearly
            // always) are compared from the lanes' registers by value, and by expert only where ranks meet.
            if (n <= 32) {
                const float2 own = lane < n ? tok.cand[lane] : make_float2(-INFINITY, 0.f);
                int rank = 0;
#pragma unroll 4
                for (int q = 0; q < n; ++q) rank += __shfl_sync(full, own.x, q) > own.x;
                if (__reduce_or_sync(full, lane < n ? 1u << rank : 0u) != 0xffffffffu >> (32 - n)) {  // n >= k >= 1
                    unsigned same = __match_any_sync(full, __float_as_uint(own.x + 0.f)) & ~(1u << lane);  // -0 is 0
                    for (same = lane < n ? same : 0u; same != 0; same &= same - 1) rank += __float_as_int(tok.cand[__ffs(same) - 1].y) < __float_as_int(own.y);
                }
                if (lane < n && rank <= a.k) sorted[warp][rank] = own;
            }
            for (int i = n <= 32 ? n : lane; i < n; i += 32) {
                const float2 own = tok.cand[i];
                int rank = 0;
#pragma unroll 4
                for (int q = 0; q < n; ++q) {
                    const float2 o = tok.cand[q];
                    rank += o.x > own.x || (o.x == own.x && __float_as_int(o.y) < __float_as_int(own.y));
                }
                if (rank <= a.k) sorted[warp][rank] = own;
            }
            __syncwarp();
        }
    }
    int pick = -1;
    float l = 0.f;
    bool out = n > kMaxCand;  // for the 64-bit path
    if (!out) {
        bool near = false;
        if (biased && lane < a.k && lane + 1 < n) {
            const float value = sorted[warp][lane].x, next = sorted[warp][lane + 1].x;
            near = !(value - next > base + 0x1p-22f * (fabsf(value) + fabsf(next)));
        }
        if (__any_sync(full, near)) {
            // That was the bound for the largest scores; two neighbours among the picks may be small ones, and their own errors tell. (Behind the last
            // pick stand all that are left, with any score: there the bound stays.)
            const float inv = 1.0f / sum;
            auto off = [&](float2 at) {
                const float l = ld_act(row, __float_as_int(at.y));
                return (a.score == kSigmoid ? (0x1p-20f + 0x1p-23f * fmaxf(-l, 0.f)) * fast_sigmoid(l) : 0x1p-16f * (expf(l - top) * inv)) + 0x1p-22f * fabsf(at.x) + 0x1p-120f;
            };
            if (near && lane + 1 < a.k) near = !(sorted[warp][lane].x - sorted[warp][lane + 1].x > off(sorted[warp][lane]) + off(sorted[warp][lane + 1]));
        }
        if (__any_sync(full, near)) {
            // the candidates once more, in 64 bits
            if (a.score == kSoftmax && sum64 == 0.0) sum64 = softmax_sum_64(row, a.E, top);
#pragma unroll 1
            for (int i = lane; i < n; i += 32) {
                const int e = __float_as_int(tok.cand[i].y);
                tok.exact[i] = score_64(ld_act(row, e), top, sum64, a.score) + (double)a.bias[e];
            }
            __syncwarp();
#pragma unroll 1
            for (int i = lane; i < n; i += 32) {
                const float2 own = tok.cand[i];
                const double v = tok.exact[i];
                int rank = 0;
#pragma unroll 1
                for (int q = 0; q < n; ++q) rank += tok.exact[q] > v || (tok.exact[q] == v && __float_as_int(tok.cand[q].y) < __float_as_int(own.y));
                if (rank <= a.k) sorted[warp][rank] = own;
            }
            __syncwarp();
        }
        if (lane < a.k) {
            pick = __float_as_int(sorted[warp][lane].y);
            l = ld_act(row, pick);
            out = (a.score == kSigmoid ? l : l - top) < -80.f;  // the score leaves FP32's normal range
        }
    }
    if (__any_sync(full, out)) {
        const RouteArgs copy = a;  // taking a's own address would move every use of it to local memory (25 -> 34 us at 16384 x 512)
        route_64(row, copy, m);
    } else {
        // The weights in FP32 from the picks' exact logits: scores, their sum, the quotient and the scale round to 2^-24 each (6.7e-8 off on average
        // at 16384 x 512; in 64 bits with one rounding it would be 2.7e-8).
        float p = 0.f;
        if (lane < a.k) {
            if (a.score == kSigmoid) {
                p = sigmoid_f(l);
            } else {
                const float x = l - top, lost = (l - (x - (x - l))) + (-top - (x - l));  // l - top = x + lost exactly
                p = expf(x);
                p = fmaf(p, lost, p);
            }
        }
        const float of_picks = a.renorm ? warp_sum(p) : sum;  // sigmoid without renorm: 1
        if (lane < a.k) {
            a.ids[m * a.A + lane] = pick;
            a.coef[m * a.A + lane] = p / of_picks * a.route_scale;
        }
    }
    if (shared != nullptr && lane == 0) a.ids[m * a.A + a.k] = a.shared_id, a.coef[m * a.A + a.k] = sigmoid_f(sl);
}

template <typename T, bool VEC>
cudaError_t launch(const void *logits, const void *shared, const RouteArgs &a, cudaStream_t st) {
    const int nv = (a.per + a.L - 1) / a.L;
    const unsigned blocks = (unsigned)((a.M + kWarps - 1) / kWarps);
    // a lane's scores stay in NV registers: the steps between powers of two pay (13665 tokens, 524 experts, nv = 17: 38.7 us with
    // 24, 44.6 with 32)
#define SB_ROUTE(NV) launch_after(router_scored_kernel<T, NV, VEC>, dim3(blocks), dim3(kWarps * 32), 0, st, 1, (const T *)logits, (const T *)shared, a)
    return nv <= 4    ? SB_ROUTE(4)
           : nv <= 8  ? SB_ROUTE(8)
           : nv <= 12 ? SB_ROUTE(12)
           : nv <= 16 ? SB_ROUTE(16)
           : nv <= 24 ? SB_ROUTE(24)
           : nv <= 32 ? SB_ROUTE(32)
                      : SB_ROUTE(64);
#undef SB_ROUTE
}

}  // namespace

extern "C" {

int strix_moe_router_scored(const void *logits, int64_t ld, int64_t M, int64_t E, int64_t k, int score, const float *bias, int64_t n_group,
                            int64_t topk_group, int64_t group_top, int renorm, float route_scale, const void *shared_logit, int64_t shared_ld,
                            int32_t shared_id, int32_t *ids, float *coef, int act, uint32_t *err, void *stream) {
    const char *fn = "moe_router_scored";
    SB_CHECK(logits != nullptr && ids != nullptr && coef != nullptr && err != nullptr, fn, ": null pointer (logits=", logits, ", ids=", (const void *)ids,
             ", coef=", (const void *)coef, ", err=", (const void *)err, ")");
    SB_CHECK(M >= 1 && M <= 0x7fffffff, fn, ": M = ", M, " tokens, expected 1..", 0x7fffffff);
    SB_CHECK(E >= 1 && E <= kMaxExperts, fn, ": E = ", E, " experts, expected 1..", kMaxExperts);
    SB_CHECK(score == kSoftmax || score == kSigmoid, fn, ": score ", score, ", expected 0 (softmax) or 1 (sigmoid)");
    SB_CHECK(n_group >= 1 && n_group <= kMaxGroups && E % n_group == 0, fn, ": n_group = ", n_group, ", expected 1..", kMaxGroups,
             " and a divisor of E = ", E);
    SB_CHECK(topk_group >= 1 && topk_group <= n_group, fn, ": topk_group = ", topk_group, ", expected 1..n_group = ", n_group);
    SB_CHECK(group_top == 1 || group_top == 2, fn, ": group_top = ", group_top, ", expected 1 or 2");
    SB_CHECK(k >= 1 && k <= kMaxTopK && k <= topk_group * (E / n_group), fn, ": k = ", k, ", expected 1..min(", kMaxTopK, ", ", topk_group * (E / n_group),
             " experts in open groups)");
    SB_CHECK(ld >= E, fn, ": logits row stride ld = ", ld, " < E = ", E);
    SB_CHECK(route_scale == route_scale && route_scale - route_scale == 0.0f, fn, ": route_scale = ", route_scale, ", expected a finite number");
    SB_CHECK(M == 1 || (ld <= (1 << 28) && (shared_logit == nullptr || shared_ld <= (1 << 28))), fn, ": row strides ", ld, " and ", shared_ld,
             ", expected up to 2^28");
    if (shared_logit != nullptr) {
        SB_CHECK(shared_ld >= 1, fn, ": shared_ld = ", shared_ld, ", expected >= 1");
        SB_CHECK(shared_id >= 0, fn, ": shared_id = ", shared_id, ", expected >= 0 (its expert row block)");
    }
    SB_CHECK(act_ok(act), fn, ": unsupported activation dtype ", act);
    auto off = [](const void *p, int64_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
    SB_CHECK(!off(logits, act_size(act)) && !off(shared_logit, act_size(act)), fn, ": logits ", logits, " and shared_logit ", shared_logit,
             " must be aligned to their elements");
    SB_CHECK(!off(bias, 4) && !off(ids, 4) && !off(coef, 4) && !off(err, 4), fn, ": bias ", (const void *)bias, ", ids ", (const void *)ids, ", coef ",
             (const void *)coef, " and err ", (const void *)err, " must be aligned to 4 bytes");
    const int64_t A = k + (shared_logit != nullptr ? 1 : 0), ob = M * A * 4;
    SB_CHECK(apart(ids, ob, coef, ob), fn, ": ids [", (const void *)ids, "] and coef [", (const void *)coef, "] (", ob, " B each) overlap");
    const int64_t lb = ((M - 1) * ld + E) * act_size(act);
    SB_CHECK(apart(ids, ob, logits, lb) && apart(coef, ob, logits, lb), fn, ": ids or coef overlaps the logits [", logits, ", +", lb, " B)");
    SB_CHECK(bias == nullptr || (apart(ids, ob, bias, E * 4) && apart(coef, ob, bias, E * 4)), fn, ": ids or coef overlaps the bias");
    const int64_t shb = ((M - 1) * shared_ld + 1) * act_size(act);
    SB_CHECK(shared_logit == nullptr || (apart(ids, ob, shared_logit, shb) && apart(coef, ob, shared_logit, shb)), fn, ": ids or coef overlaps the shared logits");
    RouteArgs a{};
    a.ld = ld, a.M = M, a.E = (int)E, a.k = (int)k, a.score = score, a.G = (int)n_group, a.topk_group = (int)topk_group, a.group_top = (int)group_top;
    a.renorm = renorm != 0, a.route_scale = route_scale, a.bias = bias, a.shared_ld = shared_ld, a.shared_id = shared_id, a.ids = ids, a.coef = coef;
    a.A = (int)A, a.err = err;
    int gp = 1;
    while (gp < a.G) gp *= 2;
    a.per = a.E / a.G, a.L = 32 / gp;
    while (1 << a.log_L < a.L) ++a.log_L;
    // runs of four where they fill the lanes of a group evenly and every row starts aligned
    const bool vec = a.per % (4 * a.L) == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % (4 * act_size(act)) == 0 && aligned16(bias);
    auto st = static_cast<cudaStream_t>(stream);
    const cudaError_t rc = act == kF32 ? (vec ? launch<float, true>(logits, shared_logit, a, st) : launch<float, false>(logits, shared_logit, a, st))
                                       : (vec ? launch<uint16_t, true>(logits, shared_logit, a, st) : launch<uint16_t, false>(logits, shared_logit, a, st));
    SB_CUDA(rc, fn, " ", act_name(act), " M=", M, " E=", E, " k=", k, " groups=", n_group);
    return 0;
}

}  // extern "C"
