// Score-based routing: softmax or sigmoid scores of the experts, a balance bias that takes part in the choice but not in the weights,
// expert groups of which a few stay open, top-k, renormalised weights.
//
//   s_e = softmax(l)_e or sigmoid(l_e);  c_e = s_e + bias_e
//   group g = experts [g * E/G, (g + 1) * E/G): value = the largest c of the group, or the sum of its two largest
//   the topk_group largest groups are open (ties: lower group); the k largest c of open groups are the picks (ties: lower expert)
//   coef = s_pick (/ the picks' sum) * route_scale
//
// The order is decided by the 64-bit values of c: two experts whose sums agree to 32 bits still have an order, and a token's experts do
// not depend on the last bit of an exponential.
#include "common.cuh"

#include "strixite_b200.h"

#include <climits>

namespace {

using namespace sb;

constexpr int kWarps = 4;
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
    uint32_t *err;
};

// Order-preserving map of a double (no NaN) to 64 bits.
__device__ __forceinline__ uint64_t order_key(double v) {
    uint64_t u = (uint64_t)__double_as_longlong(v);
    if (u == 0x8000000000000000ull) u = 0;  // -0 and +0 are equal
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// One warp per token. The lanes are dealt to the groups: with GP = G rounded up to a power of two, group g belongs to the L = 32 / GP
// lanes from g * L on, and lane `sub` of them holds the group's experts sub, sub + L, .. in registers (NV of them).
template <typename T, int NV>
__global__ void __launch_bounds__(kWarps * 32) router_scored_kernel(const T *logits, const T *shared, const RouteArgs a) {
    const unsigned full = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    const int64_t m = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (m >= a.M) return;  // whole warps leave together; no block-level barrier below
    int gp = 1;
    while (gp < a.G) gp *= 2;
    const int L = 32 / gp, g = lane / L, sub = lane % L, per = a.E / a.G;
    const T *row = logits + m * a.ld;
    auto expert = [&](int j) { return g * per + sub + L * j; };
    auto holds = [&](int j) { return g < a.G && sub + L * j < per; };

    float l[NV];
    float top = -INFINITY;
    unsigned bad = UINT_MAX;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        l[j] = -INFINITY;
        if (holds(j)) {
            l[j] = ld_act(row, expert(j));
            if (!isfinite(l[j]) || (a.bias != nullptr && !isfinite(a.bias[expert(j)]))) bad = min(bad, (unsigned)expert(j));
            top = fmaxf(top, l[j]);
        }
    }
    float sl = 0.f;
    if (shared != nullptr) {
        sl = ld_act(shared, m * a.shared_ld);
        if (!isfinite(sl)) bad = min(bad, (unsigned)a.E);
    }
    bad = __reduce_min_sync(full, bad);
    int32_t *id_row = a.ids + m * a.A;
    float *coef_row = a.coef + m * a.A;
    if (bad != UINT_MAX) {  // a non-finite logit or bias fails the token: ids -1, coefficients NaN
        if (lane == 0) raise_err(a.err, (uint32_t)m, bad);
        for (int i = lane; i < a.A; i += 32) id_row[i] = -1, coef_row[i] = qnan();
        return;
    }

    double p[NV], c[NV];
    if (a.score == kSigmoid) {
#pragma unroll
        for (int j = 0; j < NV; ++j) p[j] = holds(j) ? 1.0 / (1.0 + exp(-(double)l[j])) : 0.0;
    } else {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(full, top, off));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            p[j] = holds(j) ? exp((double)l[j] - (double)top) : 0.0;
            sum += p[j];
        }
        sum = warp_sum_d(sum);
#pragma unroll
        for (int j = 0; j < NV; ++j) p[j] /= sum;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) c[j] = holds(j) ? p[j] + (a.bias != nullptr ? (double)a.bias[expert(j)] : 0.0) : -INFINITY;

    if (a.topk_group < a.G) {
        double b1 = -INFINITY, b2 = -INFINITY;  // the two largest of the lane, then of the group
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (c[j] > b1) b2 = b1, b1 = c[j];
            else if (c[j] > b2) b2 = c[j];
        }
        for (int off = L / 2; off > 0; off >>= 1) {
            const double o1 = __shfl_xor_sync(full, b1, off), o2 = __shfl_xor_sync(full, b2, off);
            b2 = o1 > b1 ? fmax(b1, o2) : fmax(b2, o1);
            b1 = fmax(b1, o1);
        }
        const double value = a.group_top == 2 && per > 1 ? b1 + b2 : b1;
        int rank = 0;  // groups in front of this lane's
        for (int h = 0; h < a.G; ++h) {
            const double o = __shfl_sync(full, value, h * L);
            rank += o > value || (o == value && h < g);
        }
        if (g >= a.G || rank >= a.topk_group) {
#pragma unroll
            for (int j = 0; j < NV; ++j) c[j] = -INFINITY;
        }
    }

    double lv, lp;  // the lane's best candidate: value, score, expert
    int li;
    auto rescan = [&]() {
        lv = -INFINITY, lp = 0.0, li = INT_MAX;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (c[j] > lv) lv = c[j], lp = p[j], li = expert(j);  // ascending with strict >: the lower index survives a tie
    };
    rescan();
    double my_p = 0.0;
    int my_i = -1;
    for (int r = 0; r < a.k; ++r) {
        const uint64_t key = order_key(lv);
        const uint32_t hi = (uint32_t)(key >> 32), hmax = __reduce_max_sync(full, hi);
        const uint32_t lo = hi == hmax ? (uint32_t)key : 0u, lmax = __reduce_max_sync(full, lo);
        const bool best = hi == hmax && (uint32_t)key == lmax;
        const unsigned pick = __reduce_min_sync(full, best ? (unsigned)li : UINT_MAX);
        const bool mine = (unsigned)li == pick;
        const int owner = __ffs(__ballot_sync(full, mine)) - 1;
        const double score = __shfl_sync(full, lp, owner);
        if (lane == r) my_p = score, my_i = (int)pick;
        if (mine) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (holds(j) && expert(j) == (int)pick) c[j] = -INFINITY;
            rescan();
        }
    }
    const double sum = warp_sum_d(my_p);  // lanes >= k hold 0
    if (lane < a.k) {
        id_row[lane] = my_i;
        // scores that all underflow to zero stay zero
        coef_row[lane] = (float)((a.renorm ? (sum > 0.0 ? my_p / sum : 0.0) : my_p) * (double)a.route_scale);
    }
    if (shared != nullptr && lane == 0) id_row[a.k] = a.shared_id, coef_row[a.k] = sigmoid_f(sl);
}

template <typename T>
void launch(const void *logits, const void *shared, const RouteArgs &a, cudaStream_t st) {
    int gp = 1;
    while (gp < a.G) gp *= 2;
    const int L = 32 / gp, nv = (a.E / a.G + L - 1) / L;
    const unsigned blocks = (unsigned)((a.M + kWarps - 1) / kWarps);
#define SB_ROUTE(NV) router_scored_kernel<T, NV><<<blocks, kWarps * 32, 0, st>>>((const T *)logits, (const T *)shared, a)
    if (nv <= 4) SB_ROUTE(4);
    else if (nv <= 8) SB_ROUTE(8);
    else if (nv <= 16) SB_ROUTE(16);
    else if (nv <= 32) SB_ROUTE(32);
    else SB_ROUTE(64);
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
    if (shared_logit != nullptr) {
        SB_CHECK(shared_ld >= 1, fn, ": shared_ld = ", shared_ld, ", expected >= 1");
        SB_CHECK(shared_id >= 0, fn, ": shared_id = ", shared_id, ", expected >= 0 (its expert row block)");
    }
    SB_CHECK(act_ok(act), fn, ": unsupported activation dtype ", act);
    const int64_t A = k + (shared_logit != nullptr ? 1 : 0), ob = M * A * 4;
    SB_CHECK(apart(ids, ob, coef, ob), fn, ": ids [", (const void *)ids, "] and coef [", (const void *)coef, "] (", ob, " B each) overlap");
    const int64_t lb = ((M - 1) * ld + E) * act_size(act);
    SB_CHECK(apart(ids, ob, logits, lb) && apart(coef, ob, logits, lb), fn, ": ids or coef overlaps the logits [", logits, ", +", lb, " B)");
    RouteArgs a{};
    a.ld = ld, a.M = M, a.E = (int)E, a.k = (int)k, a.score = score, a.G = (int)n_group, a.topk_group = (int)topk_group, a.group_top = (int)group_top;
    a.renorm = renorm != 0, a.route_scale = route_scale, a.bias = bias, a.shared_ld = shared_ld, a.shared_id = shared_id, a.ids = ids, a.coef = coef;
    a.A = (int)A, a.err = err;
    auto st = static_cast<cudaStream_t>(stream);
    if (act == kF32) launch<float>(logits, shared_logit, a, st);
    else launch<uint16_t>(logits, shared_logit, a, st);
    SB_LAUNCH_OK(fn, " ", act_name(act), " M=", M, " E=", E, " k=", k, " groups=", n_group);
    return 0;
}

}  // extern "C"
