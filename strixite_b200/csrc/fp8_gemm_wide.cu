// The FP8 products for many rows: y[r, n] = sum_kb (xs[r, kb] * ws[n / 128, kb]) * (block sum of xq * wq), as in fp8_gemm.cu, with the rows
// of x on the accumulator's lanes and 256 weight rows as its columns.
//
// A thread that takes block sums out of tensor memory holds ONE row of x and 128 columns that share a weight block, so the scale of a
// whole block is one number per thread: the promotion is one packed FMA for two columns and nothing else. (With weight rows on the lanes
// each column has its own scale: a shared-memory load for four columns, and a warp that prepares them; at 4096^3 that took 162 us.)
//
// GROUP = 2 (dense): a cluster of two CTAs works on 256 rows x 256 columns with cta_group::2 instructions. Each CTA loads its 128 rows of
// x and half of the weight rows, 32 KB a block of K instead of 48: the feed from L2 (about 58 bytes a clock and SM, measured) is what
// bounds the one-CTA form. SPLIT: two such pairs share the K blocks of a tile, and each adds up one half of the columns (few tiles, long
// K: the chain of one tile's blocks is the time). GROUP = 1 (the experts' slots, gathered by row): an expert has seldom more than 128
// rows.
//
// Roles: warps 0-3 / 4-7 promote column half 0 / 1 (each half has two accumulators, so the tensor cores run up to three half blocks
// ahead), warp 8 issues TMA, warps 9 and 10 the MMAs of half 0 and 1 (those of CTA 0 for both CTAs), warps 11-13 gather rows of x. The
// sums leave through a 64-byte-wide staging strip per warp so that a store covers whole sectors of a row.
//
// Measured at the full clock (1965 MHz): 16384 x 4096 x 4096 245 us, 2.24 PFLOP/s, tensor pipe 61 % active; 4096 tokens x 10 of 512 experts
// [1024, 2048] 243 us, 4.9 TB/s. Called again and again for more than ~0.1 s both bring the GPU to its power limit: at 1425 to 1475 MHz 287 us
// (1.92 PFLOP/s) and, with the grouping, 308 us for 262.
// What bounds both is the chain of a block: its MMAs' commit, the promotion, the accumulator's release, ~750 clocks for 512 of MMA with
// tensor memory full (the grouped feed alone takes 181 to 190 us).
// Every mbarrier wait is bounded: on expiry the CTA raises the abort counter, waits for its copies, frees its tensor memory, returns.
#include <algorithm>

#include "fp8_gemm.cuh"

namespace {

using namespace sb;
using namespace sb::fp8;

__device__ unsigned int g_wide_aborts = 0;
__device__ unsigned int g_wide_refusals = 0;

constexpr int kRows = 128;               // rows of x per CTA = accumulator lanes
constexpr int kColTile = 256;            // weight rows per tile
constexpr int kHalf = 128;               // columns of a promotion warpgroup: one block row of weight scales
constexpr int kPromoWarps = 8;
constexpr int kTmaWarp = 8, kMmaWarp = 9, kGatherWarp = 11;  // two MMA warps
constexpr int kStripPitch = 80;          // 64 bytes of a row + 16: rows start in different banks
constexpr int kStrip = 32 * kStripPitch;

// Two warpgroups promote, one (grouped: two, for the gathers) does the rest. Registers move to the former, a thread of which holds 128
// sums: 2 * 128 * 208 + 128 * 64 <= 3 * 128 * 168 and 2 * 128 * 208 + 2 * 128 * 48 = 4 * 128 * 128, what the block is launched with.
template <bool GROUPED>
constexpr int kThreads = (GROUPED ? 16 : 12) * 32;
constexpr int kGatherWarps = 3;

template <int GROUP>
struct Cfg {
    static constexpr int ATile = kRows * kBK, BTile = kColTile / GROUP * kBK;  // per CTA and block of K
    static constexpr int StageBytes = ATile + BTile;
    static constexpr int Stages = GROUP == 2 ? 6 : 4;
};

template <int GROUP>
struct Ctl {
    uint64_t full[Cfg<GROUP>::Stages], empty[Cfg<GROUP>::Stages], acc_full[2][2], acc_empty[2][2];  // [half][buffer]
    uint32_t tmem_base;
    int abort_flag;
    Buckets buckets;  // grouped
};

template <int GROUP>
constexpr size_t smem_bytes() {
    return (size_t)Cfg<GROUP>::Stages * Cfg<GROUP>::StageBytes + kPromoWarps * kStrip + sizeof(Ctl<GROUP>) + 1024;
}
static_assert(smem_bytes<1>() > kOnePerSm && smem_bytes<2>() > kOnePerSm);

template <int GROUP>
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    if constexpr (GROUP == 1) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}
// Arrival on `bar` of this CTA (GROUP 1) or of both CTAs (GROUP 2; their bits in the cluster) when the MMAs issued so far have completed.
template <int GROUP>
__device__ __forceinline__ void commit(uint64_t *bar, uint16_t ctas) {
    if constexpr (GROUP == 1) umma_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(ctas)
                     : "memory");
}
// A box into this CTA's shared memory, counted on the barrier at cluster address `bar` (the leader's).
__device__ __forceinline__ void tma_load_pair(void *dst, const void *tmap, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// An arrival on a barrier of the pair. What it hands over is tensor memory, ordered by the tcgen05 fence in front of it; a release at
// cluster scope would wait for the scale loads in flight as well (1700 clocks a block of K, measured).
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// (a.x, a.y) += (s, s) * (v0, v1): one instruction, each lane of it an FP32 FMA.
__device__ __forceinline__ void fma2(float2 &a, float s, uint32_t v0, uint32_t v1) {
    asm("{\n\t.reg .b64 x, y, z;\n\t"
        "mov.b64 x, {%2, %2};\n\t"
        "mov.b64 y, {%3, %4};\n\t"
        "mov.b64 z, {%0, %1};\n\t"
        "fma.rn.f32x2 z, x, y, z;\n\t"
        "mov.b64 {%0, %1}, z;\n\t}"
        : "+f"(a.x), "+f"(a.y)
        : "f"(s), "r"(v0), "r"(v1));
}
// A tile: its first row of the weight stack, first weight row and block row inside its matrix, halves with weight rows in them, and this
// CTA's rows - dense: rows first .. of x; grouped: the slots list[first .. first + n).
struct Tile {
    int wrow, n0, ws_row, halves, first, n;
};

template <int GROUP, bool GROUPED, bool SPLIT>
__global__ void __launch_bounds__(kThreads<GROUPED>, 1)
    fp8_wide_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const GemmArgs a) {
    using C = Cfg<GROUP>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *strips = base + C::Stages * C::StageBytes;
    Ctl<GROUP> &ctl = *reinterpret_cast<Ctl<GROUP> *>(strips + kPromoWarps * kStrip);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    let_next_begin();
    if (warp == kTmaWarp && elect_one()) prefetch_map(&w_map), prefetch_map(&x_map);
    const uint32_t in_cluster = GROUP == 2 ? cluster_rank() : 0, rank = in_cluster & 1u, leader = in_cluster & ~1u;  // a pair is ranks 2i, 2i + 1
    constexpr int kCtas = GROUP * (SPLIT ? 2 : 1);  // that share a tile
    const int part = SPLIT ? (int)in_cluster >> 1 : 0, kb0 = SPLIT ? a.KB * part / 2 : 0, kb1 = SPLIT ? a.KB * (part + 1) / 2 : a.KB;
    const uint16_t both_ctas = (uint16_t)(3u << leader);
    if (tid == 0) {
        for (int i = 0; i < C::Stages; ++i) mbar_init(&ctl.full[i], 1), mbar_init(&ctl.empty[i], 2);  // empty: both halves' MMAs
        for (int i = 0; i < 4; ++i) mbar_init(&ctl.acc_full[i / 2][i % 2], 1), mbar_init(&ctl.acc_empty[i / 2][i % 2], 4 * GROUP);
        ctl.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        if constexpr (GROUP == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    wait_for_previous();  // nothing in front of this has read or written global memory
    RouteTables rt{};
    int x_tiles;
    bool refused = false;
    if constexpr (GROUPED) {
        rt = route_tables(a.group, a.S, a.E);
        BucketScan<kRows, kThreads<GROUPED>> scan;
        refused = !scan.load(a.group, rt, a.S, a.E, &g_wide_refusals);  // the whole grid: no tiles
        x_tiles = scan.scan(a.E, ctl.buckets, [&](int) { return (int)blockIdx.x / a.NT; });
    } else {
        x_tiles = (a.M + kRows * GROUP - 1) / (kRows * GROUP);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (GROUP == 2) cluster_sync();  // both CTAs' barriers exist before either is signalled
    tc_fence_after();
    const uint32_t tmem = ctl.tmem_base;
    volatile int *abort_flag = &ctl.abort_flag;
    const int n_tiles = refused ? 0 : x_tiles * a.NT, step = gridDim.x / kCtas;

    auto tile_of = [&](int p) {  // warp-uniform
        const int xt = p / a.NT, nt = p - xt * a.NT;
        Tile t;
        t.n0 = nt * kColTile;
        t.halves = a.N - t.n0 > kHalf ? 2 : 1;
        if constexpr (GROUPED) {
            const int e = p == (int)blockIdx.x ? ctl.buckets.first : bucket_of(ctl.buckets.prefix, a.E, xt);
            t.first = ctl.buckets.start[e] + (xt - ctl.buckets.prefix[e]) * kRows;
            t.n = min(kRows, ctl.buckets.start[e + 1] - t.first);
            t.wrow = e * a.N + t.n0, t.ws_row = e * a.NB + nt * 2;
        } else {
            t.first = (xt * GROUP + (int)rank) * kRows;
            t.n = min(kRows, a.M - t.first);  // may be negative: the pair's second CTA beyond the end
            t.wrow = t.n0, t.ws_row = nt * 2;
        }
        return t;
    };

    if (warp >= kPromoWarps) {
        if constexpr (GROUPED) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == kTmaWarp || (GROUPED && warp >= kGatherWarp && warp < kGatherWarp + kGatherWarps)) {
        // One warp for the boxes; grouped, three more for the rows of x: a gather of four rows is an instruction of its own, ~50 clocks
        // of its thread's warp each (4096 tokens x 10 of 512 experts: 298 us with one gathering warp, 257 with two).
        const int quad = (warp - kGatherWarp) + kGatherWarps * lane;  // gathering: rows 4 * quad .. of the tile
        uint32_t it = 0;
        bool ok = true;
        for (int p = blockIdx.x / kCtas; p < n_tiles && ok; p += step) {
            const Tile t = tile_of(p);
            int rows[4] = {0, 0, 0, 0};
            uint32_t bytes = (uint32_t)C::StageBytes * GROUP;
            int quads = 0;
            if constexpr (GROUPED) {
                // Rows beyond the list's end repeat its last one; whole quads beyond it are not fetched, but for the first of every
                // gathering warp: a warp without a part in a block could fall a round of the ring behind and wait for a phase long over.
                // What the lanes of such rows compute is not stored.
                quads = max((t.n + 3) / 4, kGatherWarps);
                bytes = C::BTile + (uint32_t)quads * 4 * kBK;
                if (warp >= kGatherWarp)
                    for (int j = 0; j < 4; ++j) rows[j] = rt.slots[t.first + min(quad * 4 + j, t.n - 1)] / a.div;
            }
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % C::Stages;
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl.empty[s], ((it / C::Stages) & 1u) ^ 1u, abort_flag));
                if (!ok) break;
                uint8_t *dst = base + s * C::StageBytes;
                if (GROUPED && warp >= kGatherWarp) {
                    if (quad < quads) tma_gather4(dst + quad * 4 * kBK, &x_map, kb * kBK, rows[0], rows[1], rows[2], rows[3], &ctl.full[s]);
                } else if (elect_one()) {
                    if constexpr (GROUP == 2) {
                        // the leader's barrier counts both CTAs' bytes; this CTA's weight rows are the rank-th 64 of each half, so that a
                        // half's instruction (64 rows from each CTA) covers 128 neighbouring rows
                        if (rank == 0) mbar_expect_tx(&ctl.full[s], bytes);
                        const uint32_t bar = peer_addr(&ctl.full[s], leader);
                        tma_load_pair(dst, &x_map, kb * kBK, t.first, bar);
                        tma_load_pair(dst + C::ATile, &w_map, kb * kBK, t.wrow + (int)rank * 64, bar);
                        tma_load_pair(dst + C::ATile + 64 * kBK, &w_map, kb * kBK, t.wrow + kHalf + (int)rank * 64, bar);
                    } else {
                        mbar_expect_tx(&ctl.full[s], bytes);
                        tma_load_2d(dst + C::ATile, &w_map, kb * kBK, t.wrow, &ctl.full[s]);
                        if constexpr (!GROUPED) tma_load_2d(dst, &x_map, kb * kBK, t.first, &ctl.full[s]);
                    }
                }
                __syncwarp();
            }
        }
        // The last blocks' MMAs have read their stages and signalled it; after an abandoned wait, the copies in flight have landed.
        for (uint32_t i = it > C::Stages ? it - C::Stages : 0; i < it && ok; ++i) ok = __all_sync(0xffffffffu, mbar_wait(&ctl.empty[i % C::Stages], (i / C::Stages) & 1u, abort_flag));
        if (!ok && lane == 0 && rank == 0) {
            for (uint32_t i = it > C::Stages ? it - C::Stages : 0; i < it; ++i)
                for (uint32_t n = 0; n < kSpinLimit && !mbar_try_wait(&ctl.full[i % C::Stages], (i / C::Stages) & 1u); ++n) {
                }
        }
        __syncwarp();
    } else if ((warp == kMmaWarp || warp == kMmaWarp + 1) && rank == 0) {
        // One thread per half: a half whose accumulators are still being read does not hold up the other. A probe of a barrier takes ~100
        // clocks to answer even when the phase is over (measured), so the two that a block of K needs are asked under the MMAs of the
        // block in front of it; only one that was not over then is waited for.
        if (elect_one()) {
            const int h = warp - kMmaWarp;
            const uint32_t idesc = idesc_e4m3(kRows * GROUP, kHalf);
            uint32_t it = 0, done = 0;
            bool ok = true, full = false, free = true;  // fresh accumulators are free
            for (int p = blockIdx.x / kCtas; p < n_tiles && ok; p += step) {
                const Tile t = tile_of(p);
                for (int kb = kb0; kb < kb1; ++kb) {
                    const int s = it % C::Stages;
                    if (!full) ok = mbar_wait(&ctl.full[s], (it / C::Stages) & 1u, abort_flag);
                    if (!ok) break;
                    ++it;
                    if (h < t.halves) {
                        const uint32_t b = done & 1u;
                        if (!free) ok = mbar_wait(&ctl.acc_empty[h][b], ((done >> 1) & 1u) ^ 1u, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t at = smem_u32(base + s * C::StageBytes);
                        const uint64_t da = umma_desc(at), db = umma_desc(at + C::ATile + h * (C::BTile / 2));
#pragma unroll
                        for (int k = 0; k < kBK / 32; ++k) umma_f8<GROUP>(tmem + (b * 2 + h) * kHalf, da + 2 * k, db + 2 * k, idesc, k != 0);
                        ++done;
                        free = mbar_test(&ctl.acc_empty[h][done & 1u], ((done >> 1) & 1u) ^ 1u);
                        full = mbar_test(&ctl.full[it % C::Stages], (it / C::Stages) & 1u);
                        commit<GROUP>(&ctl.acc_full[h][b], both_ctas);
                        commit<GROUP>(&ctl.empty[s], both_ctas);
                    } else {
                        full = false;
                        commit<GROUP>(&ctl.empty[s], both_ctas);  // nothing of this half reads the stage
                    }
                }
            }
        }
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int h = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + h * kHalf;
        uint8_t *strip = strips + warp * kStrip;
        const uint32_t empty_at = peer_addr(&ctl.acc_empty[0][0], leader);
        uint32_t done = 0;
        bool ok = true, met = false;
        // What a tile starts with - its rows and first scales, up to three dependent loads - is fetched before the store of the tile in
        // front of it.
        Tile t{};
        int64_t row = 0;            // of y
        const float *xp = nullptr;  // this thread's scales: null beyond the rows
        const float *wp = nullptr;
        float sx[2] = {0.f, 0.f}, sw[2] = {0.f, 0.f};  // of the next two blocks
        auto fetch = [&](int p) {
            if (p >= n_tiles) return;
            t = tile_of(p);
            if (h >= t.halves) return;
            row = t.first + r, xp = nullptr;
            if (r < t.n) {
                int64_t from = row;
                if constexpr (GROUPED) {
                    row = rt.slots[row];
                    from = (int)row / a.div;
                }
                xp = a.xs + from * a.KB;
            }
            wp = a.ws + (int64_t)(t.ws_row + h) * a.KB;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (kb0 + i < kb1) sx[i] = xp != nullptr ? xp[kb0 + i] : 0.f, sw[i] = wp[kb0 + i];
        };
        fetch(blockIdx.x / kCtas);
        for (int p = blockIdx.x / kCtas; p < n_tiles; p += step) {
            if (h >= t.halves) {
                fetch(p + step);
                continue;
            }
            float2 acc[kHalf / 2];
#pragma unroll
            for (int j = 0; j < kHalf / 2; ++j) acc[j] = make_float2(0.f, 0.f);
            // A quarter of the columns is loaded while the one in front of it is added; the last quarter of a block is added under the
            // first load of the next block, whose barrier was asked about a quarter earlier.
            uint32_t v0[32], v1[32];
            auto add = [&](const uint32_t(&v)[32], int quarter, float s) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) fma2(acc[quarter * 16 + j / 2], s, v[j], v[j + 1]);
            };
            ok = __all_sync(0xffffffffu, mbar_wait(&ctl.acc_full[h][done & 1u], (done >> 1) & 1u, abort_flag));
            if (!ok) break;
            tc_fence_after();
            tmem_ld32(lanes + (done & 1u) * 2 * kHalf, v0);
            for (int kb = kb0; kb < kb1; ++kb) {
                const float s = sx[0] * sw[0];
                sx[0] = sx[1], sw[0] = sw[1];
                if (kb + 2 < kb1) sx[1] = xp != nullptr ? xp[kb + 2] : 0.f, sw[1] = wp[kb + 2];
                const uint32_t b = done & 1u, from = lanes + b * 2 * kHalf;
                ++done;
                tmem_ld_wait();
                tmem_ld32(from + 32, v1);
                add(v0, 0, s);
                tmem_ld_wait();
                tmem_ld32(from + 64, v0);
                add(v1, 1, s);
                tmem_ld_wait();
                tmem_ld32(from + 96, v1);
                const bool more = kb + 1 < kb1, ready = more && mbar_test(&ctl.acc_full[h][done & 1u], (done >> 1) & 1u);
                add(v0, 2, s);
                tmem_ld_wait();  // everything is in registers: the accumulator is free
                tc_fence_before();
                __syncwarp();
                if (elect_one()) {
                    if constexpr (GROUP == 2) arrive_at(empty_at + (h * 2 + b) * 8);
                    else mbar_arrive(&ctl.acc_empty[h][b]);
                }
                if (more) {
                    if (!__all_sync(0xffffffffu, ready)) ok = __all_sync(0xffffffffu, mbar_wait(&ctl.acc_full[h][done & 1u], (done >> 1) & 1u, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    tmem_ld32(lanes + (done & 1u) * 2 * kHalf, v0);
                }
                add(v1, 3, s);
            }
            if (!ok) break;
            if constexpr (SPLIT) {
                // Half h of the columns belongs to the pair of part h. The other pair's sums come into the ring, which both are done with.
                cluster_sync();
                met = true;
                float4 *sums = reinterpret_cast<float4 *>(base) + r;  // [kHalf / 4][kRows]
                if (h != part) {
                    const uint32_t to = peer_addr(sums, in_cluster ^ 2u);
#pragma unroll
                    for (int j = 0; j < kHalf / 4; ++j)
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + j * kRows * 16), "f"(acc[2 * j].x), "f"(acc[2 * j].y), "f"(acc[2 * j + 1].x),
                                     "f"(acc[2 * j + 1].y)
                                     : "memory");
                }
                cluster_sync();
                if (h != part) continue;
#pragma unroll
                for (int j = 0; j < kHalf / 4; ++j) {
                    const float4 o = sums[j * kRows];
                    acc[2 * j].x += o.x, acc[2 * j].y += o.y, acc[2 * j + 1].x += o.z, acc[2 * j + 1].y += o.w;
                }
            }
            const int n_rows = t.n, n_base = t.n0 + h * kHalf;
            const int64_t out_row = row;
            fetch(p + step);
            const int live_rows = min(32, n_rows - (warp & 3) * 32);  // of this warp
            if (live_rows <= 0) continue;
            // y: 64 bytes of every row at a time through the strip; then 4 lanes write a row's 64 bytes, 8 rows an instruction
            const int es = a.out_f32 ? 4 : 2;
            const uint64_t at = reinterpret_cast<uint64_t>(a.y) | (uint64_t)a.N * es;  // what every row's start is a multiple of
            const int unit = at % 16 == 0 ? 16 : at % 4 == 0 ? 4 : 2;
            auto flush = [&](int col) {  // the strip's 64 / es columns from col on
                __syncwarp();
                if (unit == 16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = i * 8 + (lane >> 2), n = n_base + col + (lane & 3) * (16 / es);
                        const int64_t orow = __shfl_sync(0xffffffffu, out_row, rr);
                        const bool live = rr < live_rows;
                        const uint4 q = *reinterpret_cast<const uint4 *>(strip + rr * kStripPitch + (lane & 3) * 16);
                        uint8_t *dst = static_cast<uint8_t *>(a.y) + (orow * a.N + n) * es;
                        if (live && n < a.N) *reinterpret_cast<uint4 *>(dst) = q;
                    }
                } else {
                    // rows that start anywhere: neighbouring lanes write neighbouring words (16 a row, two rows an instruction) or halves.
                    // 2293 x 656 against 2112 (vectors), 2116 (words), 2115 (halves) rows: 13.2, 18.5, 26.5 us; each lane its own row: 43 us.
                    const int per = 64 / unit, mine = lane & (per - 1), n = n_base + col + mine * unit / es, times = unit == 4 ? (live_rows + 1) / 2 : live_rows;
                    const uint8_t *src = strip + mine * unit;
                    uint8_t *dst = static_cast<uint8_t *>(a.y) + (int64_t)n * es;
                    for (int i = 0; i < times; i += 4) {
                        uint8_t *to[4];
                        uint32_t v[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int rr = unit == 4 ? (i + q) * 2 + (lane >> 4) : i + q;
                            to[q] = dst + __shfl_sync(0xffffffffu, out_row, rr) * a.N * es;
                            if (rr >= live_rows || n >= a.N) to[q] = nullptr;
                            v[q] = unit == 4 ? *reinterpret_cast<const uint32_t *>(src + rr * kStripPitch) : *reinterpret_cast<const uint16_t *>(src + rr * kStripPitch);
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if (to[q] == nullptr) continue;
                            if (unit == 4) *reinterpret_cast<uint32_t *>(to[q]) = v[q];
                            else *reinterpret_cast<uint16_t *>(to[q]) = (uint16_t)v[q];
                        }
                    }
                }
                __syncwarp();
            };
            uint4 *mine = reinterpret_cast<uint4 *>(strip + lane * kStripPitch);
            if (a.out_f32) {
#pragma unroll
                for (int c = 0; c < kHalf; c += 16) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 u = acc[c / 2 + 2 * j], v = acc[c / 2 + 2 * j + 1];
                        mine[j] = make_uint4(__float_as_uint(u.x), __float_as_uint(u.y), __float_as_uint(v.x), __float_as_uint(v.y));
                    }
                    flush(c);
                }
            } else {
#pragma unroll
                for (int c = 0; c < kHalf; c += 32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 *v = &acc[c / 2 + 4 * j];
                        mine[j] = make_uint4(bf16x2(v[0].x, v[0].y), bf16x2(v[1].x, v[1].y), bf16x2(v[2].x, v[2].y), bf16x2(v[3].x, v[3].y));
                    }
                    flush(c);
                }
            }
        }
        if (SPLIT && !met) cluster_sync(), cluster_sync();  // a half without columns, or an abandoned wait
    }

    __syncwarp();
    if (SPLIT && warp >= kPromoWarps) cluster_sync(), cluster_sync();  // the ring is free (the TMA warp has waited); the sums are across
    tc_fence_before();
    if constexpr (GROUP == 2) cluster_sync();  // nobody's barriers or shared memory go while the peer signals or reads them
    __syncthreads();
    tc_fence_after();
    if (tid == 0 && ctl.abort_flag) atomicAdd(&g_wide_aborts, 1u);
    if (warp == kMmaWarp) {
        if constexpr (GROUP == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int GROUP, bool GROUPED, bool SPLIT>
int launch(const char *fn, const uint8_t *w, int64_t w_rows, const uint8_t *x, int64_t x_rows, int64_t K, GemmArgs a, int64_t tiles, cudaStream_t st) {
    static thread_local int prepared = -1;
    constexpr size_t smem = smem_bytes<GROUP>();
    int dev = 0;
    SB_CUDA(cudaGetDevice(&dev), fn);
    if (prepared != dev) {
        SB_CUDA(cudaFuncSetAttribute(fp8_wide_kernel<GROUP, GROUPED, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), fn);
        prepared = dev;
    }
    CUtensorMap wm, xm;
    SB_TRY(make_map(fn, &wm, w, w_rows, K, GROUP == 2 ? 64 : kColTile));
    SB_TRY(make_map(fn, &xm, x, x_rows, K, GROUPED ? 1 : kRows));
    a.NT = (a.N + kColTile - 1) / kColTile;
    const int64_t all = tiles * a.NT;
    constexpr int kCtas = GROUP * (SPLIT ? 2 : 1);
    const int64_t clusters = SPLIT ? all : std::min(all, (int64_t)sm_count() / GROUP);  // split: one tile each
    SB_CUDA((launch_after(fp8_wide_kernel<GROUP, GROUPED, SPLIT>, dim3((unsigned)(clusters * kCtas)), dim3(kThreads<GROUPED>), smem, st, kCtas, wm, xm, a)), fn,
            " (wide) N=", a.N, " K=", K);
    return 0;
}

}  // namespace

namespace sb {
namespace fp8 {

int wide_dense(const char *fn, const uint8_t *w, int64_t w_rows, const uint8_t *x, int64_t x_rows, int64_t K, const GemmArgs &a, cudaStream_t st) {
    const int64_t tiles = ((int64_t)a.M + 2 * kRows - 1) / (2 * kRows);
    // K over two pairs where that many clusters of four run at once (33 on 148 SMs: 34 of them took twice the time of 33; the rule stops at 32)
    // and K is long enough to pay for bringing the sums together: [4096, 7168], 256 rows 27.1 -> 19.2 us; [4096, 4096], 512: 18.5 -> 15.5;
    // [4096, 1024], 400: 9.0 -> 10.1. The sides meet between 12 and 18 blocks of K (without -> with, 12 / 16 / 18 / 20 blocks: [4096, K], 512
    // rows 10.3 -> 11.0 / 11.9 -> 11.9 / 12.5 -> 12.3 / 13.5 -> 12.8; [8192, K], 256: 10.3 -> 11.0 / 12.2 -> 12.1 / 12.8 -> 12.5 / 13.6 -> 12.9).
    if (a.KB >= 20 && tiles * ((a.N + kColTile - 1) / kColTile) * 9 <= sm_count() * 2) return launch<2, false, true>(fn, w, w_rows, x, x_rows, K, a, tiles, st);
    return launch<2, false, false>(fn, w, w_rows, x, x_rows, K, a, tiles, st);
}

int wide_grouped(const char *fn, const uint8_t *w, int64_t w_rows, const uint8_t *x, int64_t x_rows, int64_t K, const GemmArgs &a, cudaStream_t st) {
    return launch<1, true, false>(fn, w, w_rows, x, x_rows, K, a, std::min(a.S, a.E + a.S / kRows), st);
}

unsigned int wide_aborts() {
    unsigned int v = 0;
    cudaMemcpyFromSymbol(&v, g_wide_aborts, sizeof(v));
    return v;
}
unsigned int wide_ws_refusals() {
    unsigned int v = 0;
    cudaMemcpyFromSymbol(&v, g_wide_refusals, sizeof(v));
    return v;
}

}  // namespace fp8
}  // namespace sb
