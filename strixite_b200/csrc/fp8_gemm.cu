// Products in 8-bit floating point with a scale per block of 128, dense and for the experts' routed slots, on the tensor cores.
//
//   y[r, n] = sum_kb (xs[r, kb] * ws[n / 128, kb]) * (sum over the 128 k of block kb of xq[r, k] * wq[n, k])
//
// The inner sum of a block is one tcgen05 accumulation (kind::f8f6f4; the products of two e4m3 values are exact and are summed in
// FP32), the outer sum an FP32 FMA of that accumulator, taken from tensor memory, into registers: a scale per 128 columns cannot be
// applied inside the accumulation.
//
// This file: few rows (decode, verify, a few rows an expert). Weight rows are the M axis of the MMA (128 lanes: one block row of scales) and
// the rows of x its N axis, up to TOK = 16 or 32 at a time: a few rows cost a narrow instruction, and an expert's ragged slot list is
// padded to 16. fp8_gemm_wide.cu has the form for many rows. What bounds it is the stream of the weights (60 slots of 512 experts
// [2048, 512], 57 MB: 13 us), and below that the launch and one trip through the ring (6 rows of [2048, 4096]: 4.9 us). Warp roles of a CTA:
//   promotion warps   tcgen05.ld of a finished block accumulator, acc = fma(scale, block, acc); at the end the store of y
//   TMA warp          weight boxes [128 rows x 128 bytes], 128-byte swizzle, and the box of x rows
//   gather warp       rows of x by slot (the experts)
//   MMA warp          four K = 32 instructions per block into one of NBuf accumulators, two commits
//   scale warp        xs * ws of the block for the TOK columns, into the accumulator's slot of shared memory
// CTAs walk the (x tile, weight tile) pairs; where there are fewer pairs than SMs the blocks of K are split over the CTAs of a cluster:
// every CTA pushes its sums into the shared memory of the CTA that owns the column, which adds them in rank order (the same result on
// every run).
// Every mbarrier wait is bounded: on expiry the CTA raises the abort counter, waits for its copies, frees its tensor memory, returns.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "fp8_gemm.cuh"
#include "prefill_umma.cuh"
#include "strixite_b200.h"

namespace {

using namespace sb;
using namespace sb::umma;
using namespace sb::fp8;

__device__ unsigned int g_fp8_aborts = 0;
__device__ unsigned int g_fp8_refusals = 0;

constexpr int kATile = kTileM * kBK;      // 16 KB of weights
constexpr int kPromoWarps = 4, kTmaWarp = 4, kMmaWarp = 5, kScaleWarp = 6, kGatherWarp = 7;
constexpr int kThreads = 8 * 32;
// CTAs that share a pair's K blocks at most. Clusters of 8 CTAs with most of an SM's shared memory did not all start together (16 of them:
// the last ones 4.3 us after the first, measured), clusters of 4 do.
constexpr int kMaxSplit = 4;

template <int TOK>
struct Cfg {
    static_assert(TOK <= 32, "a lane of the scale warp per column");
    static constexpr int BTile = TOK * kBK, StageBytes = kATile + BTile;
    static constexpr int Stages = TOK >= 32 ? 9 : 10;
    static constexpr int NBuf = 8;  // accumulators in tensor memory, and slots of scales
    static constexpr int TmemCols = NBuf * TOK;
    static constexpr int RedBytes = TOK * kTileM * 4;  // the columns' parts from the CTAs of a cluster
};

template <int TOK>
struct Ctl {
    using C = Cfg<TOK>;
    // acc_full: the block's MMAs have completed (a commit) and its scales are there (the scale warp)
    uint64_t full[C::Stages], empty[C::Stages], acc_full[C::NBuf], acc_empty[C::NBuf];
    uint32_t tmem_base;
    int abort_flag;
    alignas(16) float scales[C::NBuf][TOK];  // read as float4
    Buckets buckets;                         // grouped
};

template <int TOK>
constexpr size_t smem_bytes() {
    return (size_t)Cfg<TOK>::Stages * Cfg<TOK>::StageBytes + Cfg<TOK>::RedBytes + sizeof(Ctl<TOK>) + 1024;
}
static_assert(smem_bytes<16>() > kOnePerSm && smem_bytes<32>() > kOnePerSm);

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void st_peer(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// One (x tile, weight tile) pair: its first row of the weight stack, first weight row and block row inside its matrix, and its columns -
// dense: rows first .. first + n of x; grouped: the slots list[first .. first + n).
struct Pair {
    int wrow, n0, ws_row, first, n;
};

template <int TOK, bool GROUPED>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const GemmArgs a) {
    using C = Cfg<TOK>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float *red = reinterpret_cast<float *>(base + C::Stages * C::StageBytes);
    Ctl<TOK> &ctl = *reinterpret_cast<Ctl<TOK> *>(base + C::Stages * C::StageBytes + C::RedBytes);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    let_next_begin();
    if (a.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int rank = a.split > 1 ? (int)cluster_rank() : 0;
    const int sh = a.split == 4 ? 2 : a.split == 2 ? 1 : 0;  // split is 1, 2 or 4
    const int kb0 = a.KB * rank >> sh, kb1 = a.KB * (rank + 1) >> sh;
    volatile int *abort_flag = &ctl.abort_flag;

    // A CTA walks neighbouring pairs: the weight tiles of one x tile, so what belongs to the rows is looked up once. With a split, a cluster
    // has one pair (or none).
    const int cluster = (int)blockIdx.x >> sh, clusters = (int)gridDim.x >> sh;
    auto first_of = [&](int n_pairs) {  // the first n_pairs % clusters walks are one pair longer
        const int each = n_pairs / clusters;
        return each * cluster + min(cluster, n_pairs - each * clusters);
    };
    // Block kb of a pair into stage s: the weights, and (dense) the rows of x.
    auto load = [&](int s, int kb, int wrow, int first, uint32_t bytes) {
        uint8_t *dst = base + s * C::StageBytes;
        mbar_expect_tx(&ctl.full[s], bytes);
        tma_load_2d(dst, &w_map, kb * kBK, wrow, &ctl.full[s]);
        if constexpr (!GROUPED) tma_load_2d(dst + kATile, &x_map, kb * kBK, first, &ctl.full[s]);
    };
    int early = 0;  // dense: blocks of the first pair that are on their way before anything else is set up
    if (warp == kTmaWarp) {
        if (elect_one()) {
            prefetch_map(&w_map), prefetch_map(&x_map);
            for (int i = 0; i < C::Stages; ++i) mbar_init(&ctl.full[i], 1), mbar_init(&ctl.empty[i], 1);
            for (int i = 0; i < C::NBuf; ++i) mbar_init(&ctl.acc_full[i], 2), mbar_init(&ctl.acc_empty[i], kPromoWarps);
            ctl.abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // this thread's copies may signal them at once
            if constexpr (!GROUPED) {
                wait_for_previous();
                const int p = first_of(((a.M + TOK - 1) / TOK) * a.NT), xt = p / a.NT;
                for (int kb = kb0; kb < kb1 && kb - kb0 < C::Stages; ++kb) load(kb - kb0, kb, (p - xt * a.NT) * kTileM, xt * TOK, C::StageBytes);
            }
        }
        if (!GROUPED) early = min(kb1 - kb0, C::Stages);
        __syncwarp();
    } else if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"((uint32_t)C::TmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    wait_for_previous();  // nothing in front of this has read or written global memory (but for the early loads, which waited too)
    RouteTables rt{};
    int x_tiles;
    bool refused = false;
    if constexpr (GROUPED) {
        rt = route_tables(a.group, a.S, a.E);
        BucketScan<TOK, kThreads> scan;
        refused = !scan.load(a.group, rt, a.S, a.E, &g_fp8_refusals);  // the whole grid: no tiles
        x_tiles = scan.scan(a.E, ctl.buckets, [&](int tiles) { return first_of(tiles * a.NT) / a.NT; });
    } else {
        x_tiles = (a.M + TOK - 1) / TOK;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (a.split > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the peers run: their shared memory may be written
    const uint32_t tmem = ctl.tmem_base;
    const int n_pairs = refused ? 0 : x_tiles * a.NT, p_first = first_of(n_pairs), each = n_pairs / clusters, p_end = p_first + each + (cluster < n_pairs - each * clusters ? 1 : 0);

    Pair t{};  // of this thread's walk; warp-uniform
    int xt = -1, nt = 0;
    auto pair_at = [&](int p) {  // for p = p_first, p_first + 1, ..; whether the rows are others than before
        if (xt >= 0 && ++nt < a.NT) {
            t.n0 += kTileM, t.wrow += kTileM, ++t.ws_row;
            return false;
        }
        const bool begin = xt < 0;
        if (begin) xt = p / a.NT, nt = p - xt * a.NT;
        else ++xt, nt = 0;
        t.n0 = nt * kTileM;
        if constexpr (GROUPED) {
            const int e = begin ? ctl.buckets.first : bucket_of(ctl.buckets.prefix, a.E, xt);
            t.first = ctl.buckets.start[e] + (xt - ctl.buckets.prefix[e]) * TOK;
            t.n = min(TOK, ctl.buckets.start[e + 1] - t.first);
            t.wrow = e * a.N + t.n0, t.ws_row = e * a.NB + nt;
        } else {
            t.wrow = t.n0, t.ws_row = nt;
            t.first = xt * TOK, t.n = min(TOK, a.M - t.first);
        }
        return true;
    };
    auto row_of = [&](int j) {  // the row of x behind column j < t.n
        if constexpr (GROUPED) return rt.slots[t.first + j] / a.div;
        else return t.first + j;
    };
    auto put = [&](int j, int r, float v) {  // y of column j, weight row r of the tile
        int64_t row = t.first + j;
        if constexpr (GROUPED) row = rt.slots[row];
        const int64_t o = row * a.N + t.n0 + r;
        if (a.out_f32) static_cast<float *>(a.y)[o] = v;
        else static_cast<uint16_t *>(a.y)[o] = f32_to_bf16_bits(v);
    };

    if (warp == kTmaWarp || (GROUPED && warp == kGatherWarp)) {
        uint32_t it = 0;
        bool ok = true;
        int rows[4] = {0, 0, 0, 0};
        for (int p = p_first; p < p_end && ok; ++p) {
            const bool other = pair_at(p);
            uint32_t bytes = C::StageBytes;
            if constexpr (GROUPED) {
                // columns beyond the list's end repeat its last row; whole quads beyond it are not fetched, and what their columns
                // compute is not stored
                bytes = kATile + (uint32_t)((t.n + 3) / 4) * 4 * kBK;
                if (warp == kGatherWarp && other)
                    for (int j = 0; j < 4; ++j) rows[j] = row_of(min(lane * 4 + j, t.n - 1));
            }
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                if ((int)it < early) continue;
                const int s = it % C::Stages;
                if (it >= C::Stages) ok = __all_sync(0xffffffffu, mbar_wait(&ctl.empty[s], ((it / C::Stages) & 1u) ^ 1u, abort_flag));
                if (!ok) break;
                if (GROUPED && warp == kGatherWarp) {
                    if (lane < TOK / 4 && lane * 4 < t.n)
                        tma_gather4(base + s * C::StageBytes + kATile + lane * 4 * kBK, &x_map, kb * kBK, rows[0], rows[1], rows[2], rows[3], &ctl.full[s]);
                } else if (elect_one()) {
                    load(s, kb, t.wrow, t.first, bytes);
                }
                __syncwarp();
            }
        }
        // The last blocks' MMAs have read their stages and signalled it; after an abandoned wait, the copies in flight have landed.
        for (uint32_t i = it > C::Stages ? it - C::Stages : 0; i < it && ok; ++i) ok = __all_sync(0xffffffffu, mbar_wait(&ctl.empty[i % C::Stages], (i / C::Stages) & 1u, abort_flag));
        if (!ok && lane == 0) {
            for (uint32_t i = it > C::Stages ? it - C::Stages : 0; i < it; ++i)
                for (uint32_t n = 0; n < kSpinLimit && !mbar_try_wait(&ctl.full[i % C::Stages], (i / C::Stages) & 1u); ++n) {
                }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // One thread; the barriers of a block are asked about under the MMAs of the block in front of it (a probe takes ~100 clocks).
        if (elect_one()) {
            uint32_t it = 0;
            bool ok = true, full = false, free = true;
            for (int p = p_first; p < p_end && ok; ++p) {
                pair_at(p);
                const uint32_t idesc = idesc_e4m3(kTileM, (t.n + 15) & ~15);
                for (int kb = kb0; kb < kb1; ++kb) {
                    const int s = it % C::Stages, b = it % C::NBuf;
                    if (!free) ok = mbar_wait(&ctl.acc_empty[b], ((it / C::NBuf) & 1u) ^ 1u, abort_flag);
                    if (ok && !full) ok = mbar_wait(&ctl.full[s], (it / C::Stages) & 1u, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at = smem_u32(base + s * C::StageBytes);
                    const uint64_t da = umma_desc(at), db = umma_desc(at + kATile);
#pragma unroll
                    for (int k = 0; k < kBK / 32; ++k) umma_f8(tmem + b * TOK, da + 2 * k, db + 2 * k, idesc, k != 0);
                    ++it;
                    free = it < C::NBuf || mbar_test(&ctl.acc_empty[it % C::NBuf], ((it / C::NBuf) & 1u) ^ 1u);
                    full = mbar_test(&ctl.full[it % C::Stages], (it / C::Stages) & 1u);
                    umma_commit(&ctl.acc_full[b]);
                    umma_commit(&ctl.empty[s]);
                }
            }
        }
        __syncwarp();
    } else if (warp == kScaleWarp) {
        uint32_t it = 0;
        bool ok = true;
        const float *xp = nullptr;  // lane j: the scales of column j's row; null beyond the columns
        for (int p = p_first; p < p_end && ok; ++p) {
            if (pair_at(p)) xp = lane < t.n ? a.xs + (int64_t)row_of(lane) * a.KB : nullptr;
            // four blocks at a time: a row's four scales share a 32-byte sector, and a round of loads is under way while the round before
            // it is handed over
            float cur[4], nxt[4];
            const float *wp = a.ws + (int64_t)t.ws_row * a.KB;
            auto fetch = [&](float(&to)[4], int kb) {
#pragma unroll
                for (int q = 0; q < 4; ++q) to[q] = kb + q < kb1 && xp != nullptr ? xp[kb + q] * wp[kb + q] : 0.f;
            };
            fetch(cur, kb0);
            for (int kb = kb0; kb < kb1 && ok; kb += 4) {
                fetch(nxt, kb + 4);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (kb + q >= kb1 || !ok) continue;
                    const int b = it % C::NBuf;
                    if (it >= C::NBuf) ok = __all_sync(0xffffffffu, mbar_wait(&ctl.acc_empty[b], ((it / C::NBuf) & 1u) ^ 1u, abort_flag));
                    if (!ok) continue;
                    if (lane < TOK) ctl.scales[b][lane] = cur[q];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl.acc_full[b]);
                    ++it;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) cur[q] = nxt[q];
            }
        }
    } else if (warp < kPromoWarps) {
        constexpr int kChunk = TOK < 32 ? TOK : 32;
        const int r = warp * 32 + lane;
        const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
        uint32_t it = 0;
        bool ok = true;
        for (int p = p_first; p < p_end && ok; ++p) {
            pair_at(p);
            float acc[TOK];
#pragma unroll
            for (int j = 0; j < TOK; ++j) acc[j] = 0.f;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int b = it % C::NBuf;
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl.acc_full[b], (it / C::NBuf) & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < TOK; c += kChunk) {
                    if (c >= t.n) continue;  // warp-uniform
                    uint32_t v[kChunk];
                    if constexpr (kChunk == 32) tmem_ld32(lane_base + b * TOK + c, v);
                    else tmem_ld16(lane_base + b * TOK + c, v);
                    float4 f[kChunk / 4];
#pragma unroll
                    for (int j = 0; j < kChunk / 4; ++j) f[j] = *reinterpret_cast<const float4 *>(&ctl.scales[b][c + 4 * j]);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < kChunk / 4; ++j) {
                        acc[c + 4 * j] = fmaf(f[j].x, __uint_as_float(v[4 * j]), acc[c + 4 * j]);
                        acc[c + 4 * j + 1] = fmaf(f[j].y, __uint_as_float(v[4 * j + 1]), acc[c + 4 * j + 1]);
                        acc[c + 4 * j + 2] = fmaf(f[j].z, __uint_as_float(v[4 * j + 2]), acc[c + 4 * j + 2]);
                        acc[c + 4 * j + 3] = fmaf(f[j].w, __uint_as_float(v[4 * j + 3]), acc[c + 4 * j + 3]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl.acc_empty[b]);
            }
            if (!ok) break;
            if (a.split > 1) {
                // column j belongs to the CTA of rank j % split: part `rank` of its (j / split)-th column
                const uint32_t at = smem_u32(red + rank * kTileM + r);
#pragma unroll
                for (int j = 0; j < TOK; ++j) {
                    if (j >= t.n) continue;
                    uint32_t dst;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(at + (uint32_t)(j & ~(a.split - 1)) * kTileM * 4), "r"(j & (a.split - 1)));
                    st_peer(dst, acc[j]);
                }
            } else if (t.n0 + r < a.N) {
#pragma unroll
                for (int j = 0; j < TOK; ++j)
                    if (j < t.n) put(j, r, acc[j]);
            }
        }
    }

    if (a.split > 1) {  // at most one pair per cluster
        __syncwarp();
        cluster_sync();
        if (warp < kPromoWarps && p_first < p_end) {
            const int r = warp * 32 + lane;
            for (int j = rank; j < t.n; j += a.split) {
                const float *part = red + (j - rank) * kTileM + r;
                float v = part[0] + part[kTileM];
                if (a.split == 4) v = v + part[2 * kTileM] + part[3 * kTileM];
                if (t.n0 + r < a.N) put(j, r, v);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (tid == 0 && ctl.abort_flag) atomicAdd(&g_fp8_aborts, 1u);
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TmemCols) : "memory");
}

}  // namespace

namespace sb {
namespace fp8 {

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static int encoder(const char *fn, EncodeFn *out) {
    static std::mutex mu;
    static EncodeFn cached = nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (cached == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        SB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q), fn, ": looking up the tensor-map encoder");
        SB_CHECK(q == cudaDriverEntryPointSuccess && p != nullptr, fn, ": the driver has no tensor-map encoder");
        cached = reinterpret_cast<EncodeFn>(p);
    }
    *out = cached;
    return 0;
}

// rows x K bytes, boxes of box_rows x 128 bytes (128-byte swizzle); bytes beyond K and rows beyond the end read as zero.
int make_map(const char *fn, CUtensorMap *m, const uint8_t *ptr, int64_t rows, int64_t K, int box_rows) {
    EncodeFn enc;
    SB_TRY(encoder(fn, &enc));
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)K};
    const cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult rc = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    SB_CHECK(rc == CUDA_SUCCESS, fn, ": cuTensorMapEncodeTiled failed with ", (int)rc, " for a [", rows, ", ", K, "] byte matrix");
    return 0;
}

}  // namespace fp8
}  // namespace sb

namespace {

// ---- host ------------------------------------------------------------------------------------------------------------

template <int TOK, bool GROUPED>
int launch(const char *fn, const uint8_t *w, int64_t w_rows, const uint8_t *x, int64_t x_rows, int64_t K, GemmArgs a, int64_t most_tiles, cudaStream_t st) {
    static thread_local int prepared = -1;
    constexpr size_t smem = smem_bytes<TOK>();
    int dev = 0;
    SB_CUDA(cudaGetDevice(&dev), fn);
    if (prepared != dev) {
        SB_CUDA(cudaFuncSetAttribute(fp8_gemm_kernel<TOK, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), fn);
        prepared = dev;
    }
    CUtensorMap wm, xm;
    SB_TRY(make_map(fn, &wm, w, w_rows, K, kTileM));
    SB_TRY(make_map(fn, &xm, x, x_rows, K, GROUPED ? 1 : TOK));
    const int64_t pairs = most_tiles * a.NT, sms = sm_count();
    a.split = 1;
    while (a.split < kMaxSplit && a.split * 2 <= a.KB && pairs * a.split * 2 <= sms) a.split *= 2;
    const dim3 grid((unsigned)(a.split > 1 ? pairs * a.split : std::min(pairs, sms)));
    SB_CUDA((launch_after(fp8_gemm_kernel<TOK, GROUPED>, grid, dim3(kThreads), smem, st, a.split, wm, xm, a)), fn, " (", TOK, " columns, split ", a.split,
            ") N=", a.N, " K=", K);
    return 0;
}

int check_view(const char *fn, const strix_fp8view *w) {
    SB_CHECK(w != nullptr && w->q != nullptr && w->scale != nullptr, fn, ": null weight view, codes or scales");
    SB_CHECK(w->N >= 1 && w->N <= 0x7fffff80 && w->K >= 16 && w->K <= (1 << 24) && w->K % 16 == 0, fn, ": weight [", w->N, ", ", w->K,
             "], expected N 1..2^31-128 and K a multiple of 16 up to 2^24");
    SB_CHECK(aligned16(w->q) && reinterpret_cast<uintptr_t>(w->scale) % 4 == 0, fn, ": weight codes ", (const void *)w->q,
             " must be 16-byte aligned, scales 4-byte");
    return 0;
}

int check_rows(const char *fn, const uint8_t *xq, const float *xs, int64_t rows, int64_t K, const void *y, int64_t y_bytes, int out_act) {
    SB_CHECK(xq != nullptr && xs != nullptr && y != nullptr, fn, ": null pointer (xq=", (const void *)xq, ", xs=", (const void *)xs, ", y=", y, ")");
    SB_CHECK(act_ok(out_act), fn, ": unsupported output dtype ", out_act);
    SB_CHECK(aligned16(xq) && reinterpret_cast<uintptr_t>(xs) % 4 == 0 && reinterpret_cast<uintptr_t>(y) % act_size(out_act) == 0, fn, ": xq ", (const void *)xq,
             " must be 16-byte aligned, xs 4-byte, y ", y, " aligned to its elements");
    SB_CHECK(apart(y, y_bytes, xq, rows * K) && apart(y, y_bytes, xs, rows * fp8_blocks(K) * 4), fn, ": output [", y, ", +", y_bytes,
             " B) overlaps the rows [", (const void *)xq, "] or their scales [", (const void *)xs, "]");
    return 0;
}

// The power of two up to 16 that the byte addresses of all rows of y are multiples of.
int64_t row_start(const void *y, int64_t N, int act) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(y) | (uint64_t)(N * act_size(act)) | 16;
    return (int64_t)(bits & (~bits + 1));
}

int grouped(const char *fn, const uint8_t *xq, const float *xs, const strix_fp8view *w, int64_t E, const void *ws, size_t ws_bytes, int64_t M, int64_t A,
            int64_t rows, void *y, int out_act, cudaStream_t st) {
    SB_TRY(check_view(fn, w));
    SB_CHECK(M >= 1 && A >= 1 && A <= 64 && M <= (1 << 20) && M * A <= (1 << 20), fn, ": M = ", M, ", A = ", A, " (A <= 64, M * A <= 2^20)");
    SB_CHECK(E >= 1 && E <= kMaxE && w->N % E == 0, fn, ": weight has ", w->N, " rows for E = ", E, " experts (E must be 1..1023 and divide the rows)");
    SB_CHECK(ws != nullptr && reinterpret_cast<uintptr_t>(ws) % 4 == 0, fn, ": null or unaligned workspace");
    const size_t need = strix_moe_route_workspace_bytes(M, A, E);
    SB_CHECK(need != 0 && ws_bytes >= need, fn, ": workspace of ", ws_bytes, " bytes, needs ", need, " for M = ", M, ", A = ", A, ", E = ", E);
    const int64_t N = w->N / E, S = M * A;
    SB_TRY(check_rows(fn, xq, xs, rows, w->K, y, S * N * act_size(out_act), out_act));
    SB_CHECK(apart(y, S * N * act_size(out_act), ws, (int64_t)need), fn, ": output overlaps the workspace");
    GemmArgs a{};
    a.xs = xs, a.ws = w->scale, a.group = static_cast<const int32_t *>(ws), a.y = y, a.out_f32 = out_act == kF32;
    a.M = (int)M, a.N = (int)N, a.KB = (int)fp8_blocks(w->K), a.NB = (int)fp8_blocks(N), a.E = (int)E, a.div = (int)(rows == S ? 1 : A), a.S = S;
    a.NT = (int)((N + kTileM - 1) / kTileM);
    // Below 8 slots an expert on average the narrow form, from there on the wide one. Measured (gate/up [1024, 2048] of 64 / 256 experts, us, narrow
    // and wide): mean 4: 22 and 29 / 75 and 83; mean 8: 26 and 31 / 99 and 89; mean 16: 33 and 33 / 142 and 101. Tiles of 32 or 64 slots in the narrow
    // form were never the fastest. The narrow one, too, while it has no more than four (slot tile, weight tile) pairs for three SMs: 43 slots of 5
    // experts [207, 592]: 4.5 and 10.5; 1024 of 8 [256, 512], 144 pairs: 5.9 and 8.1; 1024 of 32 [256, 2048], 192 pairs: 13.0 and 15.2; beyond,
    // 512 of 32 [512, 1024], 256 pairs: 9.3 and 8.7. Up to three for each SM where rows of y start off a 16-byte boundary, which costs the wide
    // form more: 2055 of 8 [281, 128], 408 pairs: 7.6 and 12.3; 2895 of 4 [310, 400], 552 pairs: 13.5 and 11.3.
    const int64_t tiles = std::min(S, E + S / 16);  // at most: every bucket may end in a partial tile
    SB_CHECK(tiles <= 0x7fffffff / a.NT, fn, ": ", S, " slots of N = ", N, " outputs are too many tiles");
    if (S < 8 * E || tiles * a.NT * 3 <= (int64_t)sm_count() * (row_start(y, N, out_act) < 16 ? 9 : 4)) return launch<16, true>(fn, w->q, w->N, xq, rows, w->K, a, tiles, st);
    return wide_grouped(fn, w->q, w->N, xq, rows, w->K, a, st);
}

}  // namespace

namespace sb {

unsigned int fp8_aborts() {
    unsigned int v = 0;
    cudaMemcpyFromSymbol(&v, g_fp8_aborts, sizeof(v));
    return v + fp8::wide_aborts();
}
unsigned int fp8_ws_refusals() {
    unsigned int v = 0;
    cudaMemcpyFromSymbol(&v, g_fp8_refusals, sizeof(v));
    return v + fp8::wide_ws_refusals();
}

}  // namespace sb

extern "C" {

int strix_linear_fp8(const uint8_t *xq, const float *xs, const strix_fp8view *w, void *y, int64_t M, int out_act, void *stream) {
    const char *fn = "linear_fp8";
    SB_TRY(check_view(fn, w));
    SB_CHECK(M >= 1 && M <= 0x7fffff00, fn, ": M = ", M, " rows, expected 1..2^31-256");
    GemmArgs a{};
    a.xs = xs, a.ws = w->scale, a.y = y, a.out_f32 = out_act == kF32;
    a.M = (int)M, a.N = (int)w->N, a.KB = (int)fp8_blocks(w->K), a.NB = (int)fp8_blocks(w->N), a.E = 1, a.div = 1, a.S = M;
    a.NT = (int)((w->N + kTileM - 1) / kTileM);
    auto st = static_cast<cudaStream_t>(stream);
    auto tiles = [&](int64_t tok) { return (M + tok - 1) / tok; };
    SB_CHECK(tiles(16) <= 0x7fffffff / a.NT, fn, ": M = ", M, " rows of N = ", w->N, " outputs are too many tiles");
    SB_TRY(check_rows(fn, xq, xs, M, w->K, y, M * w->N * act_size(out_act), out_act));
    // Tiles of 16 rows while K can be split four ways over the SMs, of 32 while there is an SM for each, else the wide form. Measured
    // ([N, K], M: us with 16 / 32 / wide): [1024, 2048], 64: 5.2 / 5.5 / 11.7, 128: 6.8 / 5.8 / 12.1, 512: 12.9 / 10.3 / 12.5, 1024: 20.9 / 15.9 / 12.7;
    // [4096, 4096], 16: 7.7 / 8.1 / 18.0, 32: 9.6 / 8.9 / 18.5, 128: 20.7 / 14.3 / 19.9, 192: 28.5 / 23.2 / 19.8. Two tiles of
    // 32 for each SM where rows of y start at odd 16-bit elements: [1001, 1024], 1024: 10.9 and 13.8, 1500: 14.8 and 13.9.
    const int64_t sms = sm_count();
    if (tiles(16) * a.NT * 4 <= sms) return launch<16, false>(fn, w->q, w->N, xq, M, w->K, a, tiles(16), st);
    if (tiles(32) * a.NT <= sms * (row_start(y, w->N, out_act) < 4 ? 2 : 1)) return launch<32, false>(fn, w->q, w->N, xq, M, w->K, a, tiles(32), st);
    return wide_dense(fn, w->q, w->N, xq, M, w->K, a, st);
}

int strix_linear_fp8_experts_gather_grouped(const uint8_t *xq, const float *xs, const strix_fp8view *w, int64_t E, const void *ws, size_t ws_bytes,
                                            int64_t M, int64_t A, void *y, int out_act, void *stream) {
    return grouped("linear_fp8_experts_gather_grouped", xq, xs, w, E, ws, ws_bytes, M, A, M, y, out_act, static_cast<cudaStream_t>(stream));
}

int strix_linear_fp8_experts_combine_grouped(const uint8_t *hq, const float *hs, const strix_fp8view *w, int64_t E, const int32_t *ids, const float *coef,
                                             const void *ws, size_t ws_bytes, float *partial, int64_t M, int64_t A, void *y, int act, void *stream) {
    const char *fn = "linear_fp8_experts_combine_grouped";
    SB_CHECK(ids != nullptr && coef != nullptr && y != nullptr, fn, ": null pointer (ids=", (const void *)ids, ", coef=", (const void *)coef, ", y=", y, ")");
    SB_CHECK(reinterpret_cast<uintptr_t>(ids) % 4 == 0 && reinterpret_cast<uintptr_t>(coef) % 4 == 0, fn, ": ids ", (const void *)ids, " and coef ",
             (const void *)coef, " must be 4-byte aligned");
    SB_CHECK(act_ok(act), fn, ": unsupported activation dtype ", act);
    SB_CHECK(reinterpret_cast<uintptr_t>(y) % act_size(act) == 0, fn, ": y ", y, " must be aligned to its elements");
    SB_CHECK(M >= 1 && A >= 1 && A <= 64 && M <= (1 << 20) && M * A <= (1 << 20), fn, ": M = ", M, ", A = ", A, " (A <= 64, M * A <= 2^20)");
    SB_TRY(check_view(fn, w));
    SB_CHECK(E >= 1 && E <= kMaxE && w->N % E == 0, fn, ": weight has ", w->N, " rows for E = ", E, " experts (E must be 1..1023 and divide the rows)");
    const int64_t N = w->N / E, yb = M * N * act_size(act), pb = M * A * N * 4;
    SB_CHECK(partial != nullptr && apart(y, yb, partial, pb), fn, ": null partial, or it overlaps y");
    SB_CHECK(apart(y, yb, ids, M * A * 4) && apart(y, yb, coef, M * A * 4) && apart(partial, pb, ids, M * A * 4) && apart(partial, pb, coef, M * A * 4), fn,
             ": y or partial overlaps ids or coef");
    SB_CHECK(ws == nullptr || apart(y, yb, ws, (int64_t)ws_bytes), fn, ": y overlaps the workspace");
    SB_CHECK(hq == nullptr || hs == nullptr || (apart(y, yb, hq, M * A * w->K) && apart(y, yb, hs, M * A * fp8_blocks(w->K) * 4)), fn,
             ": y overlaps the rows or their scales");
    auto st = static_cast<cudaStream_t>(stream);
    SB_TRY(grouped(fn, hq, hs, w, E, ws, ws_bytes, M, A, M * A, partial, kF32, st));
    return sb::combine_reduce(fn, partial, ids, coef, M, A, E, N, y, act, st, nullptr, false, static_cast<const int32_t *>(ws));
}

}  // extern "C"
