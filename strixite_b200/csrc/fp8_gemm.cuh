// Shared by the two forms of the FP8 products: narrow (fp8_gemm.cu: weight rows on the accumulator's lanes, up to 32 rows of x as its
// columns - decode, few rows an expert) and wide (fp8_gemm_wide.cu: rows of x on the lanes, 256 weight rows as columns).
#pragma once

#include <cuda.h>

#include "fp8.cuh"
#include "grouped.cuh"
#include "umma.cuh"

namespace sb {
namespace fp8 {

constexpr int kBK = 128;  // K per stage: one scale block, one 128-byte swizzle row
constexpr int kMaxE = 1023;
// More shared memory than this and an SM holds one block of these kernels at a time. That is a condition, not only a consequence: they
// let the next kernel begin before they have their tensor memory, and a block of that one must not hold it while it waits for them.
constexpr size_t kOnePerSm = 114 * 1024;

struct GemmArgs {
    const float *xs, *ws;    // scales of x rows [.., KB] and of the weight blocks [(E *) NB, KB]
    const int32_t *group;    // grouped: the workspace of moe_group_routes
    void *y;
    int out_f32;
    int M, N, KB, NB;        // dense: rows of x; rows of one matrix, blocks of K, block rows of one matrix
    int E, div;              // grouped: slot s reads row s / div
    int64_t S;
    int NT, split;           // weight tiles of one matrix; CTAs that share a tile's K blocks (narrow)
};

// rows x K bytes, boxes of box_rows x 128 bytes (128-byte swizzle); bytes beyond K and rows beyond the end read as zero.
int make_map(const char *fn, CUtensorMap *m, const uint8_t *ptr, int64_t rows, int64_t K, int box_rows);

// The wide form (fp8_gemm_wide.cu). x_tiles: tiles of x rows at most (grouped: known on the device only).
int wide_dense(const char *fn, const uint8_t *w, int64_t w_rows, const uint8_t *x, int64_t x_rows, int64_t K, const GemmArgs &a, cudaStream_t st);
int wide_grouped(const char *fn, const uint8_t *w, int64_t w_rows, const uint8_t *x, int64_t x_rows, int64_t K, const GemmArgs &a, cudaStream_t st);
unsigned int wide_aborts();
unsigned int wide_ws_refusals();

#ifdef __CUDACC__
using namespace umma;

// kind::f8f6f4: D = F32 (bits 4-5 = 1), A and B e4m3 (0), both K-major.
__device__ __forceinline__ uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
// Four rows r0..r3 of a tensor map whose box is one row of 128 bytes, to four consecutive 128-byte rows of shared memory.
__device__ __forceinline__ void tma_gather4(void *dst, const void *tmap, int x, int r0, int r1, int r2, int r3, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
        : "memory");
}
// One thread of a converged warp. The tensor instructions take their operands from uniform registers: under an elected branch the
// compiler knows that one thread is active, under `lane == 0` it does not and serialises every operand (measured on 4096^3: 215 us
// with lane == 0, 162 us with elect).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
// Whether a phase is over, without waiting (mbar_try_wait may suspend the thread for a while).
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared-memory object in the CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}

// What a grouped kernel knows of the buckets, in shared memory.
struct Buckets {
    int warp_tot[32];
    int first;              // the bucket of this block's first tile
    int prefix[kMaxE + 2];  // first tile of each bucket; [E]: their number
    int start[kMaxE + 2];   // first position of each bucket in the slot list
};

// Cuts the buckets of a grouping workspace into tiles of TILE slots; all THREADS threads of the block. The offsets are read together
// with the header that says whether the workspace is for these sizes (they lie inside it either way), so their latencies overlap.
template <int TILE, int THREADS>
struct BucketScan {
    static constexpr int kPer = (kMaxE + THREADS) / THREADS;  // neighbouring buckets of a thread
    int off[kPer + 1];
    __device__ __forceinline__ bool load(const int32_t *ws, const RouteTables &rt, int64_t S, int E, unsigned int *refusals) {
#pragma unroll
        for (int i = 0; i <= kPer; ++i) off[i] = rt.offsets[min((int)threadIdx.x * kPer + i, E)];
        return ws_is_for(ws, S, E, refusals);
    }
    // Returns the number of tiles. `first_tile` (of that number) says which tile's bucket goes to b.first. The caller's next
    // __syncthreads() makes all of it visible.
    template <typename F>
    __device__ __forceinline__ int scan(int E, Buckets &b, F first_tile) const {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        int nt[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) nt[i] = (off[i + 1] - off[i] + TILE - 1) / TILE, sum += nt[i];
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) b.warp_tot[warp] = incl;
        __syncthreads();
        int before = incl - sum, total = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) {
            const int v = b.warp_tot[i];
            before += i < warp ? v : 0;
            total += v;
        }
        const int mine = first_tile(total);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = tid * kPer + i;
            if (e <= E) b.prefix[e] = before, b.start[e] = off[i];
            if (before <= mine && mine < before + nt[i]) b.first = e;
            before += nt[i];
        }
        return total;
    }
};
// The bucket of tile t: prefix[b] <= t < prefix[b + 1].
__device__ __forceinline__ int bucket_of(const int *prefix, int E, int t) {
    int lo = 0, hi = E;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *m) { asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory"); }
#endif

}  // namespace fp8
}  // namespace sb
