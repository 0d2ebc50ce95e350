// The pages of a batch's sequences, a step at a time: sequences are cut, their pages go back onto a stack of free ones, the new
// tokens' pages come from it, and every new token gets its slot and position. With P tokens a page, up(x) = ceil(x / P) and
//     kept = min(length, keep),  back = up(length) - up(kept),  need = up(kept + new) - up(kept),
// the sums of back and need over the sequences before say where a sequence's pages lie on the stack: page i of those given
// back goes to place count + i, page i of those taken comes from place top - 1 - i. A token's page is either one that the
// sequence had, or one of those, so that slots need not wait for the table.
//
// It moves a few bytes a token and page: latencies in a row are all of it. One cluster of blocks does the whole step in one launch:
// each block works the sums out for itself in shared memory, and the cluster's barrier stands between what is read of the old
// state and what is written of the new. Tokens and pages find their sequence by bisection of the sums.
#include "attention_internal.h"

#include <algorithm>

namespace iq2 {

namespace {

constexpr int PG_THREADS = 1024, PG_WARPS = PG_THREADS / 32;
constexpr uint32_t PG_CLUSTER = 8;  // blocks of a large step

// The sum of x over the threads before, and `all` over the block. Called by all threads; `held` is used again at the next call.
__device__ __forceinline__ uint64_t sum_before(uint64_t x, uint64_t (&held)[PG_WARPS], uint64_t& all) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    uint64_t upto = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= (uint32_t)o) upto += y;
    }
    __syncthreads();
    if (lane == 31) held[warp] = upto;
    __syncthreads();
    uint64_t w = held[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint64_t y = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= (uint32_t)o) w += y;
    }
    all = __shfl_sync(0xFFFFFFFFu, w, 31);
    const uint64_t warps = __shfl_sync(0xFFFFFFFFu, w, (warp + 31) % 32);
    return upto - x + (warp == 0 ? 0 : warps);
}

// The last b of sums[0 .. n] (ascending, sums[0] = 0) with sums[b] <= x and b < n: the sequence that x falls to.
__device__ __forceinline__ uint32_t sequence_of(const uint32_t* sums, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;  // the first b with sums[b + 1] > x
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (sums[mid + 1] <= x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PG_THREADS) pages_kernel(const __grid_constant__ PagesParams p) {
    extern __shared__ uint32_t smem[];
    __shared__ uint64_t held[PG_WARPS];
    const uint32_t n = p.seqs;
    // first row of a sequence's tokens, its places among the pages given back and taken (at most 2^31 - 1), the tokens that it
    // keeps and gets
    uint32_t *const row0 = smem, *const back0 = row0 + n + 1, *const need0 = back0 + n + 1, *const kept = need0 + n + 1, *const grow = kept + n;
    const uint64_t most = min((uint64_t)p.width * p.page_size, (uint64_t)INT32_MAX);  // tokens of a sequence
    auto up = [&](uint32_t x) { return x == 0 ? 0u : p.by_page.quotient(x - 1) + 1; };
    auto small = [](uint64_t x) { return (uint32_t)min(x, (uint64_t)INT32_MAX); };
    uint64_t rows = 0, backs = 0, needs = 0;  // of the sequences before this turn's
    for (uint32_t b0 = 0; b0 < n; b0 += PG_THREADS) {
        const uint32_t b = b0 + threadIdx.x;
        uint32_t len = 0, keep = 0, fresh = 0;
        if (b < n) {
            len = (uint32_t)min((uint64_t)max(p.lens[b], 0), most);
            keep = p.keep == nullptr ? len : min(len, (uint32_t)max(p.keep[b], 0));
            fresh = (uint32_t)max(p.new_lens[b], 0);
        }
        uint64_t all_rows, all_backs, all_needs;
        const uint64_t row = rows + sum_before(fresh, held, all_rows);
        const uint64_t back = backs + sum_before(up(len) - up(keep), held, all_backs);
        const bool fits = row + fresh <= p.total && (uint64_t)keep + fresh <= most;
        const uint64_t need = needs + sum_before(fits ? up(keep + fresh) - up(keep) : 0u, held, all_needs);
        rows += all_rows, backs += all_backs, needs += all_needs;
        if (b < n) {
            row0[b] = (uint32_t)min(row, (uint64_t)p.total), back0[b] = small(back), need0[b] = small(need);
            kept[b] = keep, grow[b] = fits ? fresh : 0u;
        }
    }
    if (threadIdx.x == 0) row0[n] = (uint32_t)min(rows, (uint64_t)p.total), back0[n] = small(backs), need0[n] = small(needs);
    const uint32_t count = (uint32_t)min(max(*p.free_count, 0), (int32_t)p.pages);
    const uint32_t given = min(small(backs), p.pages - count), top = count + given;
    __syncthreads();

    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const uint32_t thread = rank * PG_THREADS + threadIdx.x, threads = blocks * PG_THREADS;
    for (uint32_t i = thread; i < given; i += threads) {
        const uint32_t b = sequence_of(back0, n, i);
        p.free_pages[count + i] = p.table[(int64_t)b * p.width + up(kept[b]) + (i - back0[b])];
    }
    // all of the old state has been read, and the stack is whole
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");

    auto served = [&](uint32_t b) { return need0[b + 1] <= top || need0[b + 1] == need0[b]; };
    auto taken = [&](uint32_t i) { return __ldcg(p.free_pages + (top - 1 - i)); };
    const uint32_t asked = need0[n];
    // what is taken: the sums up to the last one within the stack
    const uint32_t takes = asked <= top ? asked : need0[sequence_of(need0, n, top)];
    for (uint32_t i = thread; i < takes; i += threads) {
        const uint32_t b = sequence_of(need0, n, i);
        p.table[(int64_t)b * p.width + up(kept[b]) + (i - need0[b])] = taken(i);
    }
    for (uint32_t t = thread; t < p.total; t += threads) {
        const uint32_t b = t < row0[n] ? sequence_of(row0, n, t) : n;
        int32_t slot = -1, pos = 0;
        if (b < n && grow[b] != 0 && served(b)) {
            pos = (int32_t)(kept[b] + (t - row0[b]));
            const uint32_t col = p.by_page.quotient((uint32_t)pos), first = up(kept[b]);
            const int32_t page = col < first ? p.table[(int64_t)b * p.width + col] : taken(need0[b] + (col - first));
            if (page >= 0 && (uint32_t)page < p.pages) slot = (int32_t)((uint32_t)page * p.page_size + ((uint32_t)pos - col * p.page_size));
        }
        p.slots[t] = slot, p.positions[t] = pos;
    }
    if (rank != 0) return;
    uint64_t keys = 0;
    for (uint32_t b0 = 0; b0 < n; b0 += PG_THREADS) {
        const uint32_t b = b0 + threadIdx.x, got = b < n && served(b) ? grow[b] : 0u, len = b < n ? kept[b] + got : 0u;
        uint64_t all;
        const uint64_t key = keys + sum_before(len, held, all);
        keys += all;
        if (b < n) p.lens[b] = (int32_t)len, p.granted[b] = (int32_t)got, p.cu_q[b] = (int32_t)row0[b], p.cu_k[b] = (int32_t)small(key);
    }
    if (threadIdx.x == 0) p.cu_q[n] = (int32_t)row0[n], p.cu_k[n] = (int32_t)small(keys), *p.free_count = (int32_t)(top - takes);
}

}  // namespace

cudaError_t launch_kv_pages_step(const PagesParams& params, cudaStream_t stream) {
    PagesParams p = params;
    p.by_page = Divisor::of(p.page_size);
    const size_t smem = (size_t)(5 * p.seqs + 3) * sizeof(uint32_t);
    cudaError_t e = cudaFuncSetAttribute(pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * PAGES_MOST_SEQS + 3) * sizeof(uint32_t));
    if (e != cudaSuccess) return e;
    const uint32_t blocks = p.total > 2 * PG_THREADS ? PG_CLUSTER : 1;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(PG_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, pages_kernel, p);
}

}  // namespace iq2
