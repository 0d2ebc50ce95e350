// The pages of a batch's sequences, a step at a time: sequences are cut, their pages go back onto a stack of free ones, the new
// tokens' pages come from it, and every new token gets its slot and position. With P tokens a page, up(x) = ceil(x / P) and
//     kept = min(length, keep),  back = up(length) - up(kept),  need = up(kept + new) - up(kept),
// the sums of back and need over the sequences before say where a sequence's pages lie on the stack: page i of those given
// back goes to place count + i, page i of those taken comes from place top - 1 - i. A token's page is either one that the
// sequence had, or one of those, so that slots need not wait for the table.
//
// A page that is both given back and taken is read where the table had it, so that the stack is only written before the barrier.
//
// It moves a few bytes a token and page: latencies in a row are all of it. A step of few tokens is one block and one launch: it
// works the sums out in shared memory, one scan for all of them, a token's page is found by bisection of the sums while the
// state is still the old one, and a barrier stands between that and what is written of the new state. A step of many tokens
// takes a cluster of blocks for the pages, each of which works the sums out for itself, and a dependent launch over all SMs for the
// slots, from the new table (in the cluster they took 30000 cycles of eight SMs' instructions for 123099 tokens). Measured on the
// device: 64 sequences of five tokens 4.4 us, 512 of one 6.0 us, 123099 tokens of 96 prompts over 6265 pages 9.1 us (8.1, 8.9
// and 20.4 us by one kernel with a scan for each sum that reads the pages behind the barrier).
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

#include <algorithm>

namespace iq2 {

namespace {

constexpr uint32_t PG_MOST = 1024;                            // threads of a block
constexpr uint32_t PG_CLUSTER = 8, PG_ALONE = 4 * PG_MOST;    // blocks of a large step; tokens that one block takes by itself
constexpr uint32_t PG_SLOTS = 256, PG_TOK = 4;                // threads of a block that writes slots, and tokens of a thread
constexpr uint32_t PG_CAP = INT32_MAX;          // sums stay at this

__device__ __forceinline__ uint32_t capped(uint32_t a, uint32_t b) { return min(a + b, PG_CAP); }

struct Sums {
    uint32_t rows, back, need, keys;  // new tokens, pages given back and taken, tokens after the step
    __device__ __forceinline__ void add(const Sums& o) {
        rows = capped(rows, o.rows), back = capped(back, o.back), need = capped(need, o.need), keys = capped(keys, o.keys);
    }
};
__device__ __forceinline__ Sums shifted_up(const Sums& x, int by) {
    return {__shfl_up_sync(0xFFFFFFFFu, x.rows, by), __shfl_up_sync(0xFFFFFFFFu, x.back, by), __shfl_up_sync(0xFFFFFFFFu, x.need, by),
            __shfl_up_sync(0xFFFFFFFFu, x.keys, by)};
}
__device__ __forceinline__ Sums from_lane(const Sums& x, uint32_t lane) {
    return {__shfl_sync(0xFFFFFFFFu, x.rows, lane), __shfl_sync(0xFFFFFFFFu, x.back, lane), __shfl_sync(0xFFFFFFFFu, x.need, lane),
            __shfl_sync(0xFFFFFFFFu, x.keys, lane)};
}

// The sums over the threads before, and `all` over the block. Called by all threads; `held` is used again at the next call.
__device__ __forceinline__ Sums sum_before(Sums x, Sums (&held)[32], Sums& all) {
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    Sums upto = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const Sums y = shifted_up(upto, o);
        if (lane >= (uint32_t)o) upto.add(y);
    }
    const Sums own = shifted_up(upto, 1);
    __syncthreads();
    if (lane == 31) held[warp] = upto;
    __syncthreads();
    Sums w = lane < warps ? held[lane] : Sums{0, 0, 0, 0};
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const Sums y = shifted_up(w, o);
        if (lane >= (uint32_t)o) w.add(y);
    }
    all = from_lane(w, 31);
    Sums before = from_lane(w, (warp + 31) % 32);
    if (warp == 0) before = {0, 0, 0, 0};
    if (lane != 0) before.add(own);
    return before;
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

// TOKENS: the slots and positions too.
template <bool TOKENS>
__global__ void __launch_bounds__(PG_MOST) pages_kernel(const __grid_constant__ PagesParams p) {
    if (!TOKENS) pdl_launch_dependents();
    extern __shared__ uint32_t smem[];
    __shared__ Sums held[32];
    const uint32_t n = p.seqs;
    // first row of a sequence's tokens, its places among the pages given back and taken, the tokens that it keeps and gets, the
    // tokens of those before it after the step (if all get theirs)
    uint32_t *const row0 = smem, *const back0 = row0 + n + 1, *const need0 = back0 + n + 1, *const kept = need0 + n + 1, *const grow = kept + n, *const key0 = grow + n;
    const uint32_t most = (uint32_t)min((uint64_t)p.width * p.page_size, (uint64_t)INT32_MAX);  // tokens of a sequence
    const uint32_t count = (uint32_t)min(max(__ldcg(p.free_count), 0), (int32_t)p.pages);
    auto up = [&](uint32_t x) { return x == 0 ? 0u : p.by_page.quotient(x - 1) + 1; };
    Sums total{0, 0, 0, 0};  // of the sequences before this turn's
    for (uint32_t b0 = 0; b0 < n; b0 += blockDim.x) {
        const uint32_t b = b0 + threadIdx.x;
        uint32_t len = 0, keep = 0, fresh = 0;
        if (b < n) {
            len = min((uint32_t)max(p.lens[b], 0), most);
            fresh = (uint32_t)max(p.new_lens[b], 0);
            keep = p.keep == nullptr ? len : min(len, (uint32_t)max(p.keep[b], 0));
        }
        bool fits = keep + fresh <= most;
        Sums all, mine{fresh, up(len) - up(keep), fits ? up(keep + fresh) - up(keep) : 0u, fits ? keep + fresh : keep};
        Sums at = sum_before(mine, held, all);
        at.add(total);
        // (all of them fit the rows as a rule: if not, those that do not ask for no pages)
        if (capped(total.rows, all.rows) > p.total) {
            fits = fits && capped(at.rows, fresh) <= p.total;
            Sums fewer;
            const Sums again = sum_before({0, 0, fits ? mine.need : 0u, fits ? keep + fresh : keep}, held, fewer);
            at.need = capped(total.need, again.need), all.need = fewer.need;
            at.keys = capped(total.keys, again.keys), all.keys = fewer.keys;
        }
        if (b < n) {
            row0[b] = min(at.rows, p.total), back0[b] = at.back, need0[b] = at.need;
            kept[b] = keep, grow[b] = fits ? fresh : 0u, key0[b] = at.keys;
        }
        total.add(all);
    }
    if (threadIdx.x == 0) row0[n] = min(total.rows, p.total), back0[n] = total.back, need0[n] = total.need;
    const uint32_t given = min(total.back, p.pages - count), top = count + given, asked = total.need;
    __syncthreads();

    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
    const uint32_t thread = rank * blockDim.x + threadIdx.x, threads = blocks * blockDim.x;
    auto served = [&](uint32_t b) { return need0[b + 1] <= top || need0[b + 1] == need0[b]; };
    auto given_back = [&](uint32_t i) -> const int32_t* {  // where page i of those given back is read
        const uint32_t b = sequence_of(back0, n, i);
        return p.table + ((int64_t)b * p.width + up(kept[b]) + (i - back0[b]));
    };
    // (the other end of the threads than the tokens')
    for (uint32_t i = threads - 1 - thread; i < given; i += threads) p.free_pages[count + i] = *given_back(i);
    if (TOKENS) {
        for (uint32_t t = thread; t < p.total; t += threads) {
            const uint32_t b = t < row0[n] ? sequence_of(row0, n, t) : n;
            int32_t slot = -1, pos = 0;
            if (b < n && grow[b] != 0 && served(b)) {
                const uint32_t at = kept[b] + (t - row0[b]), col = p.by_page.quotient(at), first = up(kept[b]);
                const uint32_t place = top - 1 - (need0[b] + (col - first));  // of a page that is taken
                const int32_t page = *(col < first ? p.table + ((int64_t)b * p.width + col) : place < count ? p.free_pages + place : given_back(place - count));
                pos = (int32_t)at;
                if (page >= 0 && (uint32_t)page < p.pages) slot = (int32_t)((uint32_t)page * p.page_size + (at - col * p.page_size));
            }
            p.slots[t] = slot, p.positions[t] = pos;
        }
    }
    // all of the old state has been read, and the stack is whole
    if (blocks == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");

    // what is taken: the sums up to the last one within the stack
    const uint32_t takes = asked <= top ? asked : need0[sequence_of(need0, n, top)];
    for (uint32_t i = threads - 1 - thread; i < takes; i += threads) {
        const uint32_t b = sequence_of(need0, n, i);
        p.table[(int64_t)b * p.width + up(kept[b]) + (i - need0[b])] = __ldcg(p.free_pages + (top - 1 - i));
    }
    if (rank != 0) return;
    uint32_t keys = 0;
    for (uint32_t b0 = 0; b0 < n; b0 += blockDim.x) {
        const uint32_t b = b0 + threadIdx.x, got = b < n && served(b) ? grow[b] : 0u, len = b < n ? kept[b] + got : 0u;
        uint32_t key = b < n ? key0[b] : 0u;
        if (asked > top) {  // (not all of them got their pages)
            Sums all;
            key = capped(keys, sum_before({0, 0, 0, len}, held, all).keys);
            keys = capped(keys, all.keys);
        }
        if (b < n) p.lens[b] = (int32_t)len, p.granted[b] = (int32_t)got, p.cu_q[b] = (int32_t)row0[b], p.cu_k[b] = (int32_t)key;
    }
    if (threadIdx.x == 0) p.cu_q[n] = (int32_t)row0[n], p.cu_k[n] = (int32_t)(asked > top ? keys : total.keys), *p.free_count = (int32_t)(top - takes);
}

// The sequence of row t < cu[n] by a warp: 32 of the sums at a time.
__device__ __forceinline__ uint32_t sequence_by_warp(const int32_t* cu, uint32_t n, int32_t t) {
    const uint32_t lane = threadIdx.x % 32;
    uint32_t lo = 0, count = n;  // the first b of [lo, lo + count) with cu[b + 1] > t
    while (count > 1) {
        const uint32_t step = (count + 31) / 32, at = lo + min((lane + 1) * step, count);
        const uint32_t above = __ballot_sync(0xFFFFFFFFu, cu[at] > t);
        const uint32_t before = (uint32_t)__ffs(above) - 1;  // (the last one is)
        count = min(step, count - before * step), lo += before * step;
    }
    return lo;
}

// Slots and positions from the state after the step: the last granted[b] of a sequence's tokens are the new ones.
__global__ void __launch_bounds__(PG_SLOTS) slots_kernel(const __grid_constant__ PagesParams p) {
    pdl_wait();
    const uint32_t n = p.seqs, lane = threadIdx.x % 32;
    const uint32_t first = (blockIdx.x * PG_SLOTS + threadIdx.x - lane) * PG_TOK, t0 = first + lane * PG_TOK;  // of the warp; of the thread
    if (first >= p.total) return;
    const int32_t rows = p.cu_q[n];
    int32_t slot[PG_TOK], pos[PG_TOK], page[PG_TOK];
    uint32_t seq[PG_TOK];
    uint32_t lo = n, hi = n;
    if ((int32_t)first < rows) {
        lo = sequence_by_warp(p.cu_q, n, (int32_t)first);
        hi = sequence_by_warp(p.cu_q, n, (int32_t)min(first + 32 * PG_TOK, (uint32_t)rows) - 1);
    }
    while (lo < hi) {  // this thread's first
        const uint32_t mid = (lo + hi) / 2;
        if (p.cu_q[mid + 1] <= (int32_t)t0) lo = mid + 1;
        else hi = mid;
    }
#pragma unroll
    for (uint32_t i = 0; i < PG_TOK; ++i) {
        const int32_t t = (int32_t)(t0 + i);
        while (lo < n && t < rows && t >= p.cu_q[lo + 1]) ++lo;
        const int32_t got = lo < n && t < rows ? p.granted[lo] : 0;
        seq[i] = got > 0 ? lo : n;
        pos[i] = got > 0 ? p.lens[lo] - got + (t - p.cu_q[lo]) : 0;
    }
#pragma unroll
    for (uint32_t i = 0; i < PG_TOK; ++i) page[i] = seq[i] < n ? p.table[(int64_t)seq[i] * p.width + p.by_page.quotient((uint32_t)pos[i])] : -1;
#pragma unroll
    for (uint32_t i = 0; i < PG_TOK; ++i) {
        const uint32_t at = (uint32_t)pos[i];
        slot[i] = page[i] >= 0 && (uint32_t)page[i] < p.pages ? (int32_t)((uint32_t)page[i] * p.page_size + (at - p.by_page.quotient(at) * p.page_size)) : -1;
    }
    const bool vec = (reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions)) % 16 == 0;
    if (vec && t0 + PG_TOK <= p.total) {
        *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < PG_TOK; ++i)
            if (t0 + i < p.total) p.slots[t0 + i] = slot[i], p.positions[t0 + i] = pos[i];
    }
}

template <typename Kernel>
cudaError_t launch_with(Kernel kernel, uint32_t blocks, uint32_t threads, size_t smem, cudaStream_t stream, cudaLaunchAttribute attr, const PagesParams& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_kv_pages_step(const PagesParams& params, cudaStream_t stream) {
    PagesParams p = params;
    p.by_page = Divisor::of(p.page_size);
    const size_t smem = (size_t)(6 * p.seqs + 3) * sizeof(uint32_t);
    const bool alone = p.total <= PG_ALONE;
    const auto kernel = alone ? pages_kernel<true> : pages_kernel<false>;
    if (smem > 32768) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (6 * PAGES_MOST_SEQS + 3) * sizeof(uint32_t));
        if (e != cudaSuccess) return e;
    }
    if (alone) {
        uint32_t threads = 128;
        while (threads < PG_MOST && threads < std::max(p.seqs, p.total)) threads *= 2;
        kernel<<<1, threads, smem, stream>>>(p);
        return cudaGetLastError();
    }
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = PG_CLUSTER, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    const cudaError_t e = launch_with(kernel, PG_CLUSTER, PG_MOST, smem, stream, attr, p);
    if (e != cudaSuccess) return e;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    const uint32_t per = PG_SLOTS * PG_TOK;
    return launch_with(slots_kernel, p.total / per + (p.total % per != 0), PG_SLOTS, 0, stream, attr, p);
}

}  // namespace iq2
