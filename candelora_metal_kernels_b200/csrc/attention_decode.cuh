// What the kernels of the decode attention share (attention_decode.cu for 16-bit and int8 caches, attention_decode_int4.cu for
// 4-bit ones): the line of work and its parts, and the kernel that joins the parts of an item.
#pragma once

#include "attention_internal.h"
#include "iq2xxs_common.cuh"

#include <algorithm>

namespace iq2 {

namespace {

constexpr int AD_HEADS = 8;  // query heads of an item
// Units' time that starting and ending an item costs. Measured with 1 / 2 / 3: 128 x 4096 tokens 219 / 216 / 214 us,
// 1 x 100001 49.7 / 48.6 / 47.9 us.
constexpr uint32_t AD_ITEM_COST = 3;
constexpr uint32_t AD_I4_UNIT = 32;  // tokens that the line of work is cut at for 4-bit caches: a warp's tile
// Measured with 0 / 1 / 2 / 4: 128 x 4096 tokens 94.7 / 92.9 / 93.7 / 95.3 us, 1 x 333 11.4 / 9.4 / 10.8 / 11.2 us.
constexpr uint32_t AD_I4_ITEM_COST = 1;
constexpr int AD_I4_WARPS = 12;  // of a block for 4-bit caches, each with a part of its own
constexpr float LOG2E = 1.44269504f;

// What join_kernel's block of the same number has to join: the parts of blocks c0 to c1 of one item, block c0's being its
// part number `slot` (0: its first, 1: its last), the others' their first. c1 = 0: nothing.
struct JoinRecord {
    uint32_t b, item, c0, c1, slot;
};
inline size_t records_bytes(uint32_t blocks) { return (blocks * sizeof(JoinRecord) + 255) / 256 * 256; }

struct DecodeArgs {
    DecodeParams p;
    float* parts;
    JoinRecord* records;
    double inv_blocks;                      // 1 / the blocks of the launch
    uint32_t chunks_of_heads;
    Divisor by_page;                        // tokens of a page
    bool q_vec;                             // rows of q start on 16-byte boundaries
    bool block_an_item;                     // (4-bit caches) not the line of work, but a block for each item
};

inline DecodeArgs decode_args(const DecodeParams& p, void* workspace, int num_sms) {
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    return {p, reinterpret_cast<float*>(ws + records_bytes(num_sms)), reinterpret_cast<JoinRecord*>(ws), 1.0 / num_sms,
            (p.q_heads / p.c.heads + AD_HEADS - 1) / AD_HEADS, Divisor::of(p.c.page_size),
            reinterpret_cast<uintptr_t>(p.q.p) % 16 == 0 && p.q.token_stride * (p.dtype == kF32 ? 4 : 2) % 16 == 0 &&
                p.q.head_stride * (p.dtype == kF32 ? 4 : 2) % 16 == 0,
            false};
}

__host__ __device__ __forceinline__ uint32_t seq_len(const DecodeParams& p, uint32_t b) {
    const uint64_t most = min((uint64_t)p.table_width * p.c.page_size, (uint64_t)0x7FFFFFFF);
#ifdef __CUDA_ARCH__
    const int32_t len = __ldg(p.seq_lens + b);
#else
    const int32_t len = p.seq_lens[b];
#endif
    return (uint32_t)min((uint64_t)max(len, 0), most);
}

__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
    if (dtype == kF32) return static_cast<const float*>(p)[i];
    if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_elem(void* p, int64_t i, int dtype, float x) {
    if (dtype == kF32) static_cast<float*>(p)[i] = x;
    else if (dtype == kF16) static_cast<__half*>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    uint32_t r;
    if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
template <bool BF>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
    if (BF) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 2^x of an integer x in -126..127, its logarithm, and one over it.
__device__ __forceinline__ float power_of_two(float x) { return __uint_as_float((uint32_t)((int)x + 127) << 23); }
__device__ __forceinline__ float log2_of_power(float x) { return (float)((int)(__float_as_uint(x) >> 23) - 127); }
__device__ __forceinline__ float over_power(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// ---- values with row scales (int8 and 4-bit caches) ----
// Next to the largest score, held as a whole number m, a token has p = 2^(x - m), and l is the sum of these whatever the values
// are. What f16 pieces are taken of, and o with it, is w = p |value scale| 2^level, a head's own power of two f that makes the largest
// of them 2^7 to 2^8. m and f do as a rule, and move where a w, or a sum of p, has grown past AD_SCALED_LAZY.
constexpr float AD_SCALED_TOP = 7.f, AD_SCALED_LAZY = 32768.f;
constexpr float AD_MOST = 112.f;  // the highest level: p times it stays below 2^127
struct Moved {
    float m, f, keep, keep_o;  // and what l and o are taken times
    bool moved;
    // most: the largest x of the tokens to come, weighed: the largest x + log2 |value scale|.
    static __device__ __forceinline__ Moved from(float m, float f, float most, float weighed) {
        // (the level never makes o larger than it is; nothing yet: `up` is infinite)
        const float next = fmaxf(m, ceilf(most)), level = log2_of_power(f), up = next - m;
        const float to = fmaxf(fminf(fminf(ceilf(AD_SCALED_TOP - (weighed - next)), level + up), AD_MOST), -126.f);
        const bool none = m == -INFINITY;
        return {next, power_of_two(to), none ? 0.f : exp2_approx(-up), none ? 0.f : exp2_approx(to - level - up), next > m || to != level};
    }
};
// (o, m, l) as others add it up: the level goes, or values of any size would not meet in one sum. l = 2^k l' with l' in [2^-13, 2^-12),
// so that 24 of these in each of 148 parts add up to less than 1; o' = o / 2^(level + k), about the output times l'; and m + k.
struct Leveled {
    float k, l, down, off;  // o' = o * down * off
    // unit: what o is held by.
    static __device__ __forceinline__ Leveled of(float l, float f, float unit) {
        constexpr uint32_t NORM = 13;
        const uint32_t e = min(max(__float_as_uint(l) >> 23, 100u), 240u);
        const float down = __uint_as_float((254u - NORM - e) << 23);
        return {(float)e - (127.f - NORM), l * down, down * unit, over_power(f)};
    }
};

// The line of work from one unit on: the item it is in and the tokens [t0, t1) of that item in the part. The line's units are UNIT
// tokens; an item's first COST units have no tokens, and a part that ends inside them has none (the next part has the item).
// EVEN: parts differ by a unit at most, of one unit at least, so that none is empty but behind the line's end (the parts of an item
// follow one another); otherwise all but the last ones are of the same length, rounded up. What deals the work is callable on the
// host too, for tests without a GPU.
template <uint32_t UNIT, uint32_t COST, bool EVEN>
struct Cursor {
    uint64_t unit, end;
    uint32_t b, item, len, units;  // the sequence, its item (key head, group of query heads), tokens and units an item
    uint32_t k, n;                 // first unit of the item in the part, and how many
    uint32_t t0, t1;
    __host__ __device__ __forceinline__ void cut() {
        n = (uint32_t)min((uint64_t)(units - k), end - unit);
        t0 = (max(k, COST) - COST) * UNIT, t1 = min((max(k + n, COST) - COST) * UNIT, len);
    }
    static __host__ __device__ __forceinline__ uint32_t units_of(uint32_t len_) { return len_ == 0 ? 0 : (len_ + UNIT - 1) / UNIT + COST; }
    __host__ __device__ __forceinline__ bool done() const { return unit >= end; }
    __host__ __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == len; }
    __host__ __device__ __forceinline__ void next(const DecodeParams& p, uint32_t items) {
        unit += n;
        k = 0;
        if (done()) return;
        if (++item == items) {
            item = 0;
            do {
                if (++b >= p.batch) {  // (not reached while the lengths stay as they were)
                    unit = end;
                    return;
                }
                len = seq_len(p, b);
            } while (len == 0);
            units = units_of(len);
        }
        cut();
        if (t0 == t1) unit = end;
    }

    // Where the parts of the line begin: EVEN at multiples of a fraction, rounded down, the same for whoever asks.
    struct Parts {
        uint64_t units, each;  // of the line; of a part
        uint32_t parts;
        double share;          // units / parts
        __host__ __device__ __forceinline__ uint64_t begin(uint32_t part) const {
            if (EVEN) return part >= parts ? units : min((uint64_t)(part * share), units);
            return min(part * each, units);
        }
        static __host__ __device__ __forceinline__ Parts of(uint64_t units, uint32_t parts, double inv_parts) {
            Parts line{units, 0, parts, EVEN ? max((double)units * inv_parts, 1.0) : (double)units * inv_parts};
            if (!EVEN) {
                line.each = (uint64_t)line.share;  // units / parts, rounded up
                while (line.each * parts < units) ++line.each;
            }
            return line;
        }
    };
    // The part [u0, u1) of the line, which begins in sequence b_ of len_ tokens and own units an item, `before` units into the line.
    static __host__ __device__ __forceinline__ Cursor at(uint64_t u0, uint64_t u1, uint32_t b_, uint32_t len_, uint32_t own, uint64_t before) {
        Cursor cur{};
        cur.b = b_, cur.len = len_, cur.units = own;
        const uint32_t rest = (uint32_t)(u0 - before);
        cur.item = rest / own, cur.k = rest % own;
        cur.unit = u0, cur.end = u1;
        cur.cut();
        return cur;
    }
    // Whether the item is the first one of the block whose first unit is u0: its part of it is the block's number 0, others number 1.
    __host__ __device__ __forceinline__ bool first_of(uint64_t u0) const { return unit - k <= u0; }
    // Part `part` of `parts` as a cursor (done at once where there is nothing). A warp works it out by itself, from the lengths.
    // Sequences of length 0 get their zeros here, a part a sequence, from the `threads` threads that take the part.
    static __device__ __forceinline__ Cursor of_part(const DecodeArgs& a, uint32_t part, uint32_t parts, double inv_parts, uint32_t thread,
                                                     uint32_t threads, Parts& line) {
        const DecodeParams& p = a.p;
        const uint32_t lane = threadIdx.x % 32, d = p.c.d, items = p.c.heads * a.chunks_of_heads;
        uint64_t units = 0;
        uint32_t len = 0;  // of sequence b0 + lane
#pragma unroll 1
        for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
            const uint32_t b = b0 + lane;
            len = b < p.batch ? seq_len(p, b) : 0u;
            units += units_of(len);
            // sequences of length 0: zeros, a part a sequence
            uint32_t empty = __ballot_sync(0xFFFFFFFFu, len == 0 && b < p.batch && b % parts == part);
#pragma unroll 1
            for (; empty != 0; empty &= empty - 1)
#pragma unroll 1
                for (uint32_t i = thread; i < p.q_heads * d; i += threads)
                    store_elem(p.out, (int64_t)(b0 + __ffs(empty) - 1) * p.q_heads * d + i, p.dtype, 0.f);
        }
#pragma unroll
        for (int o = 16; o > 0; o /= 2) units += __shfl_xor_sync(0xFFFFFFFFu, units, o);
        units *= items;
        line = Parts::of(units, parts, inv_parts);
        const uint64_t u0 = line.begin(part), u1 = line.begin(part + 1);
        Cursor cur{};
        if (u0 < u1) {
            uint64_t before = 0;  // units of the sequences before
#pragma unroll 1
            for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
                if (p.batch > 32) len = b0 + lane < p.batch ? seq_len(p, b0 + lane) : 0u;
                const uint32_t own = units_of(len);
                uint64_t upto = (uint64_t)own * items;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                    if (lane >= (uint32_t)o) upto += x;
                }
                const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + upto > u0);
                if (hit != 0) {
                    const int lane_of = __ffs(hit) - 1;
                    cur = at(u0, u1, b0 + lane_of, __shfl_sync(0xFFFFFFFFu, len, lane_of), __shfl_sync(0xFFFFFFFFu, own, lane_of),
                             before + __shfl_sync(0xFFFFFFFFu, upto - (uint64_t)own * items, lane_of));
                    break;
                }
                before += __shfl_sync(0xFFFFFFFFu, upto, 31);
            }
        }
        return cur;
    }

    // What block `block` has to join, whose part, `per_block` ones of the line from `part` on, begins with this cursor.
    __host__ __device__ __forceinline__ JoinRecord record(const Parts& line, uint32_t block, uint32_t part, uint32_t per_block) const {
        // the first block whose part begins inside an item's tokens joins it: the block before it has the first of them
        JoinRecord r{b, item, block - 1, 0, 0};
        if (t0 == 0) return r;
        const uint64_t unit0 = unit - k, before = line.begin(part - per_block);
        if (before <= unit0 + COST) {
            r.c1 = block, r.slot = before >= unit0 ? 0 : 1;
            while (line.begin((r.c1 + 1) * per_block) < unit0 + units) ++r.c1;
        }
        return r;
    }
};

constexpr int AD_JOIN_THREADS = AD_HEADS * 32;

// The parts of an item that several blocks had: (o, m, l) = sum over them of 2^(m_c - max) (o_c, l_c), in the blocks'
// order. A block a record, a warp a head.
template <int DP>
__global__ void __launch_bounds__(AD_JOIN_THREADS, 1)
    join_kernel(const __grid_constant__ DecodeArgs a) {
    const DecodeParams& p = a.p;
    const uint32_t chunks_of_heads = a.chunks_of_heads;
    constexpr int PART = AD_HEADS * (DP + 2);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_wait();
    const JoinRecord r = a.records[blockIdx.x];
    if (r.c1 == 0) return;
    const uint32_t d = p.c.d, group = p.q_heads / p.c.heads;
    const uint32_t kv_head = r.item / chunks_of_heads, head0 = kv_head * group + (r.item % chunks_of_heads) * AD_HEADS;
    if (warp >= min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0)) return;
    auto slot = [&](uint32_t c) { return a.parts + ((uint64_t)c * 2 + (c == r.c0 ? r.slot : 0)) * PART; };
    float y[DP / 32] = {}, sum = 0.f, mx = -INFINITY;
    // lanes hold the maxima and sums of 32 parts; the parts' o are added with their weights
    for (uint32_t c1 = r.c0; c1 <= r.c1; c1 += 32) {
        const uint32_t n = min(r.c1 + 1 - c1, 32u);
        const float m = lane < n ? slot(c1 + lane)[AD_HEADS * DP + warp] : -INFINITY;
        const float l = lane < n ? slot(c1 + lane)[AD_HEADS * DP + AD_HEADS + warp] : 0.f;
        float top = fmaxf(m, mx);
        for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const float keep = top == -INFINITY ? 0.f : exp2_approx(mx - top), w = top == -INFINITY ? 0.f : exp2_approx(m - top);
        mx = top;
        float add = w * l;
        for (int o = 16; o > 0; o /= 2) add += __shfl_xor_sync(0xFFFFFFFFu, add, o);
        sum = sum * keep + add;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) y[i] *= keep;
#pragma unroll 8
        for (uint32_t c = 0; c < n; ++c) {
            const float* const o = slot(c1 + c) + warp * DP + lane;
            const float wc = __shfl_sync(0xFFFFFFFFu, w, c);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) y[i] += o[i * 32] * wc;
        }
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
        if (lane + i * 32 < d)
            store_elem(p.out, ((int64_t)r.b * p.q_heads + head0 + warp) * d + lane + i * 32, p.dtype, sum == 0.f ? 0.f : y[i] / sum);
}

// join_kernel on `blocks` blocks, as the dependent of the kernel launched before it.
template <int DP>
cudaError_t launch_join(const DecodeArgs& a, uint32_t blocks, cudaStream_t stream) {
    // (it keeps the first one's split of shared memory: changing it would drain the SMs twice a call)
    const cudaError_t e = cudaFuncSetAttribute(join_kernel<DP>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(AD_JOIN_THREADS);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<DP>, a);
}

}  // namespace

}  // namespace iq2
