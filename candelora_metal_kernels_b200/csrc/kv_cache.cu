// The paged key-value cache: the write of new tokens (with the rotation of q and k, and the quantisation of an int8
// cache) and the read of cached tokens back into packed tensors. Both move each byte once and are bound by HBM.
//
// Rotation, for the pair (a, b) = (x[i], x[i + d/2]) ("half") or (x[2i], x[2i + 1]) (interleaved):
//     a' = a c - b s,  b' = b c + a s,  c = cos[position][i], s = sin[position][i],
// with every product and sum rounded by itself in f32, so that a result does not depend on how the compiler fuses.
// int8 rows (one token and head): m = max |x|, scale = m / 127, code = rint(x * (127 / m)); m < 2^-100 gives zeros (the
// quotient would overflow), and a row with an infinity or NaN gets a NaN scale, so that it reads back as NaN.
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

#include <algorithm>

namespace iq2 {

namespace {

constexpr int KW_THREADS = 256;

constexpr float MIN_AMAX = 7.88860905e-31f;  // 2^-100

// Four values at element i. ONCE: they are not read again (the cache lines give way first).
template <bool ONCE>
__device__ __forceinline__ float4 load4(const void* base, int64_t i, int dtype, bool vec) {
    if (dtype == kF32) {
        const float* p = static_cast<const float*>(base) + i;
        if (vec) return ONCE ? __ldcs(reinterpret_cast<const float4*>(p)) : __ldg(reinterpret_cast<const float4*>(p));
        return make_float4(p[0], p[1], p[2], p[3]);
    }
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
    uint32_t lo, hi;
    if (vec) {
        const uint2 w = ONCE ? __ldcs(reinterpret_cast<const uint2*>(p)) : __ldg(reinterpret_cast<const uint2*>(p));
        lo = w.x, hi = w.y;
    } else {
        lo = p[0] | ((uint32_t)p[1] << 16), hi = p[2] | ((uint32_t)p[3] << 16);
    }
    if (dtype == kF16) {
        const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__uint_as_float(lo << 16), __uint_as_float(lo & 0xFFFF0000u), __uint_as_float(hi << 16),
                       __uint_as_float(hi & 0xFFFF0000u));
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int dtype) {
    if (dtype == kF16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Four values at element i of a 16-byte aligned tensor (i a multiple of 4).
__device__ __forceinline__ void store4(void* base, int64_t i, int dtype, float4 x) {
    if (dtype == kF32) *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = x;
    else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + i) =
            make_uint2(pack16(x.x, x.y, dtype), pack16(x.z, x.w, dtype));
}

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)), y = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x, b = y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ uint32_t codes4(float4 x, float inv) {
    // 1.5 * 2^23 more rounds |x inv| <= 127 to the nearest integer (ties to even) and leaves it in the low byte
    auto code = [&](float y) { return __float_as_uint(__fadd_rn(__fmul_rn(y, inv), 12582912.0f)); };
    return prmt(prmt(code(x.x), code(x.y), 0x0040u), prmt(code(x.z), code(x.w), 0x0040u), 0x5410u);
}

// LANES threads (a power of two >= d / 8) take a row: lane l holds elements 4l..4l+3 of each half, so that a pair of either
// rotation is in one thread and a row's maximum takes log2(LANES) shuffles. Rows are (token, head) with the heads of q, then
// k, then v. A
// thread has one row (two or three in flight: 2048 tokens 16.5 / 18.5 against 14.5 us); instructions bind next to HBM, so
// that divisions are products and codes are rounded by an addition.
template <int LANES>
__global__ void __launch_bounds__(KW_THREADS) kv_write_kernel(const __grid_constant__ KvWriteParams p, uint32_t token0, uint32_t rows) {
    const uint32_t lane = threadIdx.x % LANES, r = blockIdx.x * (KW_THREADS / LANES) + threadIdx.x / LANES;
    const uint32_t heads = p.q_heads + 2 * p.c.heads, half = p.c.d / 2;
    const bool live = r < rows, active = live && lane * 8 < p.c.d;
    const uint32_t in_launch = p.by_heads.quotient(r), t = token0 + in_launch, head = r - in_launch * heads;
    const bool is_q = head < p.q_heads, is_v = head >= p.q_heads + p.c.heads;
    const uint32_t h = head - (is_q ? 0 : is_v ? p.q_heads + p.c.heads : p.q_heads);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    int32_t slot = 0;
    if (active) {
        const RowsView& in = is_q ? p.q : is_v ? p.v : p.k;
        const int64_t at = (int64_t)t * in.token_stride + (int64_t)h * in.head_stride + lane * 4;
        a = load4<true>(in.p, at, p.dtype, p.vec);
        b = load4<true>(in.p, at + half, p.dtype, p.vec);
        if (!is_q) slot = __ldg(p.slots + t);
        if (p.cos != nullptr && !is_v) {
            const int64_t row = (int64_t)min((uint32_t)max(__ldg(p.positions + t), 0), p.rope_len - 1) * half;
            if (p.interleaved) {
                const int64_t i0 = row + lane * 2, i1 = i0 + half / 2;
                rotate(a.x, a.y, __ldg(p.cos + i0), __ldg(p.sin + i0));
                rotate(a.z, a.w, __ldg(p.cos + i0 + 1), __ldg(p.sin + i0 + 1));
                rotate(b.x, b.y, __ldg(p.cos + i1), __ldg(p.sin + i1));
                rotate(b.z, b.w, __ldg(p.cos + i1 + 1), __ldg(p.sin + i1 + 1));
            } else {
                const float4 c = load4<false>(p.cos, row + lane * 4, kF32, p.vec), s = load4<false>(p.sin, row + lane * 4, kF32, p.vec);
                rotate(a.x, b.x, c.x, s.x);
                rotate(a.y, b.y, c.y, s.y);
                rotate(a.z, b.z, c.z, s.z);
                rotate(a.w, b.w, c.w, s.w);
            }
        }
    }
    if (is_q) {
        if (active) {
            const int64_t at = ((int64_t)t * p.q_heads + h) * p.c.d + lane * 4;
            store4(p.q_out, at, p.q_out_dtype, a);
            store4(p.q_out, at + half, p.q_out_dtype, b);
        }
        if (p.c.dtype != kInt8) return;
    }
    const bool wanted = active && !is_q && slot >= 0 && (uint64_t)slot < (uint64_t)p.c.pages * p.c.page_size;
    const uint32_t page = p.by_page.quotient((uint32_t)slot & 0x7FFFFFFFu);
    const int64_t row = ((int64_t)page * p.c.heads + h) * p.c.page_size + ((uint32_t)slot - page * p.c.page_size);
    void* const cache = is_v ? p.c.v : p.c.k;
    if (p.c.dtype != kInt8) {
        if (wanted) {
            store4(cache, row * p.c.d + lane * 4, p.c.dtype, a);
            store4(cache, row * p.c.d + lane * 4 + half, p.c.dtype, b);
        }
        return;
    }
    // (the whole warp shuffles)
    float m = max_nan(max_nan(max_nan(fabsf(a.x), fabsf(a.y)), max_nan(fabsf(a.z), fabsf(a.w))),
                      max_nan(max_nan(fabsf(b.x), fabsf(b.y)), max_nan(fabsf(b.z), fabsf(b.w))));
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (!wanted) return;
    const bool finite = m < __int_as_float(0x7F800000), zero = m < MIN_AMAX;
    const float inv = finite && !zero ? __fdiv_rn(127.0f, m) : 0.0f;
    int8_t* const dst = static_cast<int8_t*>(cache) + row * p.c.d + lane * 4;
    *reinterpret_cast<uint32_t*>(dst) = finite ? codes4(a, inv) : 0u;
    *reinterpret_cast<uint32_t*>(dst + half) = finite ? codes4(b, inv) : 0u;
    if (lane == 0)
        (is_v ? p.c.v_scale : p.c.k_scale)[row] = !finite ? __int_as_float(0x7FC00000) : zero ? 0.0f : __fdiv_rn(m, 127.0f);
}

template <int LANES>
cudaError_t launch_write(const KvWriteParams& p, cudaStream_t stream) {
    const uint32_t heads = p.q_heads + 2 * p.c.heads;
    const uint32_t chunk = std::max(1u, 0x7FFFFFFFu / heads);  // rows of a launch stay below 2^31
    for (uint64_t t0 = 0; t0 < p.tokens; t0 += chunk) {
        const uint32_t rows = std::min<uint64_t>(chunk, p.tokens - t0) * heads, per = KW_THREADS / LANES;
        kv_write_kernel<LANES><<<rows / per + (rows % per != 0), KW_THREADS, 0, stream>>>(p, (uint32_t)t0, rows);
    }
    return cudaGetLastError();
}

// ---- read ----
// A block takes `tokens` tokens: it finds their rows in the cache, then groups of LANES threads (a power of two >= d / 8)
// copy a row of K and V each, eight elements a thread, KR_BATCH rows' loads in flight.
constexpr int KR_MOST = 32, KR_BATCH = 4;

struct Eight {
    uint4 w;  // 8 16-bit elements; or the 8 codes in x, y and the scale in z
};
__device__ __forceinline__ Eight read8(const KvCacheView& c, const void* src, const float* scale, int64_t row, uint32_t col) {
    Eight e;
    if (c.dtype == kInt8) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const int8_t*>(src) + row * c.d + col));
        e.w = make_uint4(w.x, w.y, __float_as_uint(__ldg(scale + row)), 0u);
    } else {
        e.w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + row * c.d + col));
    }
    return e;
}

__device__ __forceinline__ float2 widen16(uint32_t v, int dtype) {
    if (dtype == kF16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

__device__ __forceinline__ void write8(void* out, int64_t at, int out_dtype, const Eight& e, int dtype) {
    if (out_dtype == dtype) {  // 16-bit to the same type: the bits
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = e.w;
        return;
    }
    float x[8];
    if (dtype == kInt8) {
        const float s = __uint_as_float(e.w.z);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fmul_rn((float)(int8_t)((i < 4 ? e.w.x : e.w.y) >> (8 * (i & 3))), s);
    } else {
        const float2 a = widen16(e.w.x, dtype), b = widen16(e.w.y, dtype), c = widen16(e.w.z, dtype), d = widen16(e.w.w, dtype);
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
    }
    if (out_dtype == kF32) {
        float4* const o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]), o[1] = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
        make_uint4(pack16(x[0], x[1], out_dtype), pack16(x[2], x[3], out_dtype), pack16(x[4], x[5], out_dtype), pack16(x[6], x[7], out_dtype));
}

template <int LANES>
__global__ void __launch_bounds__(KW_THREADS) kv_read_kernel(const __grid_constant__ KvReadParams p, uint32_t tokens) {
    __shared__ int64_t first[KR_MOST];  // each token's row of head 0 in the cache, -1: none (its rows are zeros)
    const uint32_t t0 = blockIdx.x * tokens;
    if (threadIdx.x < tokens && t0 + threadIdx.x < p.total) {
        const int32_t t = (int32_t)(t0 + threadIdx.x);
        uint32_t lo = 0, hi = p.seqs;  // the sequence whose [cu[b], cu[b + 1]) holds t
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (__ldg(p.cu + mid + 1) <= t) lo = mid + 1;
            else hi = mid;
        }
        int64_t row = -1;
        if (lo < p.seqs && t >= __ldg(p.cu + lo)) {
            const int64_t pos = (int64_t)(t - __ldg(p.cu + lo)) + (p.starts ? p.starts[lo] : 0);
            const uint32_t col = (uint32_t)pos / p.c.page_size;
            if (pos >= 0 && pos <= INT32_MAX && col < p.table_width) {
                const int32_t page = p.block_table[(int64_t)lo * p.table_width + col];
                if (page >= 0 && (uint32_t)page < p.c.pages)
                    row = (int64_t)page * p.c.heads * p.c.page_size + ((uint32_t)pos - col * p.c.page_size);
            }
        }
        first[threadIdx.x] = row;
    }
    __syncthreads();
    constexpr uint32_t GROUPS = KW_THREADS / LANES;
    const uint32_t col = threadIdx.x % LANES * 8, rows = min(tokens, p.total - t0) * p.c.heads;
    if (col >= p.c.d) return;
    for (uint32_t r0 = threadIdx.x / LANES; r0 < rows; r0 += GROUPS * KR_BATCH) {
        Eight k[KR_BATCH], v[KR_BATCH];
#pragma unroll
        for (int i = 0; i < KR_BATCH; ++i) {
            const uint32_t r = r0 + i * GROUPS, t = r / p.c.heads;
            k[i].w = v[i].w = make_uint4(0, 0, 0, 0);
            if (r < rows && first[t] >= 0) {
                const int64_t row = first[t] + (int64_t)(r - t * p.c.heads) * p.c.page_size;
                k[i] = read8(p.c, p.c.k, p.c.k_scale, row, col);
                v[i] = read8(p.c, p.c.v, p.c.v_scale, row, col);
            }
        }
#pragma unroll
        for (int i = 0; i < KR_BATCH; ++i) {
            const uint32_t r = r0 + i * GROUPS;
            if (r >= rows) break;
            const int64_t at = ((int64_t)t0 * p.c.heads + r) * p.c.d + col;
            write8(p.k_out, at, p.out_dtype, k[i], p.c.dtype);
            write8(p.v_out, at, p.out_dtype, v[i], p.c.dtype);
        }
    }
}

template <int LANES>
cudaError_t launch_read(const KvReadParams& p, cudaStream_t stream) {
    // up to 32 tokens a block (the look-up of their rows is done once for all heads), fewer where that leaves the SMs idle
    uint32_t tokens = KR_MOST;
    while (tokens > 1 && (p.total + tokens - 1) / tokens < 4 * 148) tokens /= 2;
    kv_read_kernel<LANES><<<(p.total + tokens - 1) / tokens, KW_THREADS, 0, stream>>>(p, tokens);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteParams& params, cudaStream_t stream) {
    KvWriteParams p = params;
    p.by_heads = Divisor::of(p.q_heads + 2 * p.c.heads), p.by_page = Divisor::of(p.c.page_size);
    if (p.c.d > 64) return launch_write<16>(p, stream);
    if (p.c.d > 32) return launch_write<8>(p, stream);
    return launch_write<4>(p, stream);
}

cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream) {
    if (p.c.d > 64) return launch_read<16>(p, stream);
    if (p.c.d > 32) return launch_read<8>(p, stream);
    return launch_read<4>(p, stream);
}

}  // namespace iq2
