// The paged key-value cache: the write of new tokens (with the rotation of q and k, and the quantisation of an int8
// cache) and the read of cached tokens back into packed tensors. Both move each byte once and are bound by HBM.
//
// Rotation, for the pair (a, b) = (x[i], x[i + d/2]) ("half") or (x[2i], x[2i + 1]) (interleaved):
//     a' = a c - b s,  b' = b c + a s,  c = cos[position][i], s = sin[position][i],
// with every product and sum rounded by itself in f32, so that a result does not depend on how the compiler fuses.
// int8 rows (one token and head): m = max |x|, scale = m / 127, code = rint(x * (127 / m)); m < 2^-100 gives zeros (the
// quotient would overflow), and a row with an infinity or NaN gets a NaN scale, so that it reads back as NaN.
// Measured (8 key heads, 128 elements): write of 2048 tokens with 32 query heads, f32 to bf16, 18.3 us over 0.9 GB of inputs and
// outputs in turn, 4190 GB/s (12.8 over 0.2 GB, where the L2 keeps part of the outputs); of 8800 tokens, f32 into an int8 cache,
// with the read back 67.5 us, 5380 GB/s; read of 89091 tokens to bf16, of an int8 cache 97 us, 5680 GB/s, of a bf16 one 117 us,
// 6220 GB/s.
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

#include <algorithm>

namespace iq2 {

namespace {

constexpr int KW_THREADS = 256;

constexpr float MIN_AMAX = 7.88860905e-31f;  // 2^-100

// 16 bytes of a row at element i, as they lie in memory: the loads of a thread are all on their way before the first is
// widened. They are not read again, so that the cache lines give way first.
template <int IN>
__device__ __forceinline__ uint4 load16(const void* base, int64_t i, bool vec) {
    if (IN == kF32) {
        const uint32_t* p = static_cast<const uint32_t*>(base) + i;
        return vec ? __ldcs(reinterpret_cast<const uint4*>(p)) : make_uint4(p[0], p[1], p[2], p[3]);
    }
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
    if (vec) return __ldcs(reinterpret_cast<const uint4*>(p));
    return make_uint4(p[0] | ((uint32_t)p[1] << 16), p[2] | ((uint32_t)p[3] << 16), p[4] | ((uint32_t)p[5] << 16), p[6] | ((uint32_t)p[7] << 16));
}

__device__ __forceinline__ float2 widen16(uint32_t v, int dtype) {
    if (dtype == kF16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

template <int IN, int V>
__device__ __forceinline__ void widen(const uint4& w, float (&x)[V]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (V == 4) {
            x[i] = __uint_as_float(u[i]);
        } else {
            const float2 f = widen16(u[i], IN);
            x[2 * i % V] = f.x, x[(2 * i + 1) % V] = f.y;
        }
    }
}

// N values of a cosine or sine row.
template <int N>
__device__ __forceinline__ void load_angles(const float* p, bool vec, float (&x)[N]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __ldg(p + i);
    } else if (N == 2) {
        const float2 f = __ldg(reinterpret_cast<const float2*>(p));
        x[0] = f.x, x[1] = f.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
            x[i] = f.x, x[i + 1] = f.y, x[(i + 2) % N] = f.z, x[(i + 3) % N] = f.w;
        }
    }
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int dtype) {
    if (dtype == kF16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// V values at element i (a multiple of V) of a 16-byte aligned tensor.
template <int V>
__device__ __forceinline__ void store_values(void* base, int64_t i, int dtype, const float (&x)[V]) {
    if (dtype == kF32) {
        float4* const o = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
#pragma unroll
        for (int j = 0; j < V; j += 4) o[j / 4] = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        return;
    }
    uint32_t w[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) w[j] = pack16(x[2 * j], x[2 * j + 1], dtype);
    uint16_t* const o = static_cast<uint16_t*>(base) + i;
    if (V == 4) *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2 % (V / 2)], w[3 % (V / 2)]);
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

__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
    // 1.5 * 2^23 more rounds |x inv| <= 127 to the nearest integer (ties to even) and leaves it in the low byte
    auto code = [&](float y) { return __float_as_uint(__fadd_rn(__fmul_rn(y, inv), 12582912.0f)); };
    return prmt(prmt(code(x[0]), code(x[1]), 0x0040u), prmt(code(x[2]), code(x[3]), 0x0040u), 0x5410u);
}

// LANES threads (a power of two >= d / 2V) take a row: lane l holds the V elements from Vl of each half, 16 bytes of the input,
// so that a pair of either rotation is in one thread and a row's maximum takes log2(LANES) shuffles. Rows are (token, head)
// with the heads of q, then k, then v. A thread has one row (two or three in flight: 2048 tokens 16.5 / 18.5 against 14.5 us);
// instructions bind next to HBM, so that divisions are products, codes are rounded by an addition, and the input's type is
// the kernel's (widened as it came, in pieces of eight bytes, bf16 rows of 8800 tokens took 61.5 us into a bf16 cache, not 43.6).
// Blocks of an SM: eight for f32 rows (8800 tokens into a bf16 cache 54.0 us; with all the registers that the compiler likes
// 58.8), six for the 16 values of a thread that 16-bit rows make (43.6 us; five 45.0, seven 44.9, with spills).
template <int LANES, int IN>
__global__ void __launch_bounds__(KW_THREADS, IN == kF32 ? 8 : 6) kv_write_kernel(const __grid_constant__ KvWriteParams p, uint32_t token0, uint32_t rows) {
    constexpr int V = IN == kF32 ? 4 : 8;
    const uint32_t lane = threadIdx.x % LANES, r = blockIdx.x * (KW_THREADS / LANES) + threadIdx.x / LANES;
    const uint32_t heads = p.q_heads + 2 * p.c.heads, half = p.c.d / 2;
    const bool live = r < rows, active = live && lane * (2 * V) < p.c.d;
    const uint32_t in_launch = p.by_heads.quotient(r), t = token0 + in_launch, head = r - in_launch * heads;
    const bool is_q = head < p.q_heads, is_v = head >= p.q_heads + p.c.heads;
    const uint32_t h = head - (is_q ? 0 : is_v ? p.q_heads + p.c.heads : p.q_heads);
    float a[V] = {}, b[V] = {};
    int32_t slot = 0;
    if (active) {
        const RowsView& in = is_q ? p.q : is_v ? p.v : p.k;
        const int64_t at = (int64_t)t * in.token_stride + (int64_t)h * in.head_stride + lane * V;
        const uint4 wa = load16<IN>(in.p, at, p.vec), wb = load16<IN>(in.p, at + half, p.vec);
        if (!is_q) slot = __ldg(p.slots + t);
        const bool rotated = p.cos != nullptr && !is_v;
        const int64_t row = rotated ? (int64_t)min((uint32_t)max(__ldg(p.positions + t), 0), p.rope_len - 1) * half : 0;
        if (!rotated) {
            widen<IN>(wa, a), widen<IN>(wb, b);
        } else if (p.interleaved) {
            const int64_t i0 = row + lane * (V / 2), i1 = i0 + half / 2;
            float c0[V / 2], s0[V / 2], c1[V / 2], s1[V / 2];
            load_angles(p.cos + i0, p.vec, c0), load_angles(p.sin + i0, p.vec, s0);
            load_angles(p.cos + i1, p.vec, c1), load_angles(p.sin + i1, p.vec, s1);
            widen<IN>(wa, a), widen<IN>(wb, b);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) rotate(a[2 * i], a[2 * i + 1], c0[i], s0[i]), rotate(b[2 * i], b[2 * i + 1], c1[i], s1[i]);
        } else {
            float c[V], s[V];
            load_angles(p.cos + row + lane * V, p.vec, c), load_angles(p.sin + row + lane * V, p.vec, s);
            widen<IN>(wa, a), widen<IN>(wb, b);
#pragma unroll
            for (int i = 0; i < V; ++i) rotate(a[i], b[i], c[i], s[i]);
        }
    }
    if (is_q && active) {
        const int64_t at = ((int64_t)t * p.q_heads + h) * p.c.d + lane * V;
        store_values(p.q_out, at, p.q_out_dtype, a);
        store_values(p.q_out, at + half, p.q_out_dtype, b);
    }
    if (p.c.dtype != kInt8) {
        if (is_q) return;
    } else if (__all_sync(0xFFFFFFFFu, is_q)) {  // (a warp that goes on shuffles as a whole)
        return;
    }
    const bool wanted = active && !is_q && slot >= 0 && (uint64_t)slot < (uint64_t)p.c.pages * p.c.page_size;
    const uint32_t page = p.by_page.quotient((uint32_t)slot & 0x7FFFFFFFu);
    const int64_t row = ((int64_t)page * p.c.heads + h) * p.c.page_size + ((uint32_t)slot - page * p.c.page_size);
    void* const cache = is_v ? p.c.v : p.c.k;
    if (p.c.dtype != kInt8) {
        if (wanted) {
            store_values(cache, row * p.c.d + lane * V, p.c.dtype, a);
            store_values(cache, row * p.c.d + lane * V + half, p.c.dtype, b);
        }
        return;
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max_nan(m, max_nan(fabsf(a[i]), fabsf(b[i])));
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (!wanted) return;
    const bool finite = m < __int_as_float(0x7F800000), zero = m < MIN_AMAX;
    const float inv = finite && !zero ? __fdiv_rn(127.0f, m) : 0.0f;
    int8_t* const dst = static_cast<int8_t*>(cache) + row * p.c.d + lane * V;
    uint32_t code[V / 2];
#pragma unroll
    for (int i = 0; i < V; i += 4) code[i / 4] = finite ? codes4(a + i, inv) : 0u, code[(V + i) / 4] = finite ? codes4(b + i, inv) : 0u;
    if (V == 4) {
        *reinterpret_cast<uint32_t*>(dst) = code[0];
        *reinterpret_cast<uint32_t*>(dst + half) = code[1];
    } else {
        *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
        *reinterpret_cast<uint2*>(dst + half) = make_uint2(code[2 % (V / 2)], code[3 % (V / 2)]);
    }
    if (lane == 0)
        (is_v ? p.c.v_scale : p.c.k_scale)[row] = !finite ? __int_as_float(0x7FC00000) : zero ? 0.0f : __fdiv_rn(m, 127.0f);
}

template <int LANES, int IN>
cudaError_t launch_write(const KvWriteParams& p, cudaStream_t stream) {
    const uint32_t heads = p.q_heads + 2 * p.c.heads;
    const uint32_t chunk = std::max(1u, 0x7FFFFFFFu / heads);  // rows of a launch stay below 2^31
    for (uint64_t t0 = 0; t0 < p.tokens; t0 += chunk) {
        const uint32_t rows = std::min<uint64_t>(chunk, p.tokens - t0) * heads, per = KW_THREADS / LANES;
        kv_write_kernel<LANES, IN><<<rows / per + (rows % per != 0), KW_THREADS, 0, stream>>>(p, (uint32_t)t0, rows);
    }
    return cudaGetLastError();
}

template <int IN>
cudaError_t launch_write_of(const KvWriteParams& p, cudaStream_t stream) {
    constexpr int MOST = IN == kF32 ? 16 : 8;  // lanes of a row of 128 elements
    if (p.c.d > 64) return launch_write<MOST, IN>(p, stream);
    if (p.c.d > 32) return launch_write<MOST / 2, IN>(p, stream);
    return launch_write<MOST / 4, IN>(p, stream);
}

// ---- read ----
// A block takes `tokens` tokens: it finds their rows in the cache, then groups of LANES threads (a power of two >= d / 8)
// copy a row of K and V each, eight elements a thread, KR_BATCH rows' loads in flight. An int8 cache is read at one byte for
// two written, and the stores bind (codes widened by byte permutes instead of conversions: 96.0 us as well; stores that give
// way in the cache: 96.6).
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
    if (p.dtype == kF32) return launch_write_of<kF32>(p, stream);
    return p.dtype == kF16 ? launch_write_of<kF16>(p, stream) : launch_write_of<kBf16>(p, stream);
}

cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream) {
    if (p.c.d > 64) return launch_read<16>(p, stream);
    if (p.c.d > 32) return launch_read<8>(p, stream);
    return launch_read<4>(p, stream);
}

}  // namespace iq2
