// The paged key-value cache: the write of new tokens (with the rotation of q and k, and the quantisation of an int8
// cache) and the read of cached tokens back into packed tensors. Both move each byte once and are bound by HBM.
//
// Rotation, for the pair (a, b) = (x[i], x[i + d/2]) ("half") or (x[2i], x[2i + 1]) (interleaved):
//     a' = a c - b s,  b' = b c + a s,  c = cos[position][i], s = sin[position][i],
// with every product and sum rounded by itself in f32, so that a result does not depend on how the compiler fuses.
// int8 rows (one token and head): m = max |x|, scale = m / 127, code = rint(x * (127 / m)); m < 2^-100 gives zeros (the
// quotient would overflow), and a row with an infinity or NaN gets a NaN scale, so that it reads back as NaN.
// 4-bit rows: s = the power of two with 224 < m / 7s <= 448, a group's g = e4m3(m_g / 7s), code = the integer nearest to
// x / (s g), ties to even, at most 7 (g may be 2^-4 of itself below m_g / 7s: 7.44 still rounds to 7). Steps s g of four
// significant bits make the values exact in 16 bits, and codes of 16-bit inputs are those of the quotient itself, whatever the
// arithmetic: a code is taken from the product with 1 / (s g) and the remainder x - code s g, exact in f32, says where that is off.
// Norms: y = (x r) w, r = 1 / sqrt(mean(x^2) + eps) summed and taken in 64 bits and rounded to f32, so that r, and with it the
// codes next to borders, does not depend on the order of the sum.
// Measured (8 key heads, 128 elements): write of 2048 tokens with 32 query heads, f32 to bf16, 12.3 us over 0.9 GB of inputs and
// outputs in turn, 6240 GB/s (10.7 over 0.2 GB, where the L2 keeps part of the outputs), with norms 15.9 us, as into an int8 cache
// (bf16 to bf16 11.1 and 14.2); of 8800 tokens, f32 into an int8 cache, with the read back 61 us, 5960 GB/s, into a 4-bit cache 61 us, from
// bf16 or f16 55 us, from bf16 with norms 66 us, of which the write is 55: with 36 warps an SM it waits for its loads in between (73 %
// of the issue slots, 403 instructions for four rows). Read of 89091 tokens to bf16: of an int8 cache 96 us, 5750 GB/s, of a bf16 one
// 117 us, 6220 GB/s, of a 4-bit one 84 us, 5550 GB/s, 365 MB of the 467 written.
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
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
            x[i] = f.x, x[(i + 1) % N] = f.y, x[(i + 2) % N] = f.z, x[(i + 3) % N] = f.w;
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

// ---- write of rows or tables off the 16-byte boundaries, without norms, into 16-bit and int8 caches ----
// LANES threads (a power of two >= d / 2V) take a row: lane l holds the V elements from Vl of each half, 16 bytes of the input,
// so that a pair of either rotation is in one thread and a row's maximum takes log2(LANES) shuffles. Rows are (token, head)
// with the heads of q, then k, then v. What is loaded element by element then lies close together: 2048 tokens from f32 into a bf16
// cache take 15.9 us, 8800 61.2, where the kernel below takes 20.9 and 80.1 (from bf16 14.3 and 53.9 against 14.6 and 55.8). For
// rows on the boundaries that one is the faster, 10.8 and 51.5 us against 12.1 and 58.0 (from bf16 9.4 and 43.0 against 10.5 and 48.4).
// Blocks of an SM: eight for f32 rows (8 / 7 / 6 with element loads alone: 65.7 / 66.4 / 76.1 us for 8800 tokens), six for the 16 values
// of a thread that 16-bit rows make (6 / 5: 52.1 / 57.1).
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
        const uint4 wa = load16<IN>(in.p, at, p.vec_rows), wb = load16<IN>(in.p, at + half, p.vec_rows);
        if (!is_q) slot = __ldg(p.slots + t);
        const bool rotated = p.cos != nullptr && !is_v;
        const int64_t row = rotated ? (int64_t)min((uint32_t)max(__ldg(p.positions + t), 0), p.rope_len - 1) * half : 0;
        if (!rotated) {
            widen<IN>(wa, a), widen<IN>(wb, b);
        } else if (p.interleaved) {
            const int64_t i0 = row + lane * (V / 2), i1 = i0 + half / 2;
            float c0[V / 2], s0[V / 2], c1[V / 2], s1[V / 2];
            load_angles(p.cos + i0, false, c0), load_angles(p.sin + i0, false, s0);
            load_angles(p.cos + i1, false, c1), load_angles(p.sin + i1, false, s1);
            widen<IN>(wa, a), widen<IN>(wb, b);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) rotate(a[2 * i], a[2 * i + 1], c0[i], s0[i]), rotate(b[2 * i], b[2 * i + 1], c1[i], s1[i]);
        } else {
            float c[V], s[V];
            load_angles(p.cos + row + lane * V, false, c), load_angles(p.sin + row + lane * V, false, s);
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

// ---- write: with norms, into 4-bit caches, and of rows on the 16-byte boundaries ----
// As above, but a thread has eight elements of each half whatever the input's type (fewer threads share a row's sums, maxima and
// addresses), a block has rows of one of q, k and v, and rows off the 16-byte boundaries are a kernel of their own (their
// loads element by element are predicated away in one that has both, but issued all the same: 28 instead of 12 loads a warp; all
// of it 22.5 -> 18.4 us for 2048 tokens with norms). Of a block, whose rows end together, 32 / 64 / 96 / 128 / 256 threads take 17.6 /
// 17.7 / 18.0 / 17.8 / 18.4 us and, 8800 tokens from bf16 with norms into a 4-bit cache and back, 73.7 / 72.0 / 74.3 / 73.1 / 75.1.
// Threads of an SM, then: with norms 896 / 1024 / 1152 (56 registers) 17.7 / 17.9 / 17.3 and 70.2 / 70.2 / 67.7 us; without, 8800 tokens
// from f32 into a 4-bit cache and back, 1152 / 1280 / 1344 (40 registers, aligned rows without
// spills) / 1408 64.3 / 62.7 / 61.5 / 63.5.
constexpr int KN_THREADS = 64;
constexpr int KN = 8;
enum RowKind { ROW_Q, ROW_K, ROW_V };

// Eight elements of a row in f32.
template <int IN, bool VEC>
__device__ __forceinline__ void load_eight(const void* base, int64_t i, float (&x)[KN]) {
    if (IN == kF32) {
        const uint4 a = load16<IN>(base, i, VEC), b = load16<IN>(base, i + 4, VEC);
        float y[4], z[4];
        widen<IN>(a, y), widen<IN>(b, z);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = y[j], x[4 + j] = z[j];
    } else {
        widen<IN>(load16<IN>(base, i, VEC), x);
    }
}

// The value of e4m3 bits without a sign, and the bits nearest to two numbers >= 0.
__device__ __forceinline__ float e4m3_value(uint32_t bits) { return __uint_as_float(bits << 20) * 1.32922800e36f; }  // 2^120
__device__ __forceinline__ uint32_t e4m3_pair(float low, float high) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
    return r;
}

// Eight codes of a group as nibbles. `g` are the bits of the group's scale, `s` the row's. The product with 1 / (s g) is off by
// three roundings, 2^-20 at most.
// SHORT: x are 16-bit numbers. Their quotients by a step of four bits are ties or 2^-12 and more from one, so that rounding them to
// multiples of 2^-15 first makes ties of ties. Otherwise the remainder x - code s g says where the code may be the neighbour's,
// or a tie that goes to the even one: those threads go over their codes again. Where g is no normal number codes may pass 7.
template <bool SHORT>
__device__ __forceinline__ uint32_t codes_int4(const float (&x)[KN], uint32_t g, float s) {
    const float step = s * e4m3_value(g);
    float inv, c[KN];
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(step));
    if (g == 0) inv = 0.f;
    auto whole = [](float q) { return __fadd_rn(__fadd_rn(q, 12582912.0f), -12582912.0f); };
    if (SHORT) {
#pragma unroll
        for (int i = 0; i < KN; ++i) c[i] = whole(__fadd_rn(__fadd_rn(__fmul_rn(x[i], inv), 384.0f), -384.0f));
    } else {
        float worst = 0.f;
#pragma unroll
        for (int i = 0; i < KN; ++i) {
            c[i] = whole(__fmul_rn(x[i], inv));
            worst = fmaxf(worst, fabsf(__fmaf_rn(-c[i], step, x[i])));
        }
        if (g != 0 && worst >= 0.5f * step) {
#pragma unroll
            for (int i = 0; i < KN; ++i) {
                const float rest = __fmaf_rn(-c[i], step, x[i]), over = fabsf(rest) - 0.5f * step;
                if (over > 0.f || (over == 0.f && ((int)c[i] & 1))) c[i] += copysignf(1.f, rest);
            }
        }
    }
    if (g < 8) {
#pragma unroll
        for (int i = 0; i < KN; ++i) c[i] = fminf(fmaxf(c[i], -7.f), 7.f);
    }
    uint32_t byte[KN / 2];  // 8 + code in each half: 2^23 + 2^22 more leaves them in the lowest bits
#pragma unroll
    for (int i = 0; i < KN / 2; ++i) byte[i] = __float_as_uint(__fmaf_rn(c[2 * i + 1], 16.f, c[2 * i]) + (12582912.0f + 136.0f));
    return prmt(prmt(byte[0], byte[1], 0x0040u), prmt(byte[2], byte[3], 0x0040u), 0x5410u);
}

template <int LANES, int IN, bool NORM, bool I4, bool VEC>
__global__ void __launch_bounds__(KN_THREADS, (NORM ? 1152 : 1344) / KN_THREADS) kv_write_rows_kernel(const __grid_constant__ KvWriteParams p, uint32_t token0, uint32_t tokens) {
    constexpr uint32_t PER = KN_THREADS / LANES;
    const uint32_t lane = threadIdx.x % LANES, half = p.c.d / 2;
    const int kind = blockIdx.x < p.blocks_q ? ROW_Q : blockIdx.x < p.blocks_q + p.blocks_kv ? ROW_K : ROW_V;
    const uint32_t block = blockIdx.x - (kind == ROW_Q ? 0 : kind == ROW_K ? p.blocks_q : p.blocks_q + p.blocks_kv);
    const uint32_t heads = kind == ROW_Q ? p.q_heads : p.c.heads, r = block * PER + threadIdx.x / LANES;
    const uint32_t in_launch = kind == ROW_Q ? p.by_q.quotient(r) : p.by_kv.quotient(r), t = token0 + in_launch, h = r - in_launch * heads;
    const bool active = in_launch < tokens && lane * (2 * KN) < p.c.d;
    const RowsView& in = kind == ROW_Q ? p.q : kind == ROW_K ? p.k : p.v;
    const bool rotated = p.cos != nullptr && kind != ROW_V;
    const float* const weights = kind == ROW_Q ? p.q_norm : kind == ROW_K ? p.k_norm : nullptr;
    float a[KN] = {}, b[KN] = {}, c[KN], s[KN];  // (rows that are not there add up to nothing)
    int32_t slot = -1;
    if (active) {
        const int64_t at = (int64_t)t * in.token_stride + (int64_t)h * in.head_stride + lane * KN;
        load_eight<IN, VEC>(in.p, at, a), load_eight<IN, VEC>(in.p, at + half, b);
        if (kind != ROW_Q) slot = __ldg(p.slots + t);
        if (rotated) {
            const int64_t row = (int64_t)min((uint32_t)max(__ldg(p.positions + t), 0), p.rope_len - 1) * half;
            if (p.interleaved) {  // the pairs of a, then those of b
                float c0[KN / 2], s0[KN / 2], c1[KN / 2], s1[KN / 2];
                const int64_t i0 = row + lane * (KN / 2), i1 = i0 + half / 2;
                load_angles(p.cos + i0, VEC, c0), load_angles(p.sin + i0, VEC, s0);
                load_angles(p.cos + i1, VEC, c1), load_angles(p.sin + i1, VEC, s1);
#pragma unroll
                for (int i = 0; i < KN / 2; ++i) c[i] = c0[i], s[i] = s0[i], c[KN / 2 + i] = c1[i], s[KN / 2 + i] = s1[i];
            } else {
                load_angles(p.cos + row + lane * KN, VEC, c), load_angles(p.sin + row + lane * KN, VEC, s);
            }
        }
    }
    if (NORM && weights != nullptr) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < KN; ++i) sum = fma((double)a[i], (double)a[i], sum), sum = fma((double)b[i], (double)b[i], sum);
#pragma unroll
        for (int o = LANES / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (active) {
            const float root = (float)rsqrt(sum * p.inv_d + p.eps);
            const float* const at = weights + h * (kind == ROW_Q ? p.q_norm_stride : p.k_norm_stride) + lane * KN;
            float w[KN];
            load_angles(at, VEC, w);
#pragma unroll
            for (int i = 0; i < KN; ++i) a[i] = __fmul_rn(__fmul_rn(a[i], root), w[i]);
            load_angles(at + half, VEC, w);
#pragma unroll
            for (int i = 0; i < KN; ++i) b[i] = __fmul_rn(__fmul_rn(b[i], root), w[i]);
        }
    }
    if (active && rotated) {
        if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < KN / 2; ++i) rotate(a[2 * i], a[2 * i + 1], c[i], s[i]), rotate(b[2 * i], b[2 * i + 1], c[KN / 2 + i], s[KN / 2 + i]);
        } else {
#pragma unroll
            for (int i = 0; i < KN; ++i) rotate(a[i], b[i], c[i], s[i]);
        }
    }
    if (kind == ROW_Q) {
        if (active) {
            const int64_t at = ((int64_t)t * p.q_heads + h) * p.c.d + lane * KN;
            store_values(p.q_out, at, p.q_out_dtype, a);
            store_values(p.q_out, at + half, p.q_out_dtype, b);
        }
        return;
    }
    const bool wanted = slot >= 0 && (uint64_t)slot < (uint64_t)p.c.pages * p.c.page_size;
    const uint32_t page = p.by_page.quotient((uint32_t)slot & 0x7FFFFFFFu);
    const int64_t row = ((int64_t)page * p.c.heads + h) * p.c.page_size + ((uint32_t)slot - page * p.c.page_size);
    void* const cache = kind == ROW_V ? p.c.v : p.c.k;
    float* const scales = kind == ROW_V ? p.c.v_scale : p.c.k_scale;
    const uint32_t at_a = lane * KN, at_b = half + lane * KN;
    if (!I4 && p.c.dtype != kInt8) {
        if (wanted) {
            store_values(cache, row * p.c.d + at_a, p.c.dtype, a);
            store_values(cache, row * p.c.d + at_b, p.c.dtype, b);
        }
        return;
    }
    float ma = 0.f, mb = 0.f;
#pragma unroll
    for (int i = 0; i < KN; ++i) ma = max_nan(ma, fabsf(a[i])), mb = max_nan(mb, fabsf(b[i]));
    float m = max_nan(ma, mb);
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const bool finite = m < __int_as_float(0x7F800000), some = finite && m >= MIN_AMAX;
    if (!I4) {
        if (!wanted) return;
        const float inv = some ? __fdiv_rn(127.0f, m) : 0.0f;
        int8_t* const dst = static_cast<int8_t*>(cache) + row * p.c.d;
        *reinterpret_cast<uint2*>(dst + at_a) = finite ? make_uint2(codes4(a, inv), codes4(a + 4, inv)) : make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(dst + at_b) = finite ? make_uint2(codes4(b, inv), codes4(b + 4, inv)) : make_uint2(0u, 0u);
        if (lane == 0) scales[row] = !finite ? __int_as_float(0x7FC00000) : some ? __fdiv_rn(m, 127.0f) : 0.0f;
        return;
    }
    // the groups' maxima: of four threads side by side, or, where the halves do not begin on a group, of pieces of eight in
    // shared memory
    if (half % I4_GROUP == 0) {
#pragma unroll
        for (int o = 1; o < (int)I4_GROUP / KN; o *= 2) {
            ma = max_nan(ma, __shfl_xor_sync(0xFFFFFFFFu, ma, o));
            mb = max_nan(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, o));
        }
    } else {
        __shared__ float4 held[PER][LANES / 2];
        float* const piece = reinterpret_cast<float*>(held[threadIdx.x / LANES]);
        if (at_a < half) piece[at_a / KN] = ma, piece[at_b / KN] = mb;
        __syncwarp();
        if (at_a < half) {
            const float4 x = held[threadIdx.x / LANES][at_a / I4_GROUP], y = held[threadIdx.x / LANES][at_b / I4_GROUP];
            ma = max_nan(max_nan(x.x, x.y), max_nan(x.z, x.w)), mb = max_nan(max_nan(y.x, y.y), max_nan(y.z, y.w));
        }
    }
    if (!wanted) return;
    // s and 1 / s: the exponent of m, less 11, and one more where m's fraction passes 3136 / 2048
    const uint32_t bits = __float_as_uint(m), e = some ? (bits >> 23) - 11 + ((bits & 0x7FFFFFu) > 0x440000u) : 127u;
    const float scale = some ? __uint_as_float(e << 23) : 0.f, up = __uint_as_float((254u - e) << 23);
    const uint32_t g = some ? e4m3_pair(__fdiv_rn(ma, 7.f) * up, __fdiv_rn(mb, 7.f) * up) : 0u;
    uint8_t* const dst = static_cast<uint8_t*>(cache) + row * half;
    uint32_t wa = 0x88888888u, wb = wa;
    if (some) {
        if (IN != kF32 && kind == ROW_V) wa = codes_int4<true>(a, g & 0xFFu, scale), wb = codes_int4<true>(b, g >> 8, scale);
        else wa = codes_int4<false>(a, g & 0xFFu, scale), wb = codes_int4<false>(b, g >> 8, scale);
    }
    *reinterpret_cast<uint32_t*>(dst + at_a / 2) = wa;
    *reinterpret_cast<uint32_t*>(dst + at_b / 2) = wb;
    uint8_t* const groups = (kind == ROW_V ? p.c.v_group : p.c.k_group) + row * 4;
    if (at_a % I4_GROUP == 0) groups[at_a / I4_GROUP] = (uint8_t)g;
    if (at_b % I4_GROUP == 0) groups[at_b / I4_GROUP] = (uint8_t)(g >> 8);
    if (lane == 0) scales[row] = finite ? scale : __int_as_float(0x7FC00000);
}

template <int LANES, int IN, bool NORM, bool I4, bool VEC>
cudaError_t launch_write_rows(KvWriteParams p, cudaStream_t stream) {
    constexpr uint32_t PER = KN_THREADS / LANES;
    const uint32_t chunk = std::max(1u, 0x7FFFFFFFu / (p.q_heads + 2 * p.c.heads) / 2);  // rows of a launch, and of blocks that part full, stay below 2^31
    auto blocks = [&](uint32_t tokens, uint32_t heads) { return (uint32_t)(((uint64_t)tokens * heads + PER - 1) / PER); };
    for (uint64_t t0 = 0; t0 < p.tokens; t0 += chunk) {
        const uint32_t tokens = (uint32_t)std::min<uint64_t>(chunk, p.tokens - t0);
        p.blocks_q = blocks(tokens, p.q_heads), p.blocks_kv = blocks(tokens, p.c.heads);
        kv_write_rows_kernel<LANES, IN, NORM, I4, VEC><<<p.blocks_q + 2 * p.blocks_kv, KN_THREADS, 0, stream>>>(p, (uint32_t)t0, tokens);
    }
    return cudaGetLastError();
}

template <int IN, bool NORM, bool I4, bool VEC>
cudaError_t launch_write_rows_of(const KvWriteParams& p, cudaStream_t stream) {
    if (p.c.d > 64) return launch_write_rows<8, IN, NORM, I4, VEC>(p, stream);
    if (p.c.d > 32) return launch_write_rows<4, IN, NORM, I4, VEC>(p, stream);
    return launch_write_rows<2, IN, NORM, I4, VEC>(p, stream);
}

template <int IN, bool VEC>
cudaError_t launch_write_rows_by(const KvWriteParams& p, cudaStream_t stream) {
    const bool norm = p.q_norm != nullptr || p.k_norm != nullptr;
    if (p.c.dtype != kInt4) {
        if (norm) return launch_write_rows_of<IN, true, false, VEC>(p, stream);
        if constexpr (VEC) return launch_write_rows_of<IN, false, false, true>(p, stream);
        else return launch_write_of<IN>(p, stream);
    }
    return norm ? launch_write_rows_of<IN, true, true, VEC>(p, stream) : launch_write_rows_of<IN, false, true, VEC>(p, stream);
}

// ---- read ----
// A block takes `tokens` tokens: it finds their rows in the cache, then groups of LANES threads (a power of two >= d / 8)
// copy a row of K and V each, eight elements a thread, KR_BATCH rows' loads in flight. An int8 cache is read at one byte for
// two written, and the stores bind (codes widened by byte permutes instead of conversions: 96.0 us as well; stores that give
// way in the cache: 96.6). Threads of a block, an eighth as many tokens: of a 4-bit cache 96 / 128 / 160 / 192 / 224 / 256 / 384 take
// 85.2 / 92.4 / 84.8 / 85.3 / 91 / 96.2 / 87.8 us for 89091 tokens, 14.9 / - / 13.2 / 13.4 / - / 15.5 / - for 8800 (rows that are
// in flight together are no power of two apart), of an int8 cache 160 / 192 / 256 / 384 take 100.0 / 100.2 / 97.1 / 113.4.
constexpr int KR_BATCH = 4;
template <bool I4>
struct ReadShape {
    static constexpr uint32_t THREADS = I4 ? 160 : 256, MOST = THREADS / 8;  // of a block, and its tokens at most
};

struct Eight {
    uint4 w;  // 8 16-bit elements; or the 8 codes in x, y and the scale in z; or 8 4-bit codes in x, their group's scale in y, the row's in z
};
template <bool I4>
__device__ __forceinline__ Eight read8(const KvCacheView& c, const void* src, const float* scale, const uint8_t* group, int64_t row, uint32_t col) {
    Eight e;
    if (I4) {
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(src) + (row * c.d + col) / 2));
        e.w = make_uint4(w, __ldg(group + row * 4 + col / I4_GROUP), __float_as_uint(__ldg(scale + row)), 0u);
    } else if (c.dtype == kInt8) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const int8_t*>(src) + row * c.d + col));
        e.w = make_uint4(w.x, w.y, __float_as_uint(__ldg(scale + row)), 0u);
    } else {
        e.w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + row * c.d + col));
    }
    return e;
}

template <bool I4>
__device__ __forceinline__ void write8(void* out, int64_t at, int out_dtype, const Eight& e, int dtype) {
    if (!I4 && out_dtype == dtype) {  // 16-bit to the same type: the bits
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = e.w;
        return;
    }
    float x[8];
    if (I4) {  // (code + 8) as the f16 number of its bits, times the group's scale, exactly: code g 2^-15; then one rounding in f32
        const uint32_t moved = e.w.y << 7, two = moved | moved << 16, even = e.w.x << 2, odd = e.w.x >> 6;
        const __half2 g = *reinterpret_cast<const __half2*>(&two);  // g 2^-8
        const __half2 lo = __hmul2(g, __float2half2_rn(32768.f)), hi = __hmul2(g, __float2half2_rn(2048.f)), off = __hmul2(g, __float2half2_rn(-0.0625f));
        const uint32_t u[4] = {even & 0x003C003Cu, even & 0x03C003C0u, odd & 0x003C003Cu, odd & 0x03C003C0u};  // elements i and i + 4
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(__hfma2(*reinterpret_cast<const __half2*>(&u[i]), i % 2 ? hi : lo, off));
            x[i] = f.x, x[4 + i] = f.y;
        }
        float s = __uint_as_float(e.w.z);
        if (fabsf(s) < 5.19e33f) {  // 2^112
            s *= 32768.f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= 32768.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(x[i], s);
    } else if (dtype == kInt8) {
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

template <int LANES, bool I4>
__global__ void __launch_bounds__(ReadShape<I4>::THREADS) kv_read_kernel(const __grid_constant__ KvReadParams p, uint32_t tokens) {
    __shared__ int64_t first[ReadShape<I4>::MOST];  // each token's row of head 0 in the cache, -1: none (its rows are zeros)
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
    constexpr uint32_t GROUPS = ReadShape<I4>::THREADS / LANES;
    const uint32_t col = threadIdx.x % LANES * 8, rows = min(tokens, p.total - t0) * p.c.heads;
    if (col >= p.c.d) return;
    for (uint32_t r0 = threadIdx.x / LANES; r0 < rows; r0 += GROUPS * KR_BATCH) {
        Eight k[KR_BATCH], v[KR_BATCH];
#pragma unroll
        for (int i = 0; i < KR_BATCH; ++i) {
            const uint32_t r = r0 + i * GROUPS, t = I4 ? p.by_heads.quotient(r) : r / p.c.heads;
            k[i].w = v[i].w = make_uint4(I4 ? 0x88888888u : 0u, 0, 0, 0);
            if (r < rows && first[t] >= 0) {
                const int64_t row = first[t] + (int64_t)(r - t * p.c.heads) * p.c.page_size;
                k[i] = read8<I4>(p.c, p.c.k, p.c.k_scale, p.c.k_group, row, col);
                v[i] = read8<I4>(p.c, p.c.v, p.c.v_scale, p.c.v_group, row, col);
            }
        }
#pragma unroll
        for (int i = 0; i < KR_BATCH; ++i) {
            const uint32_t r = r0 + i * GROUPS;
            if (r >= rows) break;
            const int64_t at = ((int64_t)t0 * p.c.heads + r) * p.c.d + col;
            write8<I4>(p.k_out, at, p.out_dtype, k[i], p.c.dtype);
            write8<I4>(p.v_out, at, p.out_dtype, v[i], p.c.dtype);
        }
    }
}

template <int LANES, bool I4>
cudaError_t launch_read(const KvReadParams& p, cudaStream_t stream) {
    // up to 32 (20) tokens a block (the look-up of their rows is done once for all heads), fewer where that leaves the SMs idle
    uint32_t tokens = ReadShape<I4>::MOST;
    while (tokens > 1 && (p.total + tokens - 1) / tokens < 4 * 148) tokens /= 2;
    kv_read_kernel<LANES, I4><<<(p.total + tokens - 1) / tokens, ReadShape<I4>::THREADS, 0, stream>>>(p, tokens);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteParams& params, cudaStream_t stream) {
    KvWriteParams p = params;
    p.by_heads = Divisor::of(p.q_heads + 2 * p.c.heads), p.by_page = Divisor::of(p.c.page_size);
    p.by_q = Divisor::of(std::max(p.q_heads, 1u)), p.by_kv = Divisor::of(p.c.heads);
    if (p.dtype == kF32) return p.vec ? launch_write_rows_by<kF32, true>(p, stream) : launch_write_rows_by<kF32, false>(p, stream);
    if (p.dtype == kF16) return p.vec ? launch_write_rows_by<kF16, true>(p, stream) : launch_write_rows_by<kF16, false>(p, stream);
    return p.vec ? launch_write_rows_by<kBf16, true>(p, stream) : launch_write_rows_by<kBf16, false>(p, stream);
}

template <bool I4>
static cudaError_t launch_read_rows(const KvReadParams& p, cudaStream_t stream) {
    if (p.c.d > 64) return launch_read<16, I4>(p, stream);
    if (p.c.d > 32) return launch_read<8, I4>(p, stream);
    return launch_read<4, I4>(p, stream);
}

cudaError_t launch_kv_read(const KvReadParams& params, cudaStream_t stream) {
    KvReadParams p = params;
    p.by_heads = Divisor::of(p.c.heads);
    return p.c.dtype == kInt4 ? launch_read_rows<true>(p, stream) : launch_read_rows<false>(p, stream);
}

}  // namespace iq2
