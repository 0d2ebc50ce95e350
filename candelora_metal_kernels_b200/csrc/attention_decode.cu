// Attention of one new token a sequence over the paged cache:
//     s_j = scale q . k_j,  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)   over the sequence's tokens j < length.
// One warp a (sequence, query head): lane l holds elements 4l..4l+3 of q and o, and keeps the running maximum and sum.
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

namespace iq2 {

namespace {

__device__ __forceinline__ float load1(const void* p, int64_t i, int dtype) {
    if (dtype == kF32) return static_cast<const float*>(p)[i];
    if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    if (dtype == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return (float)static_cast<const int8_t*>(p)[i];
}

__device__ __forceinline__ void store1(void* p, int64_t i, int dtype, float x) {
    if (dtype == kF32) static_cast<float*>(p)[i] = x;
    else if (dtype == kF16) static_cast<__half*>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

__global__ void __launch_bounds__(32) decode_kernel(const DecodeParams p) {
    const uint32_t b = blockIdx.y, hq = blockIdx.x, lane = threadIdx.x, h = hq / (p.q_heads / p.c.heads), d = p.c.d;
    const bool live = lane * 4 < d;
    float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4 && live; ++i)
        q[i] = load1(p.q.p, (int64_t)b * p.q.token_stride + (int64_t)hq * p.q.head_stride + lane * 4 + i, p.dtype) * p.scale;
    const int64_t most = (int64_t)p.table_width * p.c.page_size;
    const int64_t len = min((int64_t)max(p.seq_lens[b], 0), most);
    for (int64_t j = 0; j < len; ++j) {
        const int32_t page = p.block_table[(int64_t)b * p.table_width + j / p.c.page_size];
        if (page < 0 || (uint32_t)page >= p.c.pages) continue;
        const int64_t row = ((int64_t)page * p.c.heads + h) * p.c.page_size + j % p.c.page_size;
        float s = 0.f;
        for (int i = 0; i < 4 && live; ++i) s += q[i] * load1(p.c.k, row * d + lane * 4 + i, p.c.dtype);
        for (int x = 16; x > 0; x /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        float vs = 1.f;
        if (p.c.dtype == kInt8) s *= p.c.k_scale[row], vs = p.c.v_scale[row];
        const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - top), e = expf(s - top);
        m = top, l = l * keep + e;
        for (int i = 0; i < 4 && live; ++i) o[i] = o[i] * keep + e * vs * load1(p.c.v, row * d + lane * 4 + i, p.c.dtype);
    }
    for (int i = 0; i < 4 && live; ++i)
        store1(p.out, ((int64_t)b * p.q_heads + hq) * d + lane * 4 + i, p.dtype, m == -INFINITY ? 0.f : o[i] / l);
}

}  // namespace

size_t attention_decode_workspace(uint32_t, uint32_t, uint32_t, uint32_t, int) { return 0; }

cudaError_t launch_attention_decode(const DecodeParams& p, void*, int, cudaStream_t stream) {
    decode_kernel<<<dim3(p.q_heads, p.batch), 32, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace iq2
