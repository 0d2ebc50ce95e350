// Attention of packed prompts: for query i of a sequence with Lq queries and Lk keys
//     o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max_j),  j < Lk, and j <= i + Lk - Lq if causal.
// One warp a (token, query head): lane l holds elements 4l..4l+3 of q and o, and keeps the running maximum and sum.
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

namespace iq2 {

namespace {

__device__ __forceinline__ float load16(const void* p, int64_t i, int dtype) {
    return dtype == kF16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__global__ void __launch_bounds__(128) prefill_kernel(const PrefillParams p) {
    const int32_t t = (int32_t)(blockIdx.x * 4 + threadIdx.x / 32);
    const uint32_t hq = blockIdx.y, lane = threadIdx.x % 32, h = hq / (p.q_heads / p.kv_heads), d = p.d;
    if (t >= (int32_t)p.q_tokens) return;
    uint32_t b = 0;
    while (b < p.seqs && !(t >= p.cu_q[b] && t < p.cu_q[b + 1])) ++b;
    if (b == p.seqs) return;
    const int64_t k0 = min(max(p.cu_k[b], 0), (int)p.k_tokens), k1 = min(max(p.cu_k[b + 1], (int)k0), (int)p.k_tokens), lk = k1 - k0;
    const int64_t shown = p.causal ? min(lk, (int64_t)(t - p.cu_q[b]) + 1 + lk - (p.cu_q[b + 1] - p.cu_q[b])) : lk;
    const bool live = lane * 4 < d;
    float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4 && live; ++i)
        q[i] = load16(p.q.p, (int64_t)t * p.q.token_stride + (int64_t)hq * p.q.head_stride + lane * 4 + i, p.dtype) * p.scale;
    for (int64_t j = k0; j < k0 + shown; ++j) {
        const int64_t kr = j * p.k.token_stride + (int64_t)h * p.k.head_stride + lane * 4, vr = j * p.v.token_stride + (int64_t)h * p.v.head_stride + lane * 4;
        float s = 0.f;
        for (int i = 0; i < 4 && live; ++i) s += q[i] * load16(p.k.p, kr + i, p.dtype);
        for (int x = 16; x > 0; x /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - top), e = expf(s - top);
        m = top, l = l * keep + e;
        for (int i = 0; i < 4 && live; ++i) o[i] = o[i] * keep + e * load16(p.v.p, vr + i, p.dtype);
    }
    for (int i = 0; i < 4 && live; ++i) {
        const int64_t at = ((int64_t)t * p.q_heads + hq) * d + lane * 4 + i;
        const float x = shown > 0 ? o[i] / l : 0.f;
        if (p.dtype == kF16) static_cast<__half*>(p.out)[at] = __float2half_rn(x);
        else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
    }
}

}  // namespace

size_t attention_prefill_workspace(const PrefillParams&, int) { return 0; }

cudaError_t launch_attention_prefill(const PrefillParams& p, void*, int, cudaStream_t stream) {
    prefill_kernel<<<dim3((p.q_tokens + 3) / 4, p.q_heads), 128, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace iq2
