// Internal launch interface between the C ABI of the attention operators (attention_capi.cu) and their kernels.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace iq2 {

// Element types, numbered as IQ2_DTYPE_* of the C ABI; a cache adds int8 (IQ2_KV_INT8).
constexpr int kF32 = 0, kF16 = 1, kBf16 = 2, kInt8 = 3;

// Division of n < 2^31 by a divisor that is known before the launch, as a product: with 2^s the power of two at or above
// the divisor, floor(n / divisor) = (n magic) >> (31 + s) for magic = floor(2^(31 + s) / divisor) + 1.
struct Divisor {
    uint32_t magic;
    int32_t shift;  // s - 1, -1 for a divisor of 1
    static Divisor of(uint32_t divisor) {
        Divisor d{0, -1};
        while (d.shift < 31 && (1ull << (d.shift + 1)) < divisor) ++d.shift;
        if (d.shift >= 0) d.magic = (uint32_t)((1ull << (32 + d.shift)) / divisor + 1);
        return d;
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return shift < 0 ? n : __umulhi(n, magic) >> shift; }
#endif
};

// A paged cache (iq2_kv_cache): k, v [pages][heads][page_size][d], k_scale, v_scale f32 [pages][heads][page_size]
// for int8 codes. Token `pos` of a sequence lives in page block_table[pos / page_size], row pos % page_size.
struct KvCacheView {
    void *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, heads, page_size, d;
    int dtype;
};

// Rows of a [tokens][heads][d] tensor: element strides of the first two dimensions, the last one contiguous.
struct RowsView {
    const void* p;
    int64_t token_stride, head_stride;
};

struct KvWriteParams {
    KvCacheView c;
    RowsView q, k, v;
    const int32_t *slots, *positions;
    const float *cos, *sin;  // [rope_len][d / 2], null: no rotation
    void* q_out;             // [tokens][q_heads][d]
    uint32_t tokens, q_heads, rope_len;
    int dtype, q_out_dtype;
    bool interleaved;
    bool vec;  // every row of the inputs and tables starts on a 16-byte boundary
    Divisor by_heads, by_page;  // set by the launch: heads of a token (q, k and v), tokens of a page
};
cudaError_t launch_kv_write(const KvWriteParams& p, cudaStream_t stream);

struct KvReadParams {
    KvCacheView c;
    const int32_t *block_table, *starts, *cu;  // starts: null = 0
    uint32_t table_width, seqs, total;
    void *k_out, *v_out;  // [total][heads][d]
    int out_dtype;
};
cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream);

struct DecodeParams {
    KvCacheView c;
    RowsView q;  // [batch][q_heads][d]
    void* out;   // [batch][q_heads][d], the dtype of q
    const int32_t *block_table, *seq_lens;
    uint32_t table_width, batch, q_heads;
    int dtype;
    float scale;
};
// Whether the units of a sequence's items can be numbered in 32 bits.
bool attention_decode_fits(const KvCacheView& c, uint32_t table_width, uint32_t q_heads);
size_t attention_decode_workspace(uint32_t batch, uint32_t q_heads, uint32_t kv_heads, uint32_t d, int num_sms);
cudaError_t launch_attention_decode(const DecodeParams& p, void* workspace, int num_sms, cudaStream_t stream);

struct PrefillParams {
    RowsView q, k, v;
    void* out;  // [tokens][q_heads][d]
    const int32_t *cu_q, *cu_k;
    uint32_t seqs, q_tokens, k_tokens, q_heads, kv_heads, d;
    int dtype;  // f16 or bf16
    float scale;
    bool causal;
};
size_t attention_prefill_workspace(const PrefillParams& p, int num_sms);
cudaError_t launch_attention_prefill(const PrefillParams& p, void* workspace, int num_sms, cudaStream_t stream);

}  // namespace iq2
