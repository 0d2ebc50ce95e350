// Internal launch interface between the C ABI of the attention operators (attention_capi.cu) and their kernels.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace iq2 {

// Element types, numbered as IQ2_DTYPE_* of the C ABI; a cache adds int8 (IQ2_KV_INT8) and 4-bit codes (IQ2_KV_INT4).
constexpr int kF32 = 0, kF16 = 1, kBf16 = 2, kInt8 = 3, kInt4 = 4;
constexpr uint32_t I4_GROUP = 32;  // elements of a 4-bit row that share a scale

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
// for int8 codes; 4-bit codes, two a byte, have them too and e4m3 scales k_group, v_group [pages][heads][page_size][4] of
// I4_GROUP elements each. Token `pos` of a sequence lives in page block_table[pos / page_size], row pos % page_size.
struct KvCacheView {
    void *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, heads, page_size, d;
    int dtype;
    uint8_t *k_group, *v_group;
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
    bool vec, vec_rows;  // every row of the inputs, tables and norm weights starts on a 16-byte boundary; of the inputs
    const float *q_norm, *k_norm;                 // weights of the heads' norms, null: none
    uint32_t q_norm_stride, k_norm_stride;        // from one head's weights to the next's: 0 or d
    double eps, inv_d;                            // inv_d: 1 / d
    Divisor by_heads, by_page;  // set by the launch: heads of a token (q, k and v), tokens of a page
    Divisor by_q, by_kv;        // heads of q and of k,
    uint32_t blocks_q, blocks_kv;  // and blocks that have rows of them
};
cudaError_t launch_kv_write(const KvWriteParams& p, cudaStream_t stream);

struct KvReadParams {
    KvCacheView c;
    const int32_t *block_table, *starts, *cu;  // starts: null = 0
    uint32_t table_width, seqs, total;
    void *k_out, *v_out;  // [total][heads][d]
    int out_dtype;
    Divisor by_heads;  // set by the launch
};
cudaError_t launch_kv_read(const KvReadParams& p, cudaStream_t stream);

// The pages of a batch's sequences (iq2_kv_pages) and a step of them (iq2_kv_step).
struct PagesParams {
    int32_t *table, *lens, *free_pages, *free_count;
    uint32_t seqs, width, pages, page_size;
    const int32_t *keep, *new_lens;  // keep: null = all
    uint32_t total;
    int32_t *slots, *positions, *cu_q, *cu_k, *granted;
    Divisor by_page;  // set by the launch
};
constexpr uint32_t PAGES_MOST_SEQS = 8192;
cudaError_t launch_kv_pages_step(const PagesParams& p, cudaStream_t stream);

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
cudaError_t launch_attention_decode_int4(const DecodeParams& p, void* workspace, int num_sms, cudaStream_t stream);

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
