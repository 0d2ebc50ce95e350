// C ABI of the attention operators (declared in include/candelora_iq2.h): the checks of their arguments, in the order
// dimensions, device, types, layout, buffers; the kernels are in kv_cache.cu, kv_pages.cu, attention_prefill.cu and
// attention_decode.cu.
#include <cinttypes>
#include <cmath>
#include <initializer_list>

#include "../../include/candelora_iq2.h"
#include "attention_internal.h"
#include "iq2xxs_internal.h"

namespace {

using iq2::capi_cuda_fail;
using iq2::capi_fail;

struct Pointer {
    const char* name;
    const void* p;
    size_t align;
};

// Every pointer that is given is device memory of the current device and aligned.
int check_pointers(const char* op, std::initializer_list<Pointer> pointers) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return capi_fail(IQ2_ERR_DEVICE, "%s requires a CUDA device (%s)", op, cudaGetErrorString(e));
    }
    for (const Pointer& q : pointers) {
        if (q.p == nullptr) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: NULL %s", op, q.name);
        cudaPointerAttributes a;
        e = cudaPointerGetAttributes(&a, q.p);
        if (e != cudaSuccess) cudaGetLastError();
        if (e != cudaSuccess || (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) || a.device != dev)
            return capi_fail(IQ2_ERR_DEVICE, "%s: %s is not memory of Cuda(%d)", op, q.name, dev);
        if (reinterpret_cast<uintptr_t>(q.p) % q.align != 0)
            return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: %s is not %zu-byte aligned", op, q.name, q.align);
    }
    return IQ2_OK;
}

bool float_dtype(int t) { return t >= IQ2_DTYPE_F32 && t <= IQ2_DTYPE_BF16; }
size_t size_of(int t) { return t == IQ2_DTYPE_F32 ? 4 : t == IQ2_KV_INT8 ? 1 : 2; }

int check_heads(const char* op, uint32_t q_heads, uint32_t kv_heads, uint32_t d) {
    if (q_heads == 0 || kv_heads == 0 || d == 0) return capi_fail(IQ2_ERR_ZERO_DIM, "%s expects non-zero dimensions", op);
    if (q_heads % kv_heads != 0 || q_heads / kv_heads > 128)
        return capi_fail(IQ2_ERR_UNSUPPORTED, "%s: q_heads=%u is not a multiple (at most 128) of kv_heads=%u", op, q_heads, kv_heads);
    if (d % 16 != 0 || d > 128)
        return capi_fail(IQ2_ERR_UNSUPPORTED, "%s: head_dim=%u is not a multiple of 16, at most 128", op, d);
    return IQ2_OK;
}

int check_cache(const char* op, const iq2_kv_cache* c) {
    if (c == nullptr) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: NULL cache", op);
    int rc = check_heads(op, c->kv_heads, c->kv_heads, c->head_dim);
    if (rc != IQ2_OK) return rc;
    if (c->num_pages == 0 || c->page_size == 0) return capi_fail(IQ2_ERR_ZERO_DIM, "%s expects non-zero dimensions", op);
    if (c->dtype != IQ2_DTYPE_F16 && c->dtype != IQ2_DTYPE_BF16 && c->dtype != IQ2_KV_INT8 && c->dtype != IQ2_KV_INT4)
        return capi_fail(IQ2_ERR_DTYPE, "%s unsupported cache dtype: %d", op, c->dtype);
    if (c->dtype == IQ2_KV_INT4 && c->head_dim % iq2::I4_GROUP != 0)
        return capi_fail(IQ2_ERR_UNSUPPORTED, "%s: head_dim=%u of a 4-bit cache is not a multiple of %u", op, c->head_dim, iq2::I4_GROUP);
    if ((uint64_t)c->num_pages * c->page_size > (uint64_t)INT32_MAX)  // slots are int32
        return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u pages of %u tokens are too large", op, c->num_pages, c->page_size);
    if ((rc = check_pointers(op, {{"cache k", c->k, 16}, {"cache v", c->v, 16}})) != IQ2_OK) return rc;
    if (c->dtype != IQ2_KV_INT8 && c->dtype != IQ2_KV_INT4) return IQ2_OK;
    if (c->dtype == IQ2_KV_INT8) return check_pointers(op, {{"cache k_scale", c->k_scale, 4}, {"cache v_scale", c->v_scale, 4}});
    // (16 bytes of scales at a time)
    return check_pointers(op, {{"cache k_scale", c->k_scale, 16}, {"cache v_scale", c->v_scale, 16}, {"cache k_group", c->k_group, 16},
                               {"cache v_group", c->v_group, 16}});
}

iq2::KvCacheView view(const iq2_kv_cache* c) {
    return {c->k, c->v, c->k_scale, c->v_scale, c->num_pages, c->kv_heads, c->page_size, c->head_dim, c->dtype,
            c->dtype == IQ2_KV_INT4 ? c->k_group : nullptr, c->dtype == IQ2_KV_INT4 ? c->v_group : nullptr};
}
iq2::RowsView view(const iq2_rows& r) { return {r.data, r.token_stride, r.head_stride}; }

bool rows_aligned(const iq2_rows& r, size_t elem, size_t bytes) {
    return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && r.token_stride * (int64_t)elem % (int64_t)bytes == 0 &&
           r.head_stride * (int64_t)elem % (int64_t)bytes == 0;
}

// scale as the kernels take it, or a failure.
int check_scale(const char* op, float scale, uint32_t d, float* out) {
    if (!(scale >= 0.f) || std::isinf(scale)) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: scale is not positive", op);
    *out = scale > 0.f ? scale : (float)(1.0 / std::sqrt((double)d));
    return IQ2_OK;
}

int check_workspace(const char* op, const void* workspace, size_t bytes, size_t need) {
    if (need > 0 && (workspace == nullptr || bytes < need))
        return capi_fail(IQ2_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu", op, need, workspace ? bytes : (size_t)0);
    return need > 0 ? check_pointers(op, {{"workspace", workspace, 256}}) : IQ2_OK;
}

}  // namespace

extern "C" {

static int cache_write(const char* op, const iq2_kv_cache* cache, const iq2_kv_tokens* t, const iq2_head_norms* norms, iq2_stream_t stream) {
    iq2::capi_ok();
    if (t == nullptr) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: NULL tokens", op);
    int rc = check_cache(op, cache);
    if (rc != IQ2_OK) return rc;
    const bool has_q = t->q.data != nullptr, rope = t->cos != nullptr || t->sin != nullptr;
    if (has_q && (rc = check_heads(op, t->q_heads, cache->kv_heads, cache->head_dim)) != IQ2_OK) return rc;
    if (!float_dtype(t->dtype)) return capi_fail(IQ2_ERR_DTYPE, "%s unsupported k/v dtype: %d", op, t->dtype);
    if (has_q && !float_dtype(t->q_out_dtype)) return capi_fail(IQ2_ERR_DTYPE, "%s unsupported q_out dtype: %d", op, t->q_out_dtype);
    const bool norm = norms != nullptr && (norms->q_norm != nullptr || norms->k_norm != nullptr);
    if (norm && !(norms->eps > 0.f && std::isfinite(norms->eps))) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: eps is not positive", op);
    if (norm && norms->q_norm != nullptr && !has_q) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: q_norm goes with q", op);
    if (t->tokens == 0) return IQ2_OK;
    if (t->tokens > (uint32_t)INT32_MAX) return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u tokens are too many", op, t->tokens);
    const size_t e = size_of(t->dtype);
    if ((rc = check_pointers(op, {{"k", t->k.data, e}, {"v", t->v.data, e}, {"slots", t->slots, 4}})) != IQ2_OK) return rc;
    if (has_q && (rc = check_pointers(op, {{"q", t->q.data, e}, {"q_out", t->q_out, 16}})) != IQ2_OK) return rc;
    if (rope) {
        if (t->rope_len == 0) return capi_fail(IQ2_ERR_ZERO_DIM, "%s: empty cos / sin", op);
        if ((rc = check_pointers(op, {{"positions", t->positions, 4}, {"cos", t->cos, 4}, {"sin", t->sin, 4}})) != IQ2_OK) return rc;
    }
    if (norm && norms->q_norm != nullptr && (rc = check_pointers(op, {{"q_norm", norms->q_norm, 4}})) != IQ2_OK) return rc;
    if (norm && norms->k_norm != nullptr && (rc = check_pointers(op, {{"k_norm", norms->k_norm, 4}})) != IQ2_OK) return rc;
    iq2::KvWriteParams p{};
    p.c = view(cache);
    p.k = view(t->k), p.v = view(t->v), p.q = view(t->q);
    p.slots = t->slots, p.positions = t->positions, p.cos = rope ? t->cos : nullptr, p.sin = t->sin, p.q_out = t->q_out;
    p.tokens = t->tokens, p.q_heads = has_q ? t->q_heads : 0, p.rope_len = t->rope_len;
    p.dtype = t->dtype, p.q_out_dtype = t->q_out_dtype, p.interleaved = t->interleaved != 0;
    p.vec_rows = rows_aligned(t->k, e, 16) && rows_aligned(t->v, e, 16) && (!has_q || rows_aligned(t->q, e, 16));
    p.vec = p.vec_rows && (!rope || (reinterpret_cast<uintptr_t>(t->cos) % 16 == 0 && reinterpret_cast<uintptr_t>(t->sin) % 16 == 0));
    if (norm) {
        p.q_norm = norms->q_norm, p.k_norm = norms->k_norm;
        p.q_norm_stride = norms->q_per_head ? cache->head_dim : 0, p.k_norm_stride = norms->k_per_head ? cache->head_dim : 0;
        p.eps = norms->eps, p.inv_d = 1.0 / cache->head_dim;
        p.vec = p.vec && reinterpret_cast<uintptr_t>(p.q_norm) % 16 == 0 && reinterpret_cast<uintptr_t>(p.k_norm) % 16 == 0;
    }
    const cudaError_t err = iq2::launch_kv_write(p, reinterpret_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? IQ2_OK : capi_cuda_fail(op, err);
}

int iq2_kv_cache_write(const iq2_kv_cache* cache, const iq2_kv_tokens* tokens, iq2_stream_t stream) {
    return cache_write("iq2_kv_cache_write", cache, tokens, nullptr, stream);
}

int iq2_kv_cache_write_normed(const iq2_kv_cache* cache, const iq2_kv_tokens* tokens, const iq2_head_norms* norms, iq2_stream_t stream) {
    return cache_write("iq2_kv_cache_write_normed", cache, tokens, norms, stream);
}

int iq2_kv_cache_read(const iq2_kv_cache* cache, const int32_t* block_table, uint32_t table_width, uint32_t sequences,
                      const int32_t* starts, const int32_t* cu_seqlens, uint32_t total, void* k_out, void* v_out,
                      int out_dtype, iq2_stream_t stream) {
    const char* op = "iq2_kv_cache_read";
    iq2::capi_ok();
    int rc = check_cache(op, cache);
    if (rc != IQ2_OK) return rc;
    if (!float_dtype(out_dtype)) return capi_fail(IQ2_ERR_DTYPE, "%s unsupported out dtype: %d", op, out_dtype);
    if (total == 0) return IQ2_OK;
    if (sequences == 0 || table_width == 0) return capi_fail(IQ2_ERR_ZERO_DIM, "%s expects non-zero dimensions", op);
    if (total > (uint32_t)INT32_MAX) return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u tokens are too many", op, total);
    if ((rc = check_pointers(op, {{"block_table", block_table, 4}, {"cu_seqlens", cu_seqlens, 4}, {"k_out", k_out, 16},
                                  {"v_out", v_out, 16}})) != IQ2_OK)
        return rc;
    if (starts != nullptr && (rc = check_pointers(op, {{"starts", starts, 4}})) != IQ2_OK) return rc;
    const iq2::KvReadParams p{view(cache), block_table, starts, cu_seqlens, table_width, sequences, total, k_out, v_out, out_dtype, {}};
    const cudaError_t err = iq2::launch_kv_read(p, reinterpret_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? IQ2_OK : capi_cuda_fail(op, err);
}

int iq2_kv_pages_step(const iq2_kv_pages* pages, const iq2_kv_step* step, iq2_stream_t stream) {
    const char* op = "iq2_kv_pages_step";
    iq2::capi_ok();
    if (pages == nullptr || step == nullptr) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: NULL pages or step", op);
    const iq2_kv_pages& g = *pages;
    const iq2_kv_step& t = *step;
    if (g.sequences == 0 || g.table_width == 0 || g.num_pages == 0 || g.page_size == 0)
        return capi_fail(IQ2_ERR_ZERO_DIM, "%s expects non-zero dimensions", op);
    if (g.sequences > iq2::PAGES_MOST_SEQS)
        return capi_fail(IQ2_ERR_UNSUPPORTED, "%s: %u sequences are more than %u", op, g.sequences, iq2::PAGES_MOST_SEQS);
    if ((uint64_t)g.num_pages * g.page_size > (uint64_t)INT32_MAX)
        return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u pages of %u tokens are too large", op, g.num_pages, g.page_size);
    if (t.total >= (uint32_t)INT32_MAX) return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u tokens are too many", op, t.total);
    int rc = check_pointers(op, {{"block_table", g.block_table, 4}, {"seq_lens", g.seq_lens, 4}, {"free_pages", g.free_pages, 4},
                                 {"free_count", g.free_count, 4}, {"new_lens", t.new_lens, 4}, {"cu_seqlens_q", t.cu_seqlens_q, 4},
                                 {"cu_seqlens_k", t.cu_seqlens_k, 4}, {"granted", t.granted, 4}});
    if (rc == IQ2_OK && t.keep != nullptr) rc = check_pointers(op, {{"keep", t.keep, 4}});
    if (rc == IQ2_OK && t.total > 0) rc = check_pointers(op, {{"slots", t.slots, 4}, {"positions", t.positions, 4}});
    if (rc != IQ2_OK) return rc;
    iq2::PagesParams p{g.block_table, g.seq_lens, g.free_pages, g.free_count, g.sequences, g.table_width, g.num_pages, g.page_size,
                       t.keep, t.new_lens, t.total, t.slots, t.positions, t.cu_seqlens_q, t.cu_seqlens_k, t.granted, {}};
    const cudaError_t err = iq2::launch_kv_pages_step(p, reinterpret_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? IQ2_OK : capi_cuda_fail(op, err);
}

static iq2::PrefillParams prefill_params(const iq2_attention_prompts* t, float scale) {
    return {view(t->q), view(t->k), view(t->v), t->out, t->cu_seqlens_q, t->cu_seqlens_k, t->sequences, t->q_tokens,
            t->k_tokens, t->q_heads, t->kv_heads, t->head_dim, t->dtype, scale, t->causal != 0};
}

size_t iq2_attention_prefill_workspace_size(const iq2_attention_prompts* t) {
    if (t == nullptr || t->q_tokens == 0 || t->sequences == 0 || t->q_heads == 0 || t->kv_heads == 0 || t->head_dim == 0 ||
        t->q_heads % t->kv_heads != 0)
        return 0;
    return iq2::attention_prefill_workspace(prefill_params(t, 1.f), iq2::capi_num_sms());
}

int iq2_attention_prefill(const iq2_attention_prompts* t, void* workspace, size_t workspace_bytes, iq2_stream_t stream) {
    const char* op = "iq2_attention_prefill";
    iq2::capi_ok();
    if (t == nullptr) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: NULL prompts", op);
    int rc = check_heads(op, t->q_heads, t->kv_heads, t->head_dim);
    if (rc != IQ2_OK) return rc;
    if (t->dtype != IQ2_DTYPE_F16 && t->dtype != IQ2_DTYPE_BF16) return capi_fail(IQ2_ERR_DTYPE, "%s unsupported q/k/v dtype: %d", op, t->dtype);
    float scale = 0.f;
    if ((rc = check_scale(op, t->scale, t->head_dim, &scale)) != IQ2_OK) return rc;
    if (t->q_tokens == 0) return IQ2_OK;
    if (t->sequences == 0) return capi_fail(IQ2_ERR_ZERO_DIM, "%s expects non-zero dimensions", op);
    // work items are numbered in 32 bits; tokens, with a tile past the end and an item's cost on top, in 31
    if ((uint64_t)t->q_tokens + t->k_tokens + 1024 > (uint64_t)INT32_MAX ||
        ((uint64_t)t->q_tokens + t->sequences) * t->q_heads > (uint64_t)INT32_MAX ||
        ((uint64_t)t->k_tokens + 1024) * t->kv_heads > (uint64_t)UINT32_MAX)
        return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u queries of %u heads over %u keys are too large", op, t->q_tokens, t->q_heads, t->k_tokens);
    if ((rc = check_pointers(op, {{"q", t->q.data, 16}, {"out", t->out, 16}, {"cu_seqlens_q", t->cu_seqlens_q, 4},
                                  {"cu_seqlens_k", t->cu_seqlens_k, 4}})) != IQ2_OK)
        return rc;
    if (t->k_tokens > 0 && (rc = check_pointers(op, {{"k", t->k.data, 16}, {"v", t->v.data, 16}})) != IQ2_OK) return rc;
    for (const iq2_rows* r : {&t->q, &t->k, &t->v}) {
        const uint32_t tokens = r == &t->q ? t->q_tokens : t->k_tokens, heads = r == &t->q ? t->q_heads : t->kv_heads;
        if ((tokens > 1 && r->token_stride <= 0) || (heads > 1 && r->head_stride <= 0))
            return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: strides are not positive", op);
        if ((tokens > 1 && r->token_stride % 8 != 0) || (heads > 1 && r->head_stride % 8 != 0))
            return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: rows are not 16-byte aligned", op);
    }
    const iq2::PrefillParams p = prefill_params(t, scale);
    const int sms = iq2::capi_num_sms();
    if ((rc = check_workspace(op, workspace, workspace_bytes, iq2::attention_prefill_workspace(p, sms))) != IQ2_OK) return rc;
    const cudaError_t err = iq2::launch_attention_prefill(p, workspace, sms, reinterpret_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? IQ2_OK : capi_cuda_fail(op, err);
}

size_t iq2_attention_decode_workspace_size(const iq2_kv_cache* cache, uint32_t batch, uint32_t q_heads) {
    if (cache == nullptr || cache->kv_heads == 0 || batch == 0 || q_heads == 0 || q_heads % cache->kv_heads != 0) return 0;
    return iq2::attention_decode_workspace(batch, q_heads, cache->kv_heads, cache->head_dim, iq2::capi_num_sms());
}

int iq2_attention_decode(const iq2_kv_cache* cache, const iq2_attention_tokens* t, void* workspace, size_t workspace_bytes,
                         iq2_stream_t stream) {
    const char* op = "iq2_attention_decode";
    iq2::capi_ok();
    if (t == nullptr) return capi_fail(IQ2_ERR_INVALID_ARGUMENT, "%s: NULL tokens", op);
    int rc = check_cache(op, cache);
    if (rc != IQ2_OK) return rc;
    if ((rc = check_heads(op, t->q_heads, cache->kv_heads, cache->head_dim)) != IQ2_OK) return rc;
    if (!float_dtype(t->dtype)) return capi_fail(IQ2_ERR_DTYPE, "%s unsupported q dtype: %d", op, t->dtype);
    float scale = 0.f;
    if ((rc = check_scale(op, t->scale, cache->head_dim, &scale)) != IQ2_OK) return rc;
    if (t->batch == 0) return IQ2_OK;
    if (t->table_width == 0) return capi_fail(IQ2_ERR_ZERO_DIM, "%s expects non-zero dimensions", op);
    if (!iq2::attention_decode_fits(view(cache), t->table_width, t->q_heads))
        return capi_fail(IQ2_ERR_OVERFLOW, "%s: %u pages of %u tokens are too long a sequence", op, t->table_width, cache->page_size);
    if (t->batch > 65535u) return capi_fail(IQ2_ERR_OVERFLOW, "%s: a batch of %u is too large", op, t->batch);
    const size_t e = size_of(t->dtype);
    if ((rc = check_pointers(op, {{"q", t->q.data, e}, {"out", t->out, 16}, {"block_table", t->block_table, 4},
                                  {"seq_lens", t->seq_lens, 4}})) != IQ2_OK)
        return rc;
    const int sms = iq2::capi_num_sms();
    const size_t need = iq2::attention_decode_workspace(t->batch, t->q_heads, cache->kv_heads, cache->head_dim, sms);
    if ((rc = check_workspace(op, workspace, workspace_bytes, need)) != IQ2_OK) return rc;
    const iq2::DecodeParams p{view(cache), view(t->q), t->out, t->block_table, t->seq_lens, t->table_width, t->batch,
                              t->q_heads, t->dtype, scale};
    const cudaError_t err = iq2::launch_attention_decode(p, workspace, sms, reinterpret_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? IQ2_OK : capi_cuda_fail(op, err);
}

}  // extern "C"
