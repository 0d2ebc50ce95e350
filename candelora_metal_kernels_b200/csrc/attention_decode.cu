// Attention of one new token a sequence over the paged cache:
//     s_j = scale q . k_j,  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)   over the sequence's tokens j < length.
//
// Bound by HBM: every cached byte is read once and feeds 2 G multiply-adds (G query heads share a key head). An item is
// one sequence, one key head and up to eight of its query heads; the items' lengths, cut into units of 8 warps x TOK
// tokens, form one line of work that the thread blocks (one an SM) take equal, contiguous parts of, whatever the lengths
// are. The lengths are on the device, so every block sums them up itself. A part that is not a whole item leaves its
// (max, sum, o) in the workspace, and join_kernel adds the parts of an item up in the order of the blocks.
//
// Inside a block each warp streams its own TOK tokens (K and V rows) through a ring of cp.async stages, across the items'
// ends, and computes with mma.sync m16n8k16 (used as a dot-product engine: 16-bit products, f32 sums):
//   S = Q K^T   rows 0-7: the high pieces of eight heads' q, rows 8-15: the low pieces; the two rows' sum is s
//   O = P V     rows 0-7: the high pieces of p, rows 8-15: the low pieces
// so the second piece, which gives f32 activations 22 bits (f16 pieces) or 16 (bf16 pieces), costs no instruction.
//   * bf16 caches take bf16 pieces (their range); f16 and int8 caches f16 pieces of q / 2^e, 2^e the power of two above
//     the head's largest |q|: pieces of at least 22 bits at any magnitude.
//   * int8 codes become f16 by one byte permute (1024 + code + 128, exact) and one subtraction a pair; the key scale
//     multiplies s. The value scale w_j multiplies p, with the running maximum taken over s_j + log2 w_j so that p w stays
//     at most about 1, the range of its f16 pieces; the sum of p itself stays f32.
// The maxima, sums, s, p and o are f32.
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

#include <algorithm>

namespace iq2 {

namespace {

constexpr int AD_WARPS = 8, AD_THREADS = AD_WARPS * 32, AD_STAGES = 3;
constexpr int AD_HEADS = 8;                     // query heads of an item
constexpr float AD_MIN_SCALE = 7.88860905e-31f;  // 2^-100: the smallest value scale the maximum goes by
constexpr float LOG2E = 1.44269504f;

enum CacheKind { CK_F16, CK_BF16, CK_INT8 };

template <int DP, int KIND>
struct DecodeShape {
    static constexpr int ESIZE = KIND == CK_INT8 ? 1 : 2;
    static constexpr int TOK = KIND == CK_INT8 ? 32 : 16;  // tokens of a warp's stage: 8 KB of K and V at DP = 128
    static constexpr int UNIT = TOK * AD_WARPS;
    static constexpr int ROW = DP * ESIZE;                 // bytes of a padded K or V row
    static constexpr int CHUNKS = ROW / 16;
    static constexpr int SCALES = KIND == CK_INT8 ? TOK * 8 : 0;
    static constexpr int STAGE = 2 * TOK * ROW + SCALES;
    static constexpr int RING = AD_STAGES * STAGE;
    static constexpr int Q_BYTES = 2 * AD_HEADS * DP * 2;
    static constexpr int PART = AD_HEADS * (DP + 2);       // floats of one (o, max, sum)
    static constexpr int SMEM = AD_WARPS * RING + Q_BYTES + 4 * PART * 4 + AD_HEADS * 4;
};

// What join_kernel's block of the same number has to join: the parts of blocks c0 to c1 of one item, block c0's being its
// part number `slot` (0: its first, 1: its last), the others' their first. c1 = 0: nothing.
struct JoinRecord {
    uint32_t b, item, c0, c1, slot;
};
inline size_t records_bytes(uint32_t blocks) { return (blocks * sizeof(JoinRecord) + 255) / 256 * 256; }

__device__ __forceinline__ uint32_t seq_len(const DecodeParams& p, uint32_t b) {
    const uint64_t most = min((uint64_t)p.table_width * p.c.page_size, (uint64_t)0x7FFFFFFF);
    return (uint32_t)min((uint64_t)max(__ldg(p.seq_lens + b), 0), most);
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

// Four 8 x 8 tiles of 16-bit elements, lane l giving the address of row l % 8 of tile l / 8.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// Two bytes of biased codes (code + 128) -> two f16 codes: 0x6400 | byte is 1024 + byte.
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t biased, uint32_t sel) {
    const uint32_t u = prmt(biased, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Byte offset of 16-byte chunk c of row r in a K or V stage. The readers of a phase must meet eight different 16-byte
// columns of the 128-byte bank line:
//   ldmatrix (16-bit K and V, int8 V) reads eight rows of one chunk: column ^ row;
//   int8 K is read by plain 16-byte loads, two rows of four chunks at a time: odd rows swap the halves of their line.
// 64-byte rows (int8, DP = 64) share a line in pairs: ldmatrix needs column ^ (row / 2) inside each half.
template <int CHUNKS, bool PLAIN>
__device__ __forceinline__ uint32_t stage_offset(uint32_t r, uint32_t c) {
    if (CHUNKS == 4) return r * 64 + (PLAIN ? c : c ^ ((r >> 1) & 3)) * 16;
    return (r * CHUNKS + (PLAIN ? c ^ ((r & 1) * 4) : c ^ (r & 7))) * 16;
}

// The line of work from one unit on: the item it is in and the tokens [t0, t1) of that item up to the end of the part.
struct Cursor {
    uint64_t unit, end;
    uint32_t b, item, len, units;  // the sequence, its item (key head, group of query heads), tokens and units an item
    uint32_t k;                    // first unit of the item in the part
    uint32_t n;                    // units of the item in the part
    __device__ __forceinline__ void cut() { n = (uint32_t)min((uint64_t)(units - k), end - unit); }
    __device__ __forceinline__ bool done() const { return unit >= end; }
    template <int UNIT>
    __device__ __forceinline__ void next(const DecodeParams& p, uint32_t items) {
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
            units = (len + UNIT - 1) / UNIT;
        }
        cut();
    }
};

template <int DP, int KIND>
__global__ void __launch_bounds__(AD_THREADS, 1)
    decode_kernel(const DecodeParams p, float* __restrict__ parts, JoinRecord* __restrict__ records, uint32_t chunks_of_heads) {
    using S = DecodeShape<DP, KIND>;
    constexpr bool BF = KIND == CK_BF16;
    constexpr int TOK = S::TOK, UNIT = S::UNIT, NT = DP / 8, KS = DP / 16, ST = TOK / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const q_smem = smem + AD_WARPS * S::RING;                     // [8 heads][2 pieces][DP] 16-bit
    float* const part_smem = reinterpret_cast<float*>(q_smem + S::Q_BYTES);  // 4 x (o, max, sum)
    float* const q_factor = part_smem + 4 * S::PART;                       // [8] scale log2(e) 2^e
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint32_t d = p.c.d, group = p.q_heads / p.c.heads, items = p.c.heads * chunks_of_heads;
    pdl_launch_dependents();

    // ---- this block's part of the line (every warp works it out for itself) ----
    // the ring starts as zeros: chunks past head_dim are never copied, and the matrix instructions read them
    if (d < DP)
        for (uint32_t i = lane; i < S::RING / 16; i += 32) *reinterpret_cast<uint4*>(smem + warp * S::RING + i * 16) = make_uint4(0, 0, 0, 0);
    uint64_t units = 0;
    for (uint32_t b = lane; b < p.batch; b += 32) units += (seq_len(p, b) + UNIT - 1) / UNIT;
    for (int o = 16; o > 0; o /= 2) units += __shfl_xor_sync(0xFFFFFFFFu, units, o);
    units *= items;
    const Deal deal(units, gridDim.x);
    const uint64_t u0 = deal.start(blockIdx.x), u1 = deal.start(blockIdx.x + 1);
    // sequences of length 0: zeros
    for (uint32_t b = blockIdx.x; b < p.batch; b += gridDim.x)
        if (seq_len(p, b) == 0)
            for (uint32_t i = threadIdx.x; i < p.q_heads * d; i += AD_THREADS)
                store_elem(p.out, (int64_t)b * p.q_heads * d + i, p.dtype, 0.f);
    if (u0 >= u1) {
        if (threadIdx.x == 0) records[blockIdx.x].c1 = 0;
        return;
    }
    Cursor cur{};
    uint64_t before = 0;  // units of the sequences before
    for (uint32_t b0 = 0;; b0 += 32) {
        if (b0 >= p.batch) return;  // (not reached while the lengths stay as they were)
        const uint32_t len = b0 + lane < p.batch ? seq_len(p, b0 + lane) : 0u, own = (len + UNIT - 1) / UNIT;
        uint64_t upto = (uint64_t)own * items;
        for (int o = 1; o < 32; o *= 2) {
            const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= (uint32_t)o) upto += x;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + upto > u0);
        if (hit != 0) {
            const int at = __ffs(hit) - 1;
            cur.b = b0 + at;
            cur.len = __shfl_sync(0xFFFFFFFFu, len, at), cur.units = __shfl_sync(0xFFFFFFFFu, own, at);
            const uint32_t rest = (uint32_t)(u0 - before - __shfl_sync(0xFFFFFFFFu, upto - (uint64_t)own * items, at));
            cur.item = rest / cur.units, cur.k = rest % cur.units;
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    cur.unit = u0, cur.end = u1;
    cur.cut();
    Cursor pre = cur;
    if (threadIdx.x == 0) {
        // the first block whose part begins inside an item joins it
        const uint64_t unit0 = u0 - cur.k;
        const uint32_t c0 = cur.k > 0 ? deal.block_of(unit0) : blockIdx.x;
        JoinRecord r{cur.b, cur.item, c0, 0, 0};
        if (c0 + 1 == blockIdx.x) r.c1 = deal.block_of(unit0 + cur.units - 1), r.slot = deal.start(c0) == unit0 ? 0 : 1;
        records[blockIdx.x] = r;
    }

    // ---- the copies: tile `i` (TOK tokens) of pre's piece of an item, one page lookup ahead ----
    uint8_t* const ring = smem + warp * S::RING;
    const uint32_t ring_u32 = smem_u32(ring);
    if (d < DP) __syncwarp();
    uint32_t pre_i = warp, pre_page = 0;  // the tile to copy next and this lane's token's page number
    auto pre_tokens = [&](const Cursor& c) { return min(c.len, (c.k + c.n) * UNIT) - c.k * UNIT; };
    auto find_tile = [&]() {  // the next tile of this warp, and its page numbers under way
        while (!pre.done() && pre_i * TOK >= pre_tokens(pre)) {
            pre.next<UNIT>(p, items);
            pre_i = warp;
        }
        if (pre.done()) return;
        const uint32_t tok = pre.k * UNIT + pre_i * TOK + lane;
        if (lane < TOK && tok < pre.len)
            pre_page = (uint32_t)__ldg(p.block_table + (int64_t)pre.b * p.table_width + tok / p.c.page_size);
    };
    auto copy_tile = [&](uint32_t stage) {
        if (!pre.done()) {
            const uint32_t tok = pre.k * UNIT + pre_i * TOK + lane, h = pre.item / chunks_of_heads;
            const bool valid = lane < TOK && tok < pre.len && pre_page < p.c.pages;
            const int64_t row = valid ? ((int64_t)pre_page * p.c.heads + h) * p.c.page_size + tok % p.c.page_size : -1;
            const uint32_t dst = ring_u32 + stage * S::STAGE;
            const uint32_t c = lane % S::CHUNKS, r0 = lane / S::CHUNKS;
            const uint32_t row_bytes = d * S::ESIZE;
            const bool inside = c * 16 < row_bytes;
#pragma unroll
            for (int i = 0; i < TOK * S::CHUNKS / 32; ++i) {
                const uint32_t r = r0 + i * (32 / S::CHUNKS);
                const int64_t src = __shfl_sync(0xFFFFFFFFu, row, r);
                const int64_t off = src < 0 ? 0 : src * row_bytes + c * 16;
                if (inside) {  // a token that takes no part is zeros: what its page holds cannot matter
                    cp_async_16(dst + stage_offset<S::CHUNKS, KIND == CK_INT8>(r, c), static_cast<const uint8_t*>(p.c.k) + off, src < 0 ? 0 : 16);
                    cp_async_16(dst + TOK * S::ROW + stage_offset<S::CHUNKS, false>(r, c), static_cast<const uint8_t*>(p.c.v) + off, src < 0 ? 0 : 16);
                }
            }
            if (KIND == CK_INT8) {
                const int64_t off = row < 0 ? 0 : row;
                cp_async_4(dst + 2 * TOK * S::ROW + lane * 4, p.c.k_scale + off, row < 0 ? 0 : 4);
                cp_async_4(dst + 2 * TOK * S::ROW + TOK * 4 + lane * 4, p.c.v_scale + off, row < 0 ? 0 : 4);
            }
            pre_i += AD_WARPS;
        }
        cp_async_commit();
    };
    // Tokens whose page is outside the cache are rare and take no part: a bit for each token of a stage.
    uint32_t present[AD_STAGES] = {};
    auto copy_and_find = [&](int stage) {
        if (!pre.done()) {
            const uint32_t tok = pre.k * UNIT + pre_i * TOK + lane;
            const uint32_t bits = __ballot_sync(0xFFFFFFFFu, lane < TOK && tok < pre.len && pre_page < p.c.pages);
#pragma unroll
            for (int s = 0; s < AD_STAGES; ++s)
                if (s == stage) present[s] = bits;
        }
        copy_tile(stage);
        find_tile();
    };
    // q of an item, a warp a head: loaded while the copies before it are under way
    float q_next[DP / 32];
    auto load_q = [&](const Cursor& c) {
        const uint32_t kv = c.item / chunks_of_heads, h0 = kv * group + (c.item % chunks_of_heads) * AD_HEADS;
        const bool has = warp < min((uint32_t)AD_HEADS, (kv + 1) * group - h0);
        const int64_t at = (int64_t)c.b * p.q.token_stride + (int64_t)(h0 + warp) * p.q.head_stride;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) q_next[i] = has && lane + i * 32 < d ? load_elem(p.q.p, at + lane + i * 32, p.dtype) : 0.f;
    };
    find_tile();
    load_q(cur);
    for (int s = 0; s < AD_STAGES - 1; ++s) copy_and_find(s);
    int stage = 0;

    while (!cur.done()) {
        // ---- q of the item: two 16-bit pieces of each head ----
        const uint32_t kv_head = cur.item / chunks_of_heads, head0 = kv_head * group + (cur.item % chunks_of_heads) * AD_HEADS;
        const uint32_t heads = min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0);
        {
            float x[DP / 32], top = 0.f;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) x[i] = q_next[i], top = fmaxf(top, fabsf(x[i]));
            float up = 1.f, down = 1.f;  // 2^e and 2^-e
            if (!BF) {
                for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                const int e = min(max((int)(__float_as_uint(top) >> 23) - 126, -125), 126);
                if (top > 0.f && top < INFINITY) up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
            }
            __nv_bfloat16* const qb = reinterpret_cast<__nv_bfloat16*>(q_smem) + warp * 2 * DP;
            __half* const qh = reinterpret_cast<__half*>(q_smem) + warp * 2 * DP;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const float y = x[i] * down;
                if (BF) {
                    qb[lane + i * 32] = __float2bfloat16_rn(y);
                    qb[DP + lane + i * 32] = __float2bfloat16_rn(y - __bfloat162float(qb[lane + i * 32]));
                } else {
                    qh[lane + i * 32] = __float2half_rn(y);
                    qh[DP + lane + i * 32] = __float2half_rn(y - __half2float(qh[lane + i * 32]));
                }
            }
            if (lane == 0) q_factor[warp] = p.scale * LOG2E * up;
        }
        __syncthreads();
        // A fragments of S: k index 16 ks + 2t (+1, +8, +9). For int8 the k index is a relabelled dimension, so that a
        // thread's codes of four k steps are 16 consecutive bytes of its row.
        uint32_t qa[KS][4];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint32_t lo = KIND == CK_INT8 ? (t + 4 * (ks / 4)) * 16 + (ks % 4) * 4 : ks * 16 + t * 2;
            const uint32_t hi = KIND == CK_INT8 ? lo + 2 : lo + 8;
            const uint32_t* const row = reinterpret_cast<const uint32_t*>(q_smem + g * 4 * DP);
            qa[ks][0] = row[lo / 2], qa[ks][1] = row[DP / 2 + lo / 2];
            qa[ks][2] = row[hi / 2], qa[ks][3] = row[DP / 2 + hi / 2];
        }
        const float factor = q_factor[g];
        float o[NT][4], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

        const uint32_t tokens = pre_tokens(cur);
        for (uint32_t i = warp; i * TOK < tokens; i += AD_WARPS) {
            cp_async_wait<AD_STAGES - 2>();
            __syncwarp();
            const uint32_t k_at = ring_u32 + stage * S::STAGE, v_at = k_at + TOK * S::ROW;
            uint32_t here = 0;
#pragma unroll
            for (int s = 0; s < AD_STAGES; ++s)
                if (s == stage) here = present[s];
            copy_and_find(stage == 0 ? AD_STAGES - 1 : stage - 1);  // the stage the last tile freed

            float s[ST][4];
#pragma unroll
            for (int n = 0; n < ST; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
            if (KIND == CK_INT8) {
#pragma unroll
                for (int n = 0; n < ST; ++n)
#pragma unroll
                    for (int q4 = 0; q4 < KS / 4; ++q4) {
                        const uint4 w = ld_shared_v4<0>(k_at + stage_offset<S::CHUNKS, true>(n * 8 + g, t + 4 * q4));
                        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t u = x[j] ^ 0x80808080u;
                            mma16816<BF>(s[n], qa[q4 * 4 + j], codes_to_half2(u, 0x4140u), codes_to_half2(u, 0x4342u));
                        }
                    }
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t r[4];  // tokens 0-7 chunks 2 ks, 2 ks + 1, then tokens 8-15
                    ldmatrix4(r, k_at + stage_offset<S::CHUNKS, false>((lane / 16) * 8 + lane % 8, ks * 2 + (lane / 8) % 2));
                    mma16816<BF>(s[0], qa[ks], r[0], r[1]);
                    mma16816<BF>(s[1], qa[ks], r[2], r[3]);
                }
            }

            // p = 2^(s - m), this thread's tokens 8 n + 2 t, + 1 of head g
            float x[ST][2], vs[ST][2], top = -INFINITY;
#pragma unroll
            for (int n = 0; n < ST; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t r = n * 8 + t * 2 + j;
                    float y = (s[n][j] + s[n][j + 2]) * factor, rank = 0.f;
                    vs[n][j] = 1.f;
                    if (KIND == CK_INT8) {
                        const float* const sc = reinterpret_cast<const float*>(ring + stage * S::STAGE + 2 * TOK * S::ROW);
                        y *= sc[r];
                        vs[n][j] = sc[TOK + r];
                        rank = __log2f(fmaxf(vs[n][j], AD_MIN_SCALE));
                    }
                    x[n][j] = (here >> r) & 1u ? y : -INFINITY;
                    top = fmaxf(top, x[n][j] + rank);
                }
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            if (__any_sync(0xFFFFFFFFu, top > m)) {
                const float next = fmaxf(m, top), keep = next == -INFINITY ? 1.f : exp2_approx(m - next);
                m = next;
                l *= keep;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[n][j] *= keep;
            }
            const float base = m == -INFINITY ? 0.f : m;
            uint32_t pa[TOK / 16][4];
#pragma unroll
            for (int n = 0; n < ST; ++n) {
                const float e0 = exp2_approx(x[n][0] - base), e1 = exp2_approx(x[n][1] - base);
                l += e0 + e1;
                const float w0 = e0 * vs[n][0], w1 = e1 * vs[n][1];
                const uint32_t high = pack_pair<BF>(w0, w1);
                const float2 back = unpack_pair<BF>(high);
                pa[n / 2][(n % 2) * 2] = high;
                pa[n / 2][(n % 2) * 2 + 1] = pack_pair<BF>(w0 - back.x, w1 - back.y);
            }

            if (KIND == CK_INT8) {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; ++c) {
                    uint32_t r[4];  // chunk c of tokens 0-7, 8-15, 16-23, 24-31; each word: dimensions 2g, 2g + 1 of two tokens
                    ldmatrix4_trans(r, v_at + stage_offset<S::CHUNKS, false>(lane, c));
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[j] ^= 0x80808080u;
#pragma unroll
                    for (int ks = 0; ks < TOK / 16; ++ks) {
                        mma16816<BF>(o[c * 2], pa[ks], codes_to_half2(r[ks * 2], 0x4240u), codes_to_half2(r[ks * 2 + 1], 0x4240u));
                        mma16816<BF>(o[c * 2 + 1], pa[ks], codes_to_half2(r[ks * 2], 0x4341u), codes_to_half2(r[ks * 2 + 1], 0x4341u));
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c += 2) {
                    uint32_t r[4];  // chunk c of tokens 0-7 and 8-15, then chunk c + 1
                    ldmatrix4_trans(r, v_at + stage_offset<S::CHUNKS, false>(lane % 16, c + lane / 16));
                    mma16816<BF>(o[c], pa[0], r[0], r[1]);
                    mma16816<BF>(o[c + 1], pa[0], r[2], r[3]);
                }
            }
            __syncwarp();
            stage = stage == AD_STAGES - 1 ? 0 : stage + 1;
        }
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);

        Cursor next = cur;
        next.next<UNIT>(p, items);
        if (!next.done()) load_q(next);

        // ---- the eight warps' (o, m, l) of the item, through four slots of shared memory ----
        auto put = [&](float* slot) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // int8: accumulator columns are the even and odd dimensions of a 16-dimension chunk
                const uint32_t e0 = KIND == CK_INT8 ? (n / 2) * 16 + n % 2 + t * 4 : n * 8 + t * 2, e1 = e0 + (KIND == CK_INT8 ? 2 : 1);
                slot[g * DP + e0] = o[n][0] + o[n][2];
                slot[g * DP + e1] = o[n][1] + o[n][3];
            }
            if (t == 0) slot[AD_HEADS * DP + g] = m, slot[AD_HEADS * DP + AD_HEADS + g] = l;
        };
        if (warp >= 4) put(part_smem + (warp - 4) * S::PART);
        __syncthreads();
        if (warp < 4) {
            float* const slot = part_smem + warp * S::PART;
            const float m2 = slot[AD_HEADS * DP + g], l2 = slot[AD_HEADS * DP + AD_HEADS + g];
            const float both = fmaxf(m, m2), a = both == -INFINITY ? 0.f : exp2_approx(m - both), b = both == -INFINITY ? 0.f : exp2_approx(m2 - both);
            l = l * a + l2 * b, m = both;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t e0 = KIND == CK_INT8 ? (n / 2) * 16 + n % 2 + t * 4 : n * 8 + t * 2, e1 = e0 + (KIND == CK_INT8 ? 2 : 1);
                o[n][0] = (o[n][0] + o[n][2]) * a + slot[g * DP + e0] * b, o[n][2] = 0.f;
                o[n][1] = (o[n][1] + o[n][3]) * a + slot[g * DP + e1] * b, o[n][3] = 0.f;
            }
            __syncwarp();
            put(slot);
        }
        __syncthreads();
        {
            const bool whole = cur.k == 0 && cur.n == cur.units;
            float* const part = parts + ((uint64_t)blockIdx.x * 2 + (cur.unit == u0 ? 0 : 1)) * S::PART;
            const uint32_t h = warp;  // a warp a head
            float mx = -INFINITY, w[4], sum = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s) mx = fmaxf(mx, part_smem[s * S::PART + AD_HEADS * DP + h]);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                w[s] = mx == -INFINITY ? 0.f : exp2_approx(part_smem[s * S::PART + AD_HEADS * DP + h] - mx);
                sum += part_smem[s * S::PART + AD_HEADS * DP + AD_HEADS + h] * w[s];
            }
            if (h < heads) {
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) {
                    const uint32_t e = lane + i * 32;
                    float y = 0.f;
#pragma unroll
                    for (int s = 0; s < 4; ++s) y += part_smem[s * S::PART + h * DP + e] * w[s];
                    if (!whole) part[h * DP + e] = y;
                    else if (e < d)
                        store_elem(p.out, ((int64_t)cur.b * p.q_heads + head0 + h) * d + e, p.dtype, sum == 0.f ? 0.f : y / sum);
                }
                if (!whole && lane == 0) part[AD_HEADS * DP + h] = mx, part[AD_HEADS * DP + AD_HEADS + h] = sum;
            }
        }
        cur = next;
        if (!cur.done()) __syncthreads();  // the slots and q are written again
    }
    cp_async_wait<0>();
}

// The parts of an item that several blocks had: (o, m, l) = sum over them of 2^(m_c - max) (o_c, l_c), in the blocks'
// order. A block a record, a warp a head.
template <int DP>
__global__ void __launch_bounds__(AD_THREADS, 1)
    join_kernel(const DecodeParams p, const float* __restrict__ parts, const JoinRecord* __restrict__ records, uint32_t chunks_of_heads) {
    constexpr int PART = AD_HEADS * (DP + 2);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_wait();
    const JoinRecord r = records[blockIdx.x];
    if (r.c1 == 0) return;
    const uint32_t d = p.c.d, group = p.q_heads / p.c.heads;
    const uint32_t kv_head = r.item / chunks_of_heads, head0 = kv_head * group + (r.item % chunks_of_heads) * AD_HEADS;
    if (warp >= min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0)) return;
    auto slot = [&](uint32_t c) { return parts + ((uint64_t)c * 2 + (c == r.c0 ? r.slot : 0)) * PART; };
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
#pragma unroll 4
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

template <int DP, int KIND>
cudaError_t launch(const DecodeParams& p, uint8_t* workspace, uint32_t blocks, cudaStream_t stream) {
    using S = DecodeShape<DP, KIND>;
    const uint32_t chunks = (p.q_heads / p.c.heads + AD_HEADS - 1) / AD_HEADS;
    JoinRecord* const records = reinterpret_cast<JoinRecord*>(workspace);
    float* const parts = reinterpret_cast<float*>(workspace + records_bytes(blocks));
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<DP, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return e;
    // (the second kernel keeps the first one's split of shared memory: changing it would drain the SMs twice a call)
    e = cudaFuncSetAttribute(join_kernel<DP>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    decode_kernel<DP, KIND><<<blocks, AD_THREADS, S::SMEM, stream>>>(p, parts, records, chunks);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(AD_THREADS);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<DP>, p, static_cast<const float*>(parts),
                              static_cast<const JoinRecord*>(records), chunks);
}

template <int DP>
cudaError_t launch_kind(const DecodeParams& p, uint8_t* ws, uint32_t blocks, cudaStream_t stream) {
    if (p.c.dtype == kInt8) return launch<DP, CK_INT8>(p, ws, blocks, stream);
    if (p.c.dtype == kBf16) return launch<DP, CK_BF16>(p, ws, blocks, stream);
    return launch<DP, CK_F16>(p, ws, blocks, stream);
}

}  // namespace

size_t attention_decode_workspace(uint32_t, uint32_t, uint32_t, uint32_t d, int num_sms) {
    return records_bytes(num_sms) + (size_t)num_sms * 2 * AD_HEADS * ((d > 64 ? 128 : 64) + 2) * sizeof(float);
}

cudaError_t launch_attention_decode(const DecodeParams& p, void* workspace, int num_sms, cudaStream_t stream) {
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    return p.c.d > 64 ? launch_kind<128>(p, ws, num_sms, stream) : launch_kind<64>(p, ws, num_sms, stream);
}

}  // namespace iq2
