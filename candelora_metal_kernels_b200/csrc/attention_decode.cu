// Attention of one new token a sequence over the paged cache:
//     s_j = scale q . k_j,  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)   over the sequence's tokens j < length.
//
// Bound by HBM: every cached byte is read once and feeds 2 G multiply-adds (G query heads share a key head). An item is
// one sequence, one key head and up to eight of its query heads; the items, each as long as its tokens in units of 4 TOK
// and AD_ITEM_COST more, form one line of work that the thread blocks (one an SM) take equal, contiguous parts of, whatever
// the lengths are. The lengths are on the device, so every block sums them up itself. A part that is not a whole item leaves its
// (max, sum, o) in the workspace, and join_kernel adds the parts of an item up in the order of the blocks.
//
// Inside a block each warp streams its own TOK tokens (K and V rows) through a ring of cp.async stages, across the items'
// ends, and computes with mma.sync m16n8k16 (used as a dot-product engine: 16-bit products, f32 sums):
//   S = Q K^T   rows 0-7: the high pieces of eight heads' q, rows 8-15: the low pieces; the two rows' sum is s
//   O = P V     rows 0-7: the high pieces of p, rows 8-15: the low pieces
// so the second piece, which gives f32 activations 22 bits (f16 pieces) or 16 (bf16 pieces), costs no instruction.
//   * bf16 caches take bf16 pieces (their range); f16 and int8 caches f16 pieces of q / 2^e, 2^e the power of two above
//     the head's largest |q|. A low piece is held times 2^11, which the sum of the two rows takes off, so that it is not
//     held among f16's smallest numbers; and the largest p is 2^7 to 2^15. So q keeps 22 bits down to 2^-14 of the head's
//     largest and p (times its value scale) down to 2^-21 of the largest, and what is smaller is off by no more than 2^-36 and
//     2^-43 of those: a token that takes all of the weight leaves the others' digits as they are (2^-25 without the two).
//   * A bf16 cache under f32 activations takes a third piece (a second pair of products), or p would end at 2^-17.
//   * int8 codes: the byte code + 128 with a zero byte above it is the f16 number (code + 128) 2^-24 (a subnormal, exact and
//     full speed in the matrix instructions), so a pair costs half an exclusive or and one byte permute. The 128s are taken
//     off as products with the constant 128 2^-24: S starts from minus them, O has them as one more column of P V. The
//     sums are some four times as large for it (hundreds of times where one channel of q stands far above the others and
//     the keys have little there), which the 2^-8 of bf16 activations hides. For f32 and f16 ones (8e-6 against 1e-6 over
//     the whole) a byte with 0x64 above it is 1024 + code + 128, and a subtraction makes it the code itself: 51.0 instead of
//     49.2 us for 100001 tokens.
//   * The key scale multiplies s, the value scale multiplies p, and a power of two of the head keeps these products to the range of
//     f16 (attention_decode.cuh). The reference m of a head's exponents moves when one of them, or p, has grown past 2^15 (16-bit
//     caches: when p has grown by more than 2^8).
// The maxima, sums, s, p and o are f32.
//
// Measured (8 key heads, 128 elements): 128 sequences of up to 4096 tokens, bf16 cache, 214 us: 6260 GB/s, 0.96 of the copy
// rate; one of 100001 tokens, int8 cache and 8 query heads a key head, 49 us: 4300 GB/s, of which about 8 us are start,
// merge of the warps and join, and in the stream the widening of the codes binds as well (issue slots 50 % used); 16 of up to
// 2048, int8, f32 q, 22 us, of which the stream is 7; one of 333 tokens 9.6 us, latencies one after another. 16 of up to
// 2048, f32 q: 24.0 us over an f16 cache, 27.7 over a bf16 one (the third piece); 64 of up to 4096, int8, bf16 q: 91.1 us with
// pages of 64 tokens, 103 with 16 or 48 (a tile of 32 tokens then lies in several pages, and each row is looked up). The parts added
// up inside this kernel (by the block that finishes last) instead of by a dependent launch: 11.4 and 53.8 us for the
// one of 333 and the one of 100001 tokens.
#include "attention_decode.cuh"

namespace iq2 {

namespace {

constexpr int AD_WARPS = 8, AD_THREADS = AD_WARPS * 32, AD_STAGES = 3;
// 16-bit caches: the power of two that p has at the reference, and how far it may grow before that moves.
template <bool BF>
constexpr float AD_TOP = BF ? 0.f : 7.f;
template <bool BF>
constexpr float AD_LAZY = BF ? 256.f : 32768.f;
template <bool BF>
constexpr float AD_LOW = BF ? 1.f : 2048.f;      // what low pieces are held times
constexpr uint32_t CODE_ZERO = 0x00800080u;      // two codes of 0 as f16: 128 2^-24
constexpr float CODE_UNIT = 16777216.f;          // 2^24
enum CacheKind { CK_F16, CK_BF16, CK_INT8 };

template <int DP, int KIND, bool WIDE>
struct DecodeShape {
    static constexpr int PIECES = WIDE && KIND == CK_BF16 ? 3 : 2;
    static constexpr int ESIZE = KIND == CK_INT8 ? 1 : 2;
    static constexpr int TOK = KIND == CK_INT8 ? 32 : 16;  // tokens of a warp's stage: 8 KB of K and V at DP = 128
    static constexpr int UNIT = TOK * 4;                   // tokens that the line of work is cut at: 32 KB at DP = 128
    static constexpr int ROW = DP * ESIZE;                 // bytes of a padded K or V row
    static constexpr int CHUNKS = ROW / 16;
    static constexpr int SCALES = KIND == CK_INT8 ? TOK * 8 : 0;
    static constexpr int STAGE = 2 * TOK * ROW + SCALES;
    static constexpr int RING = AD_STAGES * STAGE;
    static constexpr int Q_BYTES = PIECES * AD_HEADS * DP * 2;
    static constexpr int PART = AD_HEADS * (DP + 2);       // floats of one (o, max, sum)
    static constexpr int SMEM = AD_WARPS * RING + Q_BYTES + 4 * PART * 4 + AD_HEADS * 4;
};

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

// Two bytes of codes + 128 as f16: (code + 128) 2^-24, or the codes themselves.
template <bool SHIFTED>
__device__ __forceinline__ uint32_t code_pair(uint32_t bytes, uint32_t sel) {
    if (SHIFTED) return prmt(bytes, 0u, sel);
    const uint32_t u = prmt(bytes, 0x64646464u, sel);
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

template <int DP, int KIND, bool WIDE>
__global__ void __launch_bounds__(AD_THREADS, 1)
    decode_kernel(const __grid_constant__ DecodeArgs a) {
    using S = DecodeShape<DP, KIND, WIDE>;
    // WIDE: f32 activations, and f16 ones over int8 codes
    constexpr bool BF = KIND == CK_BF16, I8 = KIND == CK_INT8, THIRD = BF && WIDE, SHIFTED = I8 && !WIDE;
    constexpr int TOK = S::TOK, UNIT = S::UNIT, NT = DP / 8, KS = DP / 16, ST = TOK / 8;
    constexpr uint32_t ALL = TOK == 32 ? 0xFFFFFFFFu : (1u << TOK) - 1;
    const DecodeParams& p = a.p;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const q_smem = smem + AD_WARPS * S::RING;                     // [8 heads][pieces][DP] 16-bit
    float* const part_smem = reinterpret_cast<float*>(q_smem + S::Q_BYTES);  // 4 x (o, max, sum)
    float* const q_factor = part_smem + 4 * S::PART;                       // [8] scale log2(e) 2^e
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint32_t d = p.c.d, group = p.q_heads / p.c.heads, items = p.c.heads * a.chunks_of_heads;
    pdl_launch_dependents();

    // ---- this block's part of the line (every warp works it out for itself) ----
    // the ring starts as zeros: chunks past head_dim are never copied, and the matrix instructions read them
    if (d < DP)
        for (uint32_t i = lane; i < S::RING / 16; i += 32) *reinterpret_cast<uint4*>(smem + warp * S::RING + i * 16) = make_uint4(0, 0, 0, 0);
    using Cursor = iq2::Cursor<UNIT, AD_ITEM_COST, false>;
    typename Cursor::Parts line;
    Cursor cur = Cursor::of_part(a, blockIdx.x, gridDim.x, a.inv_blocks, threadIdx.x, AD_THREADS, line);
    const uint64_t u0 = line.begin(blockIdx.x);
    if (threadIdx.x == 0) a.records[blockIdx.x] = cur.record(line, blockIdx.x, blockIdx.x, 1);
    if (cur.t0 == cur.t1) return;  // nothing, or nothing but an item's start
    Cursor pre = cur;

    // ---- the copies: tile `i` (TOK tokens) of pre's piece of an item, one page lookup ahead ----
    uint8_t* const ring = smem + warp * S::RING;
    const uint32_t ring_u32 = smem_u32(ring);
    if (d < DP) __syncwarp();
    // a tile's rows lie side by side in one page, or each lane looks one row up
    const bool side_by_side = p.c.page_size % TOK == 0;
    const uint32_t row_bytes = d * S::ESIZE, chunk = lane % S::CHUNKS, row0 = lane / S::CHUNKS;
    constexpr int ROWS = 32 / S::CHUNKS;  // rows that the warp copies at a time
    auto page_of = [&](uint32_t tok) { return a.by_page.quotient(tok); };
    uint32_t pre_i = warp, pre_page = 0, pre_first = 0;  // the tile to copy next, its page, the first token of that page
    uint32_t lane_page = 0, ahead = 0;                    // pages of this warp's next 32 tiles, a lane each; tiles since
    auto look_up = [&](uint32_t tok, uint32_t& page) {
        if (tok < pre.t1) page = (uint32_t)__ldg(p.block_table + (int64_t)pre.b * p.table_width + page_of(tok));
    };
    auto find_tile = [&]() {  // the next tile of this warp, and its page numbers under way
        bool fresh = ahead == 32;
        while (!pre.done() && pre.t0 + pre_i * TOK >= pre.t1) {
            pre.next(p, items);
            pre_i = warp, fresh = true;
        }
        if (pre.done()) return;
        const uint32_t tok = pre.t0 + pre_i * TOK;
        if (side_by_side) {
            if (fresh || pre_i == warp) look_up(tok + lane * (AD_WARPS * TOK), lane_page), ahead = 0;
            pre_page = __shfl_sync(0xFFFFFFFFu, lane_page, ahead++);
            pre_first = page_of(tok) * p.c.page_size;
        } else {
            look_up(tok + lane, pre_page);
            pre_first = page_of(tok + lane) * p.c.page_size;
        }
    };
    // Copies the tile and returns a bit for each token that takes part: rows of tokens past the end, or of pages outside
    // the cache, are zeros, and what such pages hold cannot matter.
    auto copy_tile = [&](uint32_t stage) {
        const uint32_t tok = pre.t0 + pre_i * TOK, h = pre.item / a.chunks_of_heads, dst = ring_u32 + stage * S::STAGE;
        const uint32_t left = pre.t1 - tok, in_page = tok + (side_by_side ? 0 : lane) - pre_first;
        const int64_t row = ((int64_t)pre_page * p.c.heads + h) * p.c.page_size + in_page;
        const uint8_t *const k = static_cast<const uint8_t*>(p.c.k), *const v = static_cast<const uint8_t*>(p.c.v);
        const bool inside = chunk * 16 < row_bytes;
        uint32_t here = ALL;
        if (side_by_side && left >= TOK && pre_page < p.c.pages) {
            const int64_t off = row * row_bytes + row0 * row_bytes + chunk * 16;
            const uint8_t *pk = k + off, *pv = v + off;
            if (inside) {
#pragma unroll
                for (int i = 0; i < TOK / ROWS; ++i, pk += ROWS * row_bytes, pv += ROWS * row_bytes) {
                    cp_async_16(dst + stage_offset<S::CHUNKS, I8>(row0 + i * ROWS, chunk), pk);
                    cp_async_16(dst + TOK * S::ROW + stage_offset<S::CHUNKS, false>(row0 + i * ROWS, chunk), pv);
                }
            }
            if (I8) {
                cp_async_4(dst + 2 * TOK * S::ROW + lane * 4, p.c.k_scale + row + lane, 4);
                cp_async_4(dst + 2 * TOK * S::ROW + TOK * 4 + lane * 4, p.c.v_scale + row + lane, 4);
            }
        } else {
            const bool valid = lane < TOK && lane < left && pre_page < p.c.pages;
            here = __ballot_sync(0xFFFFFFFFu, valid);
            const int64_t mine = !valid ? -1 : side_by_side ? row + lane : row;
#pragma unroll 1
            for (int i = 0; i < TOK / ROWS; ++i) {
                const uint32_t r = row0 + i * ROWS;
                const int64_t src = __shfl_sync(0xFFFFFFFFu, mine, r);
                const int64_t off = src < 0 ? 0 : src * row_bytes + chunk * 16;
                if (inside) {
                    cp_async_16(dst + stage_offset<S::CHUNKS, I8>(r, chunk), k + off, src < 0 ? 0 : 16);
                    cp_async_16(dst + TOK * S::ROW + stage_offset<S::CHUNKS, false>(r, chunk), v + off, src < 0 ? 0 : 16);
                }
            }
            if (I8) {
                cp_async_4(dst + 2 * TOK * S::ROW + lane * 4, p.c.k_scale + (valid ? mine : 0), valid ? 4 : 0);
                cp_async_4(dst + 2 * TOK * S::ROW + TOK * 4 + lane * 4, p.c.v_scale + (valid ? mine : 0), valid ? 4 : 0);
            }
        }
        pre_i += AD_WARPS;
        return here;
    };
    uint32_t present[AD_STAGES] = {};
    auto copy_and_find = [&](int stage) {
        if (!pre.done()) {
            const uint32_t here = copy_tile(stage);
#pragma unroll
            for (int s = 0; s < AD_STAGES; ++s)
                if (s == stage) present[s] = here;
            find_tile();
        }
        cp_async_commit();
    };
    // q of an item, a warp a head: loaded while the copies before it are under way
    float q_next[DP / 32];
    auto load_q = [&](const Cursor& c) {
        const uint32_t kv = c.item / a.chunks_of_heads, h0 = kv * group + (c.item % a.chunks_of_heads) * AD_HEADS;
        const bool has = warp < min((uint32_t)AD_HEADS, (kv + 1) * group - h0);
        const int64_t at = (int64_t)c.b * p.q.token_stride + (int64_t)(h0 + warp) * p.q.head_stride;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) q_next[i] = has && lane + i * 32 < d ? load_elem(p.q.p, at + lane + i * 32, p.dtype) : 0.f;
    };
    find_tile();
    load_q(cur);
#pragma unroll 1
    for (int s = 0; s < AD_STAGES - 1; ++s) copy_and_find(s);
    int stage = 0;

    while (!cur.done()) {
        // ---- q of the item: the 16-bit pieces of each head ----
        const uint32_t kv_head = cur.item / a.chunks_of_heads, head0 = kv_head * group + (cur.item % a.chunks_of_heads) * AD_HEADS;
        const uint32_t heads = min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0);
        {
            float top = 0.f, up = 1.f, down = 1.f;  // 2^e and 2^-e
            if (!BF) {
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) top = fmaxf(top, fabsf(q_next[i]));
                for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
                const int e = min(max((int)(__float_as_uint(top) >> 23) - 126, -125), 126);
                if (top > 0.f && top < INFINITY) up = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
            }
            uint16_t* const q = reinterpret_cast<uint16_t*>(q_smem) + warp * S::PIECES * DP;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                float rest = q_next[i] * down;
#pragma unroll
                for (int piece = 0; piece < S::PIECES; ++piece) {
                    const uint32_t h = pack_pair<BF>(rest, 0.f);
                    q[piece * DP + lane + i * 32] = (uint16_t)h;
                    rest = (rest - unpack_pair<BF>(h).x) * AD_LOW<BF>;
                }
            }
            if (lane == 0) q_factor[warp] = p.scale * LOG2E * up * (SHIFTED ? CODE_UNIT : 1.f);
        }
        __syncthreads();
        // A fragments of S: k index 16 ks + 2t (+1, +8, +9). For int8 the k index is a relabelled dimension, so that a
        // thread's codes of four k steps are 16 consecutive bytes of its row.
        auto k_lo = [&](int ks) { return I8 ? (t + 4 * (ks / 4)) * 16 + (ks % 4) * 4 : ks * 16 + t * 2; };
        const uint32_t* const q_row = reinterpret_cast<const uint32_t*>(q_smem) + g * S::PIECES * (DP / 2);
        uint32_t qa[KS][4];
        float minus[4] = {0.f, 0.f, 0.f, 0.f};  // where S starts: minus its products with the 128s
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const uint32_t lo = k_lo(ks) / 2, hi = lo + (I8 ? 1 : 4);
            qa[ks][0] = q_row[lo], qa[ks][1] = q_row[DP / 2 + lo];
            qa[ks][2] = q_row[hi], qa[ks][3] = q_row[DP / 2 + hi];
            if (SHIFTED) mma16816<BF>(minus, qa[ks], CODE_ZERO, CODE_ZERO);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) minus[j] = -minus[j];
        auto joined = [](float high, float low) { return fmaf(low, 1.f / AD_LOW<BF>, high); };
        const float factor = q_factor[g];
        float o[NT][4], o_off[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f, f = power_of_two(AD_MOST);  // (int8 caches: f)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

        const uint32_t tokens = cur.t1 - cur.t0;
#pragma unroll 1
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
            for (int n = 0; n < ST; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = minus[j];
            if (I8) {
#pragma unroll
                for (int q4 = 0; q4 < KS / 4; ++q4) {
                    uint4 w[ST];
#pragma unroll
                    for (int n = 0; n < ST; ++n) w[n] = ld_shared_v4<0>(k_at + stage_offset<S::CHUNKS, true>(n * 8 + g, t + 4 * q4));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int n = 0; n < ST; ++n) {
                            const uint32_t u = (j == 0 ? w[n].x : j == 1 ? w[n].y : j == 2 ? w[n].z : w[n].w) ^ 0x80808080u;
                            mma16816<BF>(s[n], qa[q4 * 4 + j], code_pair<SHIFTED>(u, 0x4140u), code_pair<SHIFTED>(u, 0x4342u));
                        }
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t r[4];  // tokens 0-7 chunks 2 ks, 2 ks + 1, then tokens 8-15
                    ldmatrix4(r, k_at + stage_offset<S::CHUNKS, false>((lane / 16) * 8 + lane % 8, ks * 2 + (lane / 8) % 2));
                    mma16816<BF>(s[0], qa[ks], r[0], r[1]);
                    mma16816<BF>(s[1], qa[ks], r[2], r[3]);
                    if (THIRD) {
                        const uint32_t third[4] = {q_row[DP + k_lo(ks) / 2], 0u, q_row[DP + k_lo(ks) / 2 + 4], 0u};
                        mma16816<BF>(s[0], third, r[0], r[1]);
                        mma16816<BF>(s[1], third, r[2], r[3]);
                    }
                }
            }

            // x = log2(e) scale q . k, this thread's tokens 8 n + 2 t, + 1 of head g; w = 2^(x - m), times f and the value scale
            float x[ST][2], e[ST][2], w[ST][2], vs[ST][2], sum;
            const float2* const scales = reinterpret_cast<const float2*>(ring + stage * S::STAGE + 2 * TOK * S::ROW) + t;
#pragma unroll
            for (int n = 0; n < ST; ++n) {
                float2 ks2 = make_float2(factor, factor), vs2 = make_float2(1.f, 1.f);
                if (I8) {
                    const float2 sk = scales[n * 4], sv = scales[TOK / 2 + n * 4];
                    ks2 = make_float2(sk.x * factor, sk.y * factor);
                    vs2 = sv;
                }
                x[n][0] = joined(s[n][0], s[n][2]) * ks2.x, x[n][1] = joined(s[n][1], s[n][3]) * ks2.y;
                vs[n][0] = vs2.x, vs[n][1] = vs2.y;
            }
            if (here != ALL) {
#pragma unroll
                for (int n = 0; n < ST; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (!((here >> (n * 8 + t * 2 + j)) & 1u)) x[n][j] = -INFINITY;
            }
            // The reference does as a rule: the products are made with it, and made again in the rare case that it moves.
            for (;;) {
                const float base = m == -INFINITY ? 0.f : I8 ? m : m - AD_TOP<BF>;
                float top = 0.f;
                sum = 0.f;
#pragma unroll
                for (int n = 0; n < ST; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        e[n][j] = exp2_approx(x[n][j] - base);
                        w[n][j] = I8 ? e[n][j] * f * vs[n][j] : e[n][j];
                        top = fmaxf(top, I8 ? fabsf(w[n][j]) : w[n][j]);
                        if (I8) sum += e[n][j];
                    }
                if (I8) top = fmaxf(top, sum);
                if (!__any_sync(0xFFFFFFFFu, top > (I8 ? AD_SCALED_LAZY : AD_LAZY<BF>) || m == -INFINITY)) break;
                // the largest x of the head's tokens, and the largest x + log2 |value scale|
                float most = -INFINITY, weighed = -INFINITY;
#pragma unroll
                for (int n = 0; n < ST; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        most = fmaxf(most, x[n][j]);
                        if (I8) weighed = fmaxf(weighed, x[n][j] + __log2f(fabsf(vs[n][j])));
                    }
#pragma unroll
                for (int b = 1; b < 4; b *= 2) {
                    most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, b));
                    if (I8) weighed = fmaxf(weighed, __shfl_xor_sync(0xFFFFFFFFu, weighed, b));
                }
                const float next = fmaxf(m, most), keep = m == -INFINITY ? 0.f : exp2_approx(m - next);
                const Moved to = I8 ? Moved::from(m, f, most, weighed) : Moved{next, f, keep, keep, next > m};
                if (!__any_sync(0xFFFFFFFFu, to.moved)) break;
                if (to.moved) {
                    m = to.m, f = to.f;
                    l *= to.keep;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[n][j] *= to.keep_o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o_off[j] *= to.keep_o;
                }
            }
            if (I8) l += sum;
            uint32_t pa[TOK / 16][4], pa3[TOK / 16][4];
#pragma unroll
            for (int n = 0; n < ST; ++n) {
                if (!I8) l += e[n][0] + e[n][1];
                const uint32_t high = pack_pair<BF>(w[n][0], w[n][1]);
                const float2 h = unpack_pair<BF>(high);
                const uint32_t low = pack_pair<BF>((w[n][0] - h.x) * AD_LOW<BF>, (w[n][1] - h.y) * AD_LOW<BF>);
                pa[n / 2][(n % 2) * 2] = high;
                pa[n / 2][(n % 2) * 2 + 1] = low;
                if (THIRD) {
                    const float2 h2 = unpack_pair<BF>(low);
                    pa3[n / 2][(n % 2) * 2] = pack_pair<BF>(w[n][0] - h.x - h2.x, w[n][1] - h.y - h2.y);
                    pa3[n / 2][(n % 2) * 2 + 1] = 0u;
                }
            }

            if (I8) {
#pragma unroll
                for (int ks = 0; ks < TOK / 16; ++ks)
                    if (SHIFTED) mma16816<BF>(o_off, pa[ks], CODE_ZERO, CODE_ZERO);
#pragma unroll
                for (int c = 0; c < S::CHUNKS; ++c) {
                    uint32_t r[4];  // chunk c of tokens 0-7, 8-15, 16-23, 24-31; each word: dimensions 2g, 2g + 1 of two tokens
                    ldmatrix4_trans(r, v_at + stage_offset<S::CHUNKS, false>(lane, c));
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[j] ^= 0x80808080u;
#pragma unroll
                    for (int ks = 0; ks < TOK / 16; ++ks) {
                        mma16816<BF>(o[c * 2], pa[ks], code_pair<SHIFTED>(r[ks * 2], 0x4240u), code_pair<SHIFTED>(r[ks * 2 + 1], 0x4240u));
                        mma16816<BF>(o[c * 2 + 1], pa[ks], code_pair<SHIFTED>(r[ks * 2], 0x4341u), code_pair<SHIFTED>(r[ks * 2 + 1], 0x4341u));
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c += 2) {
                    uint32_t r[4];  // chunk c of tokens 0-7 and 8-15, then chunk c + 1
                    ldmatrix4_trans(r, v_at + stage_offset<S::CHUNKS, false>(lane % 16, c + lane / 16));
                    mma16816<BF>(o[c], pa[0], r[0], r[1]);
                    mma16816<BF>(o[c + 1], pa[0], r[2], r[3]);
                    if (THIRD) {
                        mma16816<BF>(o[c], pa3[0], r[0], r[1]);
                        mma16816<BF>(o[c + 1], pa3[0], r[2], r[3]);
                    }
                }
            }
            __syncwarp();
            stage = stage == AD_STAGES - 1 ? 0 : stage + 1;
        }
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        if (I8) {  // the 128s and the level off, and the codes' unit on
            const Leveled piece = Leveled::of(l, f, SHIFTED ? CODE_UNIT : 1.f);
            m += piece.k, l = piece.l;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][j] = (SHIFTED ? o[n][j] - o_off[j] : o[n][j]) * piece.down * piece.off;
        }

        Cursor next = cur;
        next.next(p, items);
        if (!next.done()) load_q(next);

        // ---- the eight warps' (o, m, l) of the item, through four slots of shared memory ----
        auto put = [&](float* slot) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // int8: accumulator columns are the even and odd dimensions of a 16-dimension chunk
                const uint32_t e0 = KIND == CK_INT8 ? (n / 2) * 16 + n % 2 + t * 4 : n * 8 + t * 2, e1 = e0 + (KIND == CK_INT8 ? 2 : 1);
                slot[g * DP + e0] = joined(o[n][0], o[n][2]);
                slot[g * DP + e1] = joined(o[n][1], o[n][3]);
            }
            if (t == 0) slot[AD_HEADS * DP + g] = m, slot[AD_HEADS * DP + AD_HEADS + g] = l;
        };
        if (warp >= 4) put(part_smem + (warp - 4) * S::PART);
        __syncthreads();
        if (warp < 4) {
            float* const slot = part_smem + warp * S::PART;
            const float m2 = slot[AD_HEADS * DP + g], l2 = slot[AD_HEADS * DP + AD_HEADS + g];
            const float both = fmaxf(m, m2), f1 = both == -INFINITY ? 0.f : exp2_approx(m - both), f2 = both == -INFINITY ? 0.f : exp2_approx(m2 - both);
            l = l * f1 + l2 * f2, m = both;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t e0 = KIND == CK_INT8 ? (n / 2) * 16 + n % 2 + t * 4 : n * 8 + t * 2, e1 = e0 + (KIND == CK_INT8 ? 2 : 1);
                o[n][0] = joined(o[n][0], o[n][2]) * f1 + slot[g * DP + e0] * f2, o[n][2] = 0.f;
                o[n][1] = joined(o[n][1], o[n][3]) * f1 + slot[g * DP + e1] * f2, o[n][3] = 0.f;
            }
            __syncwarp();
            put(slot);
        }
        __syncthreads();
        {
            const bool whole = cur.whole();
            float* const part = a.parts + ((uint64_t)blockIdx.x * 2 + (cur.first_of(u0) ? 0 : 1)) * S::PART;
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

template <int DP, int KIND, bool WIDE>
cudaError_t launch(const DecodeArgs& a, uint32_t blocks, cudaStream_t stream) {
    using S = DecodeShape<DP, KIND, WIDE>;
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<DP, KIND, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return e;
    decode_kernel<DP, KIND, WIDE><<<blocks, AD_THREADS, S::SMEM, stream>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return launch_join<DP>(a, blocks, stream);
}

template <int DP>
cudaError_t launch_kind(const DecodeArgs& a, uint32_t blocks, cudaStream_t stream) {
    const bool wide = a.p.dtype == kF32;
    if (a.p.c.dtype == kInt8) return a.p.dtype != kBf16 ? launch<DP, CK_INT8, true>(a, blocks, stream) : launch<DP, CK_INT8, false>(a, blocks, stream);
    if (a.p.c.dtype == kF16) return launch<DP, CK_F16, false>(a, blocks, stream);
    return wide ? launch<DP, CK_BF16, true>(a, blocks, stream) : launch<DP, CK_BF16, false>(a, blocks, stream);
}

}  // namespace

bool attention_decode_fits(const KvCacheView& c, uint32_t table_width, uint32_t q_heads) {
    const uint32_t cost = c.dtype == kInt4 ? AD_I4_ITEM_COST : AD_ITEM_COST;
    const uint32_t unit = c.dtype == kInt4 ? AD_I4_UNIT : c.dtype == kInt8 ? DecodeShape<64, CK_INT8, false>::UNIT : DecodeShape<64, CK_F16, false>::UNIT;
    const uint64_t tokens = std::min<uint64_t>((uint64_t)table_width * c.page_size, INT32_MAX);
    const uint64_t items = (uint64_t)c.heads * ((q_heads / c.heads + AD_HEADS - 1) / AD_HEADS);
    return ((tokens + unit - 1) / unit + cost) * items <= (uint64_t)UINT32_MAX;
}

size_t attention_decode_workspace(uint32_t, uint32_t, uint32_t, uint32_t d, int num_sms) {
    return records_bytes(num_sms) + (size_t)num_sms * 2 * AD_HEADS * ((d > 64 ? 128 : 64) + 2) * sizeof(float);
}

cudaError_t launch_attention_decode(const DecodeParams& p, void* workspace, int num_sms, cudaStream_t stream) {
    if (p.c.dtype == kInt4) return launch_attention_decode_int4(p, workspace, num_sms, stream);
    const DecodeArgs a = decode_args(p, workspace, num_sms);
    return p.c.d > 64 ? launch_kind<128>(a, num_sms, stream) : launch_kind<64>(a, num_sms, stream);
}

}  // namespace iq2
