// Attention of one new token a sequence over a 4-bit paged cache: the line of work, its parts and their join are those of
// attention_decode.cu, the products are turned round.
//
// A cached element is code g s (iq2_kv_cache): 72 bytes for a row of 128, so that widening the codes costs as much as HBM. The
// products have the tokens (or the values' dimensions) as the sixteen rows of mma.sync m16n8k16 and eight query heads as its columns:
//   S^T = K Q^T  (32 tokens x 8 heads a warp's tile),  O^T = V^T P^T  (DP dimensions x 8 heads)
// so that all rows of an accumulator are in use: 32 + 8 registers at 128 elements, half of what heads as rows take, which
// leaves room for twice the warps.
//   * Codes become f16 values code g 2^-15 by one AND and one multiply-add a pair: four bits u among the lowest ten are the f16
//     numbers u 2^-22 or u 2^-18, which A = G 2^15 or G 2^11 and B = -G 2^-4 make (u - 8) G 2^-7 of, exactly (g has four significant
//     bits and is a multiple of 2^-9); G = g 2^-8 are the e4m3 bits moved by seven places.
//   * A product's inner index may be relabelled as long as both sides agree. For S a thread's inner elements are DP / 4 consecutive
//     ones of a key row, one group: one wide load and one scale a key. For O a thread's rows are DP / 8 consecutive dimensions, again
//     one group, of the two tokens whose p it holds; tokens are relabelled so that both kinds of loads are free of bank conflicts.
//   * q of 32 bits and p are sums of two f16 pieces in one accumulator: q is held times the power of two that brings a head's
//     largest |q| to 2^12, so that its 22 bits end at 2^-36 of it. q of 16 bits is one piece, which has all bits of bf16 elements down to
//     2^-29 and of f16 ones down to 2^-26 of the head's largest, and below is off by 2^-37 of that; p of bf16 q is rounded to f16 once.
//   * The row scales of keys multiply s, those of values multiply p. p next to the largest score's, whose sum is l, ends at 2^-126 as
//     f32's exponential does, whatever the values; what f16 pieces are taken of is p times the value's row scale times 2^level, a
//     head's own power of two that makes the largest of these 2^7 to 2^8 (they may grow to 2^15), so that 22 bits end at 2^-31 of the
//     largest. (With the row scales in the reference instead, a product and a sum less, 2 % faster, rows of 3e38 lost the tokens below
//     2^-7 of the largest weight, and rows of zeros all of their weight beside rows of 1e9.)
// The maxima, sums, s, p and o are f32.
//
// A warp has a part of the line of its own, copies its tiles into two stages by itself and waits for nobody; at the end the block
// adds up the pieces of items that its warps share. (Items dealt to blocks, tiles to the block's warps in turn: two barriers an
// item, 143 us for 128 x 4096 tokens in place of 104.)
//
// Measured (8 key heads, 128 elements, bf16 q unless said): 128 sequences of up to 4096 tokens 90 us, 4200 GB/s, 0.64 of the copy
// rate. Latency binds: 710 instructions for a tile of 32 tokens and a key head are 52 us at full issue, less than HBM's 58, but three
// warps a scheduler, whose loads, products and exponentials wait for one another, fill 65 % of the issue slots (ALU pipe 48 %).
// 64 of up to 4096 50.5 us, with f16 q 55.6, with f32 q 61.5, with pages of 16 or 48 tokens 54.6, of 96 / 64 / 32 elements 59.4 / 38.4 /
// 40; 512 of up to 512 75 us; one of 100001 tokens, 64 query heads, 36 us; 16 of up to 2048, f32 q, 18 us, f16 q 16.6. One of 333
// tokens 8.0 us where the table has no more than 800 tokens' pages, 9.2 where it has 8192; 18 of up to 760 9.8 and 14.1. The first version here,
// heads as rows as in attention_decode.cu, took 185, 55 and 22.5 us for 128 x 4096, 1 x 100001 and 16 x 2048. Warps of a block: 8 / 11 /
// 12 / 16 103 / 98 / 93.6 / 95 us for 128 x 4096 (16 spill); tiles of 64 tokens with 8 warps 102 (with 12, of 32, 103 then).
#include "attention_decode.cuh"

namespace iq2 {

namespace {

constexpr int A4_WARPS = AD_I4_WARPS, A4_THREADS = A4_WARPS * 32;
static_assert(2 * A4_WARPS <= 32, "a lane a piece");
constexpr int A4_TOK = 32, A4_NT = A4_TOK / 8;  // tokens of a warp's stage, and eights of them
constexpr int A4_RUN = 8;                // tokens that lie side by side in a page of a multiple of these
constexpr float A4_FACTOR = 1024.f;      // factors of scores above this are applied in two steps
constexpr float A4_VALUE = 32768.f;      // 2^15: what values are held by

template <int DP>
struct Shape4 {
    static constexpr int ROW = DP / 2, CHUNKS = ROW / 16;  // bytes and 16-byte chunks of a padded row
    static constexpr int KS = DP / 16, MT = DP / 16;       // steps of S's inner index, row tiles of O
    static constexpr int SCALES = 2 * A4_TOK * ROW;        // of a stage: row scales of K and V, then group scales, a word a token
    static constexpr int STAGE = SCALES + 4 * A4_TOK * 4;
    static constexpr int RING = 2 * STAGE;
    static constexpr int HEAD = DP + 4;                    // floats of a head in a piece's slot
    static constexpr int MAXIMA = AD_HEADS * HEAD, SUMS = MAXIMA + AD_HEADS, SLOT = SUMS + AD_HEADS;  // floats of one (o, max, sum)
    static constexpr int PART = AD_HEADS * (DP + 2);       // and in the workspace
    static constexpr int SMEM = A4_WARPS * (RING + SLOT * 4);
    static_assert(SLOT * 4 <= RING, "a warp's last piece lies in its ring");
};

// Where a token of a tile lies among the eight that share an accumulator's rows: a thread's pairs 2t, 2t + 1 are the rows
// (0, 3), (1, 2), (4, 7), (5, 6), of which rows 4 to 7 have the halves of their 64 bytes swapped. So the four rows that the
// threads of a column read together, 0 1 4 5 or 2 3 6 7, fall to different banks, and so do two rows side by side.
__device__ __forceinline__ uint32_t row_of(uint32_t i) { return (0x65742130u >> (i * 4)) & 7u; }

// Byte offset of 16-byte chunk c of row r in a K or V stage.
template <int CHUNKS>
__device__ __forceinline__ uint32_t chunk_offset(uint32_t r, uint32_t c) {
    return r * (CHUNKS * 16) + (CHUNKS == 4 ? c ^ ((r >> 1) & 2) : c) * 16;
}

// What makes f16 values of codes: A for the lower and the upper bits of a byte, and B, for the two halves of a word.
struct CodeScale {
    __half2 lo, hi, off;
};
// bytes: the e4m3 scales of the two halves in bytes 1 and 3, zeros in 0 and 2.
__device__ __forceinline__ CodeScale code_scale(uint32_t bytes) {
    const uint32_t moved = bytes >> 1;
    const __half2 g = *reinterpret_cast<const __half2*>(&moved);
    return {__hmul2(g, __float2half2_rn(32768.f)), __hmul2(g, __float2half2_rn(2048.f)), __hmul2(g, __float2half2_rn(-0.0625f))};
}
// The values of a word's codes: v[0], v[1] the lower and upper bits of bytes 0 and 2, v[2], v[3] of bytes 1 and 3.
__device__ __forceinline__ void code_values(uint32_t w, const CodeScale& s, uint32_t (&v)[4]) {
    const uint32_t even = w << 2, odd = w >> 6;
    const uint32_t u[4] = {even & 0x003C003Cu, even & 0x03C003C0u, odd & 0x003C003Cu, odd & 0x03C003C0u};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&u[i]), i % 2 ? s.hi : s.lo, s.off);
        v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}

// An 8 x 8 matrix of 16-bit elements, a row's pairs in the four lanes of a column of threads, turned round.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t ld_shared(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

// N consecutive elements of a row of q as f32, zeros unless `there`; `vec`: rows start on 16-byte boundaries.
template <int N>
__device__ __forceinline__ void load_row(const void* base, int64_t at, int dtype, bool there, bool vec, float (&x)[N]) {
    if (!there) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.f;
    } else if (!vec) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = load_elem(base, at + i, dtype);
    } else if (dtype == kF32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(base) + at + i));
            x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at + i));
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = dtype == kF16 ? unpack_pair<false>(u[j]) : unpack_pair<true>(u[j]);
                x[i + 2 * j] = f.x, x[i + 2 * j + 1] = f.y;
            }
        }
    }
}

// N consecutive elements of a 16-byte aligned output row.
template <int N>
__device__ __forceinline__ void store_row(void* base, int64_t at, int dtype, const float (&y)[N]) {
    if (dtype == kF32) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(static_cast<float*>(base) + at + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i += 8) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = dtype == kF16 ? pack_pair<false>(y[i + 2 * j], y[i + 2 * j + 1]) : pack_pair<true>(y[i + 2 * j], y[i + 2 * j + 1]);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at + i) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// A warp's piece of an item that is not all of it. valid: 0, or 1, and 2 where it has the item's first token, 4 its last one, 8
// where the item is the first of the block.
struct Piece {
    uint32_t b, item, valid;
};
// Where piece `i` lies: a warp's first one behind the rings, its last one in its ring.
template <typename S>
__device__ __forceinline__ float* slot_of(uint8_t* smem, uint32_t i) {
    return reinterpret_cast<float*>(smem + (i % 2 == 0 ? A4_WARPS * S::RING + i / 2 * (S::SLOT * 4) : i / 2 * S::RING));
}

// WIDE: q of 32 bits, in two pieces (of 16 bits it is one). FINE: p in two pieces. One piece is for bf16 outputs, which are rounded
// to 2^-8 of themselves anyway, p to 2^-11: 50.5 us against 55.0 for 64 x 4096 tokens. FULL: head_dim is DP.
template <int DP, bool WIDE, bool FINE, bool FULL>
__global__ void __launch_bounds__(A4_THREADS, 1) decode4_kernel(const __grid_constant__ DecodeArgs a) {
    using S = Shape4<DP>;
    constexpr int TOK = A4_TOK, NT = A4_NT, KS = S::KS, MT = S::MT;
    using Cursor = iq2::Cursor<AD_I4_UNIT, AD_I4_ITEM_COST, true>;
    const DecodeParams& p = a.p;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Piece pieces[2 * A4_WARPS];  // of each warp its first and its last, of those that are not a whole item
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint32_t d = FULL ? DP : p.c.d, group = p.q_heads / p.c.heads, items = p.c.heads * a.chunks_of_heads;
    pdl_launch_dependents();

    // the ring starts as zeros: chunks past head_dim are never copied, and the matrix instructions read them
    if (!FULL)
        for (uint32_t i = lane; i < S::RING / 16; i += 32) *reinterpret_cast<uint4*>(smem + warp * S::RING + i * 16) = make_uint4(0, 0, 0, 0);
    if (lane < 2) pieces[warp * 2 + lane].valid = 0;
    // where a warp reads and where it copies from, and the block's first unit, each warp's own: in shared memory, since registers
    // are short and they change from one piece to the next only
    __shared__ Cursor cursors[A4_WARPS][2];
    __shared__ uint64_t block_u0[A4_WARPS];
    __shared__ __align__(8) float factor_rest[A4_WARPS][AD_HEADS];  // how many times A4_FACTOR the heads' factors are, 1 or more
    Cursor& cur_held = cursors[warp][0];
    Cursor& pre_held = cursors[warp][1];
    bool live;  // there is a tile to copy
    uint32_t pre_tok, pre_t1;
    if (a.block_an_item) {
        const uint32_t b = blockIdx.x / items, item = blockIdx.x % items, len = seq_len(p, b), tiles = (len + TOK - 1) / TOK;
        if (len == 0) {
            const uint32_t kv_head = item / a.chunks_of_heads, first = kv_head * group + item % a.chunks_of_heads * AD_HEADS;
            for (uint32_t i = threadIdx.x; i < min((uint32_t)AD_HEADS, (kv_head + 1) * group - first) * d; i += A4_THREADS)
                store_elem(p.out, ((int64_t)b * p.q_heads + first) * d + i, p.dtype, 0.f);
            return;
        }
        pre_tok = warp * tiles / A4_WARPS * TOK, pre_t1 = min((warp + 1) * tiles / A4_WARPS * TOK, len);
        live = pre_tok < pre_t1;
        const Cursor cur{0, live ? 1u : 0u, b, item, len, 1, 0, 1, pre_tok, pre_t1};
        if (lane == 0) cur_held = cur, pre_held = cur, block_u0[warp] = 0;
    } else {
        typename Cursor::Parts line;
        const uint32_t part0 = blockIdx.x * A4_WARPS;  // the block's parts of the line, one a warp
        Cursor cur = Cursor::of_part(a, part0 + warp, gridDim.x * A4_WARPS, a.inv_blocks * (1.0 / A4_WARPS), lane, 32, line);
        if (threadIdx.x == 0) a.records[blockIdx.x] = cur.record(line, blockIdx.x, part0, A4_WARPS);
        if (cur.t0 == cur.t1) cur.unit = cur.end;  // nothing, or nothing but an item's start
        if (lane == 0) cur_held = cur, pre_held = cur, block_u0[warp] = line.begin(part0);
        live = !cur.done(), pre_tok = cur.t0, pre_t1 = cur.t1;
    }
    auto advance = [&](Cursor& held) {
        Cursor c = held;
        c.next(p, items);
        __syncwarp();
        if (lane == 0) held = c;
        __syncwarp();
        return !c.done();
    };

    // ---- the copies: pre's tile from token pre_tok on, whose pages have been looked up ----
    const uint32_t ring = smem_u32(smem + warp * S::RING);
    __syncwarp();
    // a tile's rows lie side by side in one page, or in runs of eight, or each lane looks its row up
    const bool whole_tiles = p.c.page_size % TOK == 0, runs = p.c.page_size % A4_RUN == 0;
    constexpr int ROWS = 32 / S::CHUNKS;  // rows that the warp copies at a time
    const uint32_t row_bytes = d / 2, chunk = lane % S::CHUNKS, row0 = lane / S::CHUNKS;
    const uint32_t page_rows = p.c.heads * p.c.page_size;
    const bool inside = FULL || chunk * 16 < row_bytes;
    const uint8_t* const k_from = static_cast<const uint8_t*>(p.c.k) + chunk * 16;
    const int64_t v_less_k = static_cast<const uint8_t*>(p.c.v) - static_cast<const uint8_t*>(p.c.k);
    // 32 words of each kind of scale, 16 bytes a lane: row scales of K and V, then group scales
    const uint8_t* const scales_from = (lane < 8 ? reinterpret_cast<const uint8_t*>(p.c.k_scale) : lane < 16 ? reinterpret_cast<const uint8_t*>(p.c.v_scale)
                                        : lane < 24 ? p.c.k_group : p.c.v_group);
    uint32_t pre_in = 0, pre_head = 0;  // the tile's place in its page (whole tiles), rows of the heads before
    const int32_t* table = nullptr;     // the sequence's pages
    uint32_t page = 0, ahead = 0;       // this lane's page of those looked up; tiles since
    bool fresh = true;
    auto look_up = [&](uint32_t tok) {
        return tok < pre_t1 ? (uint32_t)__ldg(table + a.by_page.quotient(tok)) : 0xFFFFFFFFu;
    };
    auto in_page = [&](uint32_t tok) { return tok - a.by_page.quotient(tok) * p.c.page_size; };
    auto find_tile = [&]() {  // the next tile of this warp, and its page numbers under way
        if (pre_tok >= pre_t1) {
            live = advance(pre_held);
            pre_tok = pre_held.t0, pre_t1 = pre_held.t1, fresh = true;
        }
        if (!live) return;
        if (fresh) {
            pre_head = pre_held.item / a.chunks_of_heads * p.c.page_size;
            table = p.block_table + (int64_t)pre_held.b * p.table_width;
        }
        if (whole_tiles) {  // lanes hold the pages of this warp's next 32 tiles
            if (fresh || ahead == 32) page = look_up(pre_tok + lane * TOK), pre_in = in_page(pre_tok), ahead = 0;
        } else {            // of the tile's runs, or of its tokens
            page = look_up(pre_tok + (runs ? lane % (TOK / A4_RUN) * A4_RUN : lane));
        }
        fresh = false;
    };
    // Copies the tile and returns a bit for each token that takes part: rows of tokens past the end, or of pages outside
    // the cache, are zeros, and what such pages hold cannot matter.
    auto copy_tile = [&](uint32_t dst) {
        const uint32_t left = pre_t1 - pre_tok;
        int64_t mine;  // the row of token `lane`, -1: none
        if (whole_tiles) {
            const uint32_t at = __shfl_sync(0xFFFFFFFFu, page, ahead++);
            const int64_t row = (int64_t)((uint64_t)at * page_rows + (pre_head + pre_in));
            pre_in = pre_in + TOK == p.c.page_size ? 0 : pre_in + TOK;
            if (at < p.c.pages && left >= TOK) {
                const uint8_t* const pk = k_from + (row + row0) * row_bytes;
                const uint8_t* const pv = pk + v_less_k;
                if (inside) {
#pragma unroll
                    for (int i = 0; i < TOK / ROWS; ++i) {
                        cp_async_16(dst + chunk_offset<S::CHUNKS>(row0 + i * ROWS, chunk), pk + i * ROWS * row_bytes);
                        cp_async_16(dst + TOK * S::ROW + chunk_offset<S::CHUNKS>(row0 + i * ROWS, chunk), pv + i * ROWS * row_bytes);
                    }
                }
                cp_async_16(dst + S::SCALES + lane * 16, scales_from + (row * 4 + lane % 8 * 16));
                return 0xFFFFFFFFu;
            }
            mine = at < p.c.pages && lane < left ? row + lane : -1;
        } else if (runs) {
            const int64_t run = page < p.c.pages ? (int64_t)((uint64_t)page * page_rows + (pre_head + in_page(pre_tok + lane % (TOK / A4_RUN) * A4_RUN))) : -1;
            if (left >= TOK && __all_sync(0xFFFFFFFFu, run >= 0)) {
#pragma unroll
                for (int i = 0; i < TOK / ROWS; ++i) {
                    const uint32_t r = row0 + i * ROWS;
                    const uint8_t* const pk = k_from + (__shfl_sync(0xFFFFFFFFu, run, r / A4_RUN) + r % A4_RUN) * row_bytes;
                    if (inside) {
                        cp_async_16(dst + chunk_offset<S::CHUNKS>(r, chunk), pk);
                        cp_async_16(dst + TOK * S::ROW + chunk_offset<S::CHUNKS>(r, chunk), pk + v_less_k);
                    }
                }
                cp_async_16(dst + S::SCALES + lane * 16, scales_from + (__shfl_sync(0xFFFFFFFFu, run, lane % 8 / 2) * 4 + lane % 2 * 16));
                return 0xFFFFFFFFu;
            }
            const int64_t from = __shfl_sync(0xFFFFFFFFu, run, lane / A4_RUN);
            mine = from >= 0 && lane < left ? from + lane % A4_RUN : -1;
        } else {
            mine = page < p.c.pages ? (int64_t)((uint64_t)page * page_rows + (pre_head + in_page(pre_tok + lane))) : -1;
        }
#pragma unroll 1
        for (int i = 0; i < TOK / ROWS; ++i) {
            const uint32_t r = row0 + i * ROWS;
            const int64_t src = __shfl_sync(0xFFFFFFFFu, mine, r);
            const uint8_t* const pk = k_from + (src < 0 ? 0 : src * row_bytes);
            if (inside) {
                cp_async_16(dst + chunk_offset<S::CHUNKS>(r, chunk), pk, src < 0 ? 0 : 16);
                cp_async_16(dst + TOK * S::ROW + chunk_offset<S::CHUNKS>(r, chunk), pk + v_less_k, src < 0 ? 0 : 16);
            }
        }
        const int64_t at = max(mine, (int64_t)0);
        const uint32_t bytes = mine < 0 ? 0 : 4, to = dst + S::SCALES + lane * 4;
        cp_async_4(to, p.c.k_scale + at, bytes);
        cp_async_4(to + TOK * 4, p.c.v_scale + at, bytes);
        cp_async_4(to + TOK * 8, p.c.k_group + at * 4, bytes);
        cp_async_4(to + TOK * 12, p.c.v_group + at * 4, bytes);
        return __ballot_sync(0xFFFFFFFFu, mine >= 0);
    };
    uint32_t there = 0;  // the tokens of the tile that was copied last
    auto copy_and_find = [&](uint32_t dst) {
        if (live) {
            there = copy_tile(dst);
            pre_tok += TOK;
            find_tile();
        }
        cp_async_commit();
    };
    const bool live_at_start = live;
    if (live) find_tile();
    copy_and_find(ring);
    uint32_t at = ring;  // the stage to take next

    // this thread's places: its key row and chunk, its two value rows and their bytes, its groups' scales as bytes 1 and 3
    const uint32_t k_row = row_of(g), v_row0 = row_of(2 * t), v_row1 = row_of(2 * t + 1);
    const uint32_t k_at = DP == 128 ? chunk_offset<S::CHUNKS>(k_row, t) : k_row * S::ROW + t * 8;
    const uint32_t v_at0 = TOK * S::ROW + (DP == 128 ? chunk_offset<S::CHUNKS>(v_row0, g / 2) + g % 2 * 8 : v_row0 * S::ROW + g * 4);
    const uint32_t v_at1 = TOK * S::ROW + (DP == 128 ? chunk_offset<S::CHUNKS>(v_row1, g / 2) + g % 2 * 8 : v_row1 * S::ROW + g * 4);
    const uint32_t k_group = t * (DP / 4) / I4_GROUP, v_group = g * (DP / 8) / I4_GROUP;
    const uint32_t k_sel = k_group * I4_GROUP < d ? 0x0404u | k_group * 0x1010u : 0x4444u;  // (zeros past head_dim)
    const uint32_t v_sel = 0x4C08u + v_group * 0x1111u;  // (8 + i is the sign of byte i in all bits: none)

    bool first_piece = true;
    for (bool more = live_at_start; more; more = advance(cur_held)) {
        // ---- q of the item: the pieces of head g, elements t DP / 4 and on ----
        // (of the item: its first head, and how many it has)
        auto heads_of = [&](uint32_t item, uint32_t& head0) {
            const uint32_t kv_head = item / a.chunks_of_heads;
            head0 = kv_head * group + (item % a.chunks_of_heads) * AD_HEADS;
            return min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0);
        };
        uint32_t q_high[KS][2], q_low[KS][2];
        float factor[2];  // scale log2(e) 2^(e + 2) of the heads 2t, 2t + 1, or A4_FACTOR where it is more
        {
            float x[DP / 4], top = 0.f, unit = 1.f, down = 1.f;  // 2^e and 2^(13 - e); q of zeros has any
            uint32_t head0;
            const uint32_t heads = heads_of(cur_held.item, head0);
            load_row<DP / 4>(p.q.p, (int64_t)cur_held.b * p.q.token_stride + (int64_t)(head0 + g) * p.q.head_stride + t * (DP / 4), p.dtype,
                             g < heads && t * (DP / 4) < d, a.q_vec, x);
#pragma unroll
            for (int i = 0; i < DP / 4; ++i) top = fmaxf(top, fabsf(x[i]));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int e = min(max((int)(__float_as_uint(top) >> 23) - 126, -110), 126);
            if (top > 0.f && top < INFINITY) unit = __uint_as_float((uint32_t)(e + 127) << 23), down = __uint_as_float((uint32_t)(140 - e) << 23);
            // (times a key's row scale, 2^117 at most, what is left of it is finite: where s is 0 the score is)
            const float all = fminf(p.scale * (4.f * LOG2E) * unit, 3e38f), f = fminf(all, A4_FACTOR);
            if (t == 0) factor_rest[warp][g] = fmaxf(all * (1.f / A4_FACTOR), 1.f);
            __syncwarp();
            factor[0] = __shfl_sync(0xFFFFFFFFu, f, t * 8), factor[1] = __shfl_sync(0xFFFFFFFFu, f, t * 8 + 4);
            // elements j and j + 4 of a word's eight are a pair: j = 0, 1 of one step, j = 2, 3 of the next
#pragma unroll
            for (int i = 0; i < DP / 32; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x0 = x[i * 8 + j] * down, x1 = x[i * 8 + j + 4] * down;
                    const uint32_t high = pack_pair<false>(x0, x1);
                    const float2 back = unpack_pair<false>(high);
                    q_high[i * 2 + j / 2][j % 2] = high;
                    q_low[i * 2 + j / 2][j % 2] = WIDE ? pack_pair<false>(x0 - back.x, x1 - back.y) : 0u;
                }
        }
        // o is held times 2^level of the head, f = 2^level
        float o[MT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, f[2] = {power_of_two(AD_MOST), power_of_two(AD_MOST)};
#pragma unroll
        for (int n = 0; n < MT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

#pragma unroll 1
        for (uint32_t left = cur_held.t1 - cur_held.t0; left != 0; left -= min(left, (uint32_t)TOK)) {
            cp_async_wait<0>();
            __syncwarp();
            const uint32_t here = there;
            copy_and_find(2 * ring + S::STAGE - at);  // the stage that the last tile freed

            // ---- S^T: rows are tokens row_of(g) of each eight, columns the heads 2t, 2t + 1 ----
            float x[NT][2];
#pragma unroll
            for (int mt = 0; mt < NT / 2; ++mt) {
                uint32_t w[2][DP / 32];
                CodeScale scale[2];
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t from = at + k_at + (mt * 2 + r) * 8 * S::ROW;
                    if (DP == 128) {
                        const uint4 u = ld_shared_v4<0>(from);
                        w[r][0] = u.x, w[r][1] = u.y, w[r][2 % (DP / 32)] = u.z, w[r][3 % (DP / 32)] = u.w;
                    } else {
                        const uint2 u = ld_shared_v2_volatile(from);
                        w[r][0] = u.x, w[r][1] = u.y;
                    }
                    scale[r] = code_scale(prmt(ld_shared(at + S::SCALES + TOK * 8 + ((mt * 2 + r) * 8 + k_row) * 4), 0u, k_sel));
                }
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    uint32_t v0[4], v1[4];
                    code_values(w[0][j], scale[0], v0), code_values(w[1][j], scale[1], v1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t k[4] = {v0[2 * h], v1[2 * h], v0[2 * h + 1], v1[2 * h + 1]};
                        mma16816<false>(s, k, q_high[2 * j + h][0], q_high[2 * j + h][1]);
                        if (WIDE) mma16816<false>(s, k, q_low[2 * j + h][0], q_low[2 * j + h][1]);
                    }
                }
                x[mt * 2][0] = s[0], x[mt * 2][1] = s[1], x[mt * 2 + 1][0] = s[2], x[mt * 2 + 1][1] = s[3];
            }

            // x = log2(e) scale q . k, rounded before the reference is taken off (which is one of them); e = 2^(x - m), w = e f times
            // the value scale
            float e[NT][2], w[NT][2], sum[2] = {0.f, 0.f}, vs[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t from = at + S::SCALES + (n * 8 + k_row) * 4;
                const float ks = __uint_as_float(ld_shared(from));
                vs[n] = __uint_as_float(ld_shared(from + TOK * 4));
                x[n][0] *= ks * factor[0], x[n][1] *= ks * factor[1];
            }
            if (here != 0xFFFFFFFFu) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    if (!((here >> (n * 8 + k_row)) & 1u)) x[n][0] = x[n][1] = -INFINITY;
            }
            // Reference and level do as a rule: the products are made with them, and made again in the rare case that they move.
            bool first = __any_sync(0xFFFFFFFFu, m[0] == -INFINITY || m[1] == -INFINITY || factor[0] >= A4_FACTOR || factor[1] >= A4_FACTOR);
            for (;;) {
                if (!first) {
                    float top = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float base = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            e[n][h] = exp2_approx(x[n][h] - base);
                            w[n][h] = e[n][h] * f[h] * vs[n];
                            top = fmaxf(top, fabsf(w[n][h]));
                        }
                        sum[h] = (e[0][h] + e[1][h]) + (e[2][h] + e[3][h]);
                        top = fmaxf(top, sum[h]);
                    }
                    if (!__any_sync(0xFFFFFFFFu, top > AD_SCALED_LAZY)) break;
                }
                if (first) {  // (x is not whole yet where the factor is more than A4_FACTOR)
                    const float2 rest = *reinterpret_cast<const float2*>(factor_rest[warp] + 2 * t);
#pragma unroll
                    for (int n = 0; n < NT; ++n) x[n][0] *= rest.x, x[n][1] *= rest.y;
                }
                bool moved = false;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // the largest x of the head's tokens, and the largest x + log2 |value scale|
                    float most = -INFINITY, weighed = -INFINITY;
#pragma unroll
                    for (int n = 0; n < NT; ++n) most = fmaxf(most, x[n][h]), weighed = fmaxf(weighed, x[n][h] + __log2f(fabsf(vs[n])));
#pragma unroll
                    for (int b = 4; b < 32; b *= 2) {
                        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, b));
                        weighed = fmaxf(weighed, __shfl_xor_sync(0xFFFFFFFFu, weighed, b));
                    }
                    const Moved to = Moved::from(m[h], f[h], most, weighed);
                    moved = moved || to.moved;
                    m[h] = to.m, f[h] = to.f;
                    l[h] *= to.keep;
#pragma unroll
                    for (int n = 0; n < MT; ++n) o[n][h] *= to.keep_o, o[n][2 + h] *= to.keep_o;
                }
                if (!__any_sync(0xFFFFFFFFu, moved) && !first) break;
                first = false;
            }
            l[0] += sum[0], l[1] += sum[1];
            uint32_t high[NT], low[NT];  // the pieces of p, with heads as rows and tokens as columns
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t hi = pack_pair<false>(w[n][0], w[n][1]);
                high[n] = transposed(hi);
                if (FINE) {
                    const float2 back = unpack_pair<false>(hi);
                    low[n] = transposed(pack_pair<false>(w[n][0] - back.x, w[n][1] - back.y));
                }
            }

            // ---- O^T: rows are this thread's DP / 8 dimensions, two a tile ----
#pragma unroll
            for (int ks = 0; ks < NT / 2; ++ks) {
                uint32_t y[2][DP / 32];  // the codes of the two tokens of eight, four of one in the lower half and of the other in the upper
                CodeScale scale[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int n = ks * 2 + r;
                    const uint32_t from0 = at + v_at0 + n * 8 * S::ROW, from1 = at + v_at1 + n * 8 * S::ROW;
                    if (DP == 128) {
                        const uint2 u0 = ld_shared_v2_volatile(from0), u1 = ld_shared_v2_volatile(from1);
                        y[r][0] = prmt(u0.x, u1.x, 0x5410u), y[r][1] = prmt(u0.x, u1.x, 0x7632u);
                        y[r][2 % (DP / 32)] = prmt(u0.y, u1.y, 0x5410u), y[r][3 % (DP / 32)] = prmt(u0.y, u1.y, 0x7632u);
                    } else {
                        const uint32_t u0 = ld_shared(from0), u1 = ld_shared(from1);
                        y[r][0] = prmt(u0, u1, 0x5410u), y[r][1] = prmt(u0, u1, 0x7632u);
                    }
                    const uint32_t groups = at + S::SCALES + TOK * 12 + n * 32;
                    scale[r] = code_scale(prmt(ld_shared(groups + v_row0 * 4), ld_shared(groups + v_row1 * 4), v_sel));
                }
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    uint32_t v0[4], v1[4];
                    code_values(y[0][j], scale[0], v0), code_values(y[1][j], scale[1], v1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t v[4] = {v0[2 * h], v0[2 * h + 1], v1[2 * h], v1[2 * h + 1]};
                        mma16816<false>(o[2 * j + h], v, high[ks * 2], high[ks * 2 + 1]);
                        if (FINE) mma16816<false>(o[2 * j + h], v, low[ks * 2], low[ks * 2 + 1]);
                    }
                }
            }
            __syncwarp();
            at = 2 * ring + S::STAGE - at;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 4; b < 32; b *= 2) l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], b);

        // ---- the end of the piece: a whole item's output, or (o, m, l) for the block to add up ----
        const Cursor cur = cur_held;
        uint32_t head0;
        const uint32_t heads = heads_of(cur.item, head0);
        if (cur.whole()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (2 * t + h < heads && g * (DP / 8) < d) {
                    auto value = [&](float x) { return l[h] == 0.f ? 0.f : x * A4_VALUE / l[h] * over_power(f[h]); };
                    float y[DP / 8];
#pragma unroll
                    for (int j = 0; j < DP / 32; ++j)
                        y[4 * j] = value(o[2 * j][h]), y[4 * j + 1] = value(o[2 * j][2 + h]), y[4 * j + 2] = value(o[2 * j + 1][h]), y[4 * j + 3] = value(o[2 * j + 1][2 + h]);
                    store_row<DP / 8>(p.out, ((int64_t)cur.b * p.q_heads + head0 + 2 * t + h) * d + g * (DP / 8), p.dtype, y);
                }
            }
        } else {
            // (the last piece takes the ring: all of the warp's copies are done then)
            float* const slot = slot_of<S>(smem, warp * 2 + !first_piece);
            if (!first_piece) {
                cp_async_wait<0>();
                __syncwarp();
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const Leveled piece = Leveled::of(l[h], f[h], A4_VALUE);
                auto value = [&](float x) { return x * piece.down * piece.off; };
#pragma unroll
                for (int j = 0; j < DP / 32; ++j)
                    *reinterpret_cast<float4*>(slot + (2 * t + h) * S::HEAD + g * (DP / 8) + j * 4) =
                        make_float4(value(o[2 * j][h]), value(o[2 * j][2 + h]), value(o[2 * j + 1][h]), value(o[2 * j + 1][2 + h]));
                if (g == 0) slot[S::MAXIMA + 2 * t + h] = m[h] + piece.k, slot[S::SUMS + 2 * t + h] = piece.l;
            }
            if (lane == 0)
                pieces[warp * 2 + !first_piece] = {cur.b, cur.item, 1u | (cur.t0 == 0 ? 2u : 0u) | (cur.t1 == cur.len ? 4u : 0u) | (cur.first_of(block_u0[warp]) ? 8u : 0u)};
        }
        first_piece = false;
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- the warps' pieces: those of one item follow one another. A warp an item and head ----
    const Piece mine = lane < 2 * A4_WARPS ? pieces[lane] : Piece{0, 0, 0};
    const uint32_t held = __ballot_sync(0xFFFFFFFFu, mine.valid != 0);
    const int before = 31 - __clz(held & ((1u << lane) - 1));  // the piece before this lane's, -1: none
    const uint32_t b_before = __shfl_sync(0xFFFFFFFFu, mine.b, max(before, 0)), item_before = __shfl_sync(0xFFFFFFFFu, mine.item, max(before, 0));
    uint32_t starts = __ballot_sync(0xFFFFFFFFu, mine.valid != 0 && (before < 0 || b_before != mine.b || item_before != mine.item));
    uint32_t turn = warp;  // (item, head) pairs until this warp's next
#pragma unroll 1
    while (starts != 0) {
        const int at = __ffs(starts) - 1;
        starts &= starts - 1;
        const uint32_t ours = held & ~((1u << at) - 1) & (starts != 0 ? (starts & -starts) - 1 : 0xFFFFFFFFu);
        const int last = 31 - __clz(ours);
        const uint32_t b = __shfl_sync(0xFFFFFFFFu, mine.b, at), item = __shfl_sync(0xFFFFFFFFu, mine.item, at);
        const uint32_t from = __shfl_sync(0xFFFFFFFFu, mine.valid, at), to = __shfl_sync(0xFFFFFFFFu, mine.valid, last);
        const bool whole = (from & 2u) != 0 && (to & 4u) != 0;
        const uint32_t kv_head = item / a.chunks_of_heads, head0 = kv_head * group + (item % a.chunks_of_heads) * AD_HEADS;
        const uint32_t heads = min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0);
        float* const part = a.parts + ((uint64_t)blockIdx.x * 2 + ((from & 8u) != 0 ? 0 : 1)) * S::PART;
        for (; turn < AD_HEADS; turn += A4_WARPS) {
            const uint32_t h = turn;
            if (h >= heads) continue;
            float mx = -INFINITY, sum = 0.f, y[DP / 32] = {};
            for (uint32_t rest = ours; rest != 0; rest &= rest - 1) mx = fmaxf(mx, slot_of<S>(smem, __ffs(rest) - 1)[S::MAXIMA + h]);
#pragma unroll 2
            for (uint32_t rest = ours; rest != 0; rest &= rest - 1) {
                const float* const slot = slot_of<S>(smem, __ffs(rest) - 1);
                const float w = mx == -INFINITY ? 0.f : exp2_approx(slot[S::MAXIMA + h] - mx);
                sum += slot[S::SUMS + h] * w;
#pragma unroll
                for (int i = 0; i < DP / 32; ++i) y[i] += slot[h * S::HEAD + lane + i * 32] * w;
            }
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const uint32_t el = lane + i * 32;
                if (!whole) part[h * DP + el] = y[i];
                else if (el < d) store_elem(p.out, ((int64_t)b * p.q_heads + head0 + h) * d + el, p.dtype, sum == 0.f ? 0.f : y[i] / sum);
            }
            if (!whole && lane == 0) part[AD_HEADS * DP + h] = mx, part[AD_HEADS * DP + AD_HEADS + h] = sum;
        }
        turn -= AD_HEADS;
    }
}

template <int DP, bool WIDE, bool FINE, bool FULL>
cudaError_t launch4(const DecodeArgs& a, uint32_t blocks, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(decode4_kernel<DP, WIDE, FINE, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape4<DP>::SMEM);
    if (e != cudaSuccess) return e;
    decode4_kernel<DP, WIDE, FINE, FULL><<<blocks, A4_THREADS, Shape4<DP>::SMEM, stream>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess || a.block_an_item) return e;
    return launch_join<DP>(a, blocks, stream);
}

template <int DP>
cudaError_t launch4_of(const DecodeArgs& a, uint32_t blocks, cudaStream_t stream) {
    const bool full = a.p.c.d == DP;
    if (a.p.dtype == kF32) return full ? launch4<DP, true, true, true>(a, blocks, stream) : launch4<DP, true, true, false>(a, blocks, stream);
    if (a.p.dtype == kF16) return full ? launch4<DP, false, true, true>(a, blocks, stream) : launch4<DP, false, true, false>(a, blocks, stream);
    return full ? launch4<DP, false, false, true>(a, blocks, stream) : launch4<DP, false, false, false>(a, blocks, stream);
}

}  // namespace

cudaError_t launch_attention_decode_int4(const DecodeParams& p, void* workspace, int num_sms, cudaStream_t stream) {
    DecodeArgs a = decode_args(p, workspace, num_sms);
    // A block an item leaves nothing to join, which saves a launch (2 us on the device and 3 on the host), but its warps wait for
    // the longest item. The lengths are on the device, so that the tables' width has to say how long items may be: under a server's
    // tables, as wide as the longest sequence may become, the line of work is taken. A block an item is taken where the SMs have
    // a block for each and the tables allow no more than four tiles a warp, and no more than two above what the line of work
    // gives (calls by it / by the line: 1 x 760 tokens of 8 key heads 12.2 / 14.3 us, 9 x 350 12.0 / 14.3, 18 x 1500 15.3 /
    // 17.4; 1 x 1500 14.8 / 14.4, 9 x 2500 20.4 / 16.9, 16 x 2048 21.0 / 20.5, 37 x 350 in two rounds 16.8 / 16.0).
    const uint64_t items = (uint64_t)p.batch * p.c.heads * a.chunks_of_heads, sms = num_sms;
    const uint64_t tiles = ((uint64_t)p.table_width * p.c.page_size + A4_TOK - 1) / A4_TOK;  // of a sequence at most
    a.block_an_item = items <= sms && tiles <= 4 * A4_WARPS && tiles * (sms - items) <= 2 * A4_WARPS * sms;
    const uint32_t blocks = a.block_an_item ? (uint32_t)items : num_sms;
    return p.c.d > 64 ? launch4_of<128>(a, blocks, stream) : launch4_of<64>(a, blocks, stream);
}

}  // namespace iq2
