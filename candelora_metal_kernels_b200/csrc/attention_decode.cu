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
//   * The key scale multiplies s, the value scale w multiplies p. The reference m of a head's exponents moves when a product
//     p w has grown by more than 2^8, so that p w keeps to the range of f16; the sum of p itself is f32 (int8 caches: held by
//     2^-16 of itself, since p alone may reach 2^122).
// The maxima, sums, s, p and o are f32.
//
// Measured (8 key heads, 128 elements): 128 sequences of up to 4096 tokens, bf16 cache, 214 us: 6260 GB/s, 0.96 of the copy
// rate; one of 100001 tokens, int8 cache and 8 query heads a key head, 49 us: 4300 GB/s, of which about 8 us are start,
// merge of the warps and join, and in the stream the widening of the codes binds as well (issue slots 48 % used); 16 of up to
// 2048, int8, f32 q, 22 us, of which the stream is 7; one of 333 tokens 9.6 us, latencies one after another. 16 of up to
// 2048, f32 q: 24.2 us over an f16 cache, 28.0 over a bf16 one (the third piece); 64 of up to 4096, int8, bf16 q: 89.8 us with
// pages of 64 tokens, 102 with 16 or 48 (a tile of 32 tokens then lies in several pages, and each row is looked up). The parts added
// up inside this kernel (by the block that finishes last) instead of by a dependent launch: 11.4 and 53.8 us for the
// one of 333 and the one of 100001 tokens.
#include "attention_internal.h"
#include "iq2xxs_common.cuh"

#include <algorithm>

namespace iq2 {

namespace {

constexpr int AD_WARPS = 8, AD_THREADS = AD_WARPS * 32, AD_STAGES = 3;
constexpr int AD_HEADS = 8;                     // query heads of an item
// Units' time that starting and ending an item costs. Measured with 1 / 2 / 3: 128 x 4096 tokens 219 / 216 / 214 us,
// 1 x 100001 49.7 / 48.6 / 47.9 us.
constexpr uint32_t AD_ITEM_COST = 3;
// 2^-107, just below the smallest value scale that a row of the cache has (its largest value, 2^-100 or more, over 127). A row of
// zeros has 0 and counts as this, so that the reference stays finite; its codes are zeros.
constexpr float AD_MIN_SCALE = 6.16297582e-33f;
// p times the value scale: the power of two that it has at the reference, and how far it may grow before that moves.
template <bool BF>
constexpr float AD_TOP = BF ? 0.f : 7.f;
template <bool BF>
constexpr float AD_LAZY = BF ? 256.f : 32768.f;
template <bool BF>
constexpr float AD_LOW = BF ? 1.f : 2048.f;      // what low pieces are held times
constexpr float AD_SUM = 1.f / 65536.f;          // int8 caches: what the sums of p, and with them o, are held times
constexpr uint32_t CODE_ZERO = 0x00800080u;      // two codes of 0 as f16: 128 2^-24
constexpr float CODE_UNIT = 16777216.f;          // 2^24
constexpr float LOG2E = 1.44269504f;

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

// What join_kernel's block of the same number has to join: the parts of blocks c0 to c1 of one item, block c0's being its
// part number `slot` (0: its first, 1: its last), the others' their first. c1 = 0: nothing.
struct JoinRecord {
    uint32_t b, item, c0, c1, slot;
};
inline size_t records_bytes(uint32_t blocks) { return (blocks * sizeof(JoinRecord) + 255) / 256 * 256; }

struct DecodeArgs {
    DecodeParams p;
    float* parts;
    JoinRecord* records;
    double inv_blocks;                      // 1 / the blocks of the launch
    uint32_t chunks_of_heads;
    Divisor by_page;                        // tokens of a page
};

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

// Two bytes of codes + 128 as f16: (code + 128) 2^-24, or the codes themselves.
template <bool SHIFTED>
__device__ __forceinline__ uint32_t code_pair(uint32_t bytes, uint32_t sel) {
    if (SHIFTED) return prmt(bytes, 0u, sel);
    const uint32_t u = prmt(bytes, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
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

// The line of work from one unit on: the item it is in and the tokens [t0, t1) of that item in the part. An item's first
// AD_ITEM_COST units have no tokens; a part that ends inside them has none (the next block has the item).
struct Cursor {
    uint64_t unit, end;
    uint32_t b, item, len, units;  // the sequence, its item (key head, group of query heads), tokens and units an item
    uint32_t k, n;                 // first unit of the item in the part, and how many
    uint32_t t0, t1;
    template <int UNIT>
    __device__ __forceinline__ void cut() {
        n = (uint32_t)min((uint64_t)(units - k), end - unit);
        t0 = (max(k, AD_ITEM_COST) - AD_ITEM_COST) * UNIT, t1 = min((max(k + n, AD_ITEM_COST) - AD_ITEM_COST) * UNIT, len);
    }
    template <int UNIT>
    static __device__ __forceinline__ uint32_t units_of(uint32_t len_) { return len_ == 0 ? 0 : (len_ + UNIT - 1) / UNIT + AD_ITEM_COST; }
    __device__ __forceinline__ bool done() const { return unit >= end; }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == len; }
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
            units = units_of<UNIT>(len);
        }
        cut<UNIT>();
        if (t0 == t1) unit = end;
    }
};

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
    uint64_t units = 0;
    uint32_t len = 0;  // of sequence b0 + lane
#pragma unroll 1
    for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
        const uint32_t b = b0 + lane;
        len = b < p.batch ? seq_len(p, b) : 0u;
        units += Cursor::units_of<UNIT>(len);
        // sequences of length 0: zeros, a block a sequence
        uint32_t empty = __ballot_sync(0xFFFFFFFFu, len == 0 && b < p.batch && b % gridDim.x == blockIdx.x);
#pragma unroll 1
        for (; empty != 0; empty &= empty - 1)
#pragma unroll 1
            for (uint32_t i = threadIdx.x; i < p.q_heads * d; i += AD_THREADS)
                store_elem(p.out, (int64_t)(b0 + __ffs(empty) - 1) * p.q_heads * d + i, p.dtype, 0.f);
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) units += __shfl_xor_sync(0xFFFFFFFFu, units, o);
    units *= items;
    uint64_t each = (uint64_t)((double)units * a.inv_blocks);  // units / blocks, rounded up
    while (each * gridDim.x < units) ++each;
    const uint64_t u0 = min(blockIdx.x * each, units), u1 = min(u0 + each, units);
    Cursor cur{};
    if (u0 < u1) {
        uint64_t before = 0;  // units of the sequences before
#pragma unroll 1
        for (uint32_t b0 = 0; b0 < p.batch; b0 += 32) {
            if (p.batch > 32) len = b0 + lane < p.batch ? seq_len(p, b0 + lane) : 0u;
            const uint32_t own = Cursor::units_of<UNIT>(len);
            uint64_t upto = (uint64_t)own * items;
#pragma unroll
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
                cur.unit = u0, cur.end = u1;
                cur.cut<UNIT>();
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
    }
    if (threadIdx.x == 0) {
        // the first block whose part begins inside an item's tokens joins it: the block before it has the first of them
        const uint64_t unit0 = u0 - cur.k;
        JoinRecord r{cur.b, cur.item, blockIdx.x - 1, 0, 0};
        if (cur.t0 > 0 && u0 - each <= unit0 + AD_ITEM_COST) {
            r.c1 = blockIdx.x, r.slot = u0 - each >= unit0 ? 0 : 1;
            while ((r.c1 + 1) * each < unit0 + cur.units) ++r.c1;
        }
        a.records[blockIdx.x] = r;
    }
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
            pre.next<UNIT>(p, items);
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
        float o[NT][4], o_off[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
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

            // x = log2(e) scale q . k, this thread's tokens 8 n + 2 t, + 1 of head g; w = 2^(x - m) times the value scale
            float x[ST][2], e[ST][2], w[ST][2], vs[ST][2];
            const float2* const scales = reinterpret_cast<const float2*>(ring + stage * S::STAGE + 2 * TOK * S::ROW) + t;
#pragma unroll
            for (int n = 0; n < ST; ++n) {
                float2 ks2 = make_float2(factor, factor), vs2 = make_float2(1.f, 1.f);
                if (I8) {
                    const float2 sk = scales[n * 4], sv = scales[TOK / 2 + n * 4];
                    ks2 = make_float2(sk.x * factor, sk.y * factor);
                    vs2 = make_float2(max_nan(sv.x, AD_MIN_SCALE), max_nan(sv.y, AD_MIN_SCALE));
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
                const float base = m == -INFINITY ? 0.f : m - AD_TOP<BF>;
                float top = 0.f;
#pragma unroll
                for (int n = 0; n < ST; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        e[n][j] = exp2_approx(x[n][j] - base);
                        w[n][j] = I8 ? e[n][j] * vs[n][j] : e[n][j];
                        top = fmaxf(top, w[n][j]);
                    }
                if (!__any_sync(0xFFFFFFFFu, top > AD_LAZY<BF> || m == -INFINITY)) break;
                // the largest x + log2(value scale) of the head's tokens
                float most = -INFINITY;
#pragma unroll
                for (int n = 0; n < ST; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) most = fmaxf(most, I8 ? x[n][j] + __log2f(vs[n][j]) : x[n][j]);
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
                const float next = fmaxf(m, most), keep = m == -INFINITY ? 0.f : exp2_approx(m - next);
                const bool moved = next > m;
                if (!__any_sync(0xFFFFFFFFu, moved)) break;
                if (moved) {
                    m = next;
                    l *= keep;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[n][j] *= keep;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o_off[j] *= keep;
                }
            }
            uint32_t pa[TOK / 16][4], pa3[TOK / 16][4];
#pragma unroll
            for (int n = 0; n < ST; ++n) {
                l = fmaf(e[n][0] + e[n][1], I8 ? AD_SUM : 1.f, l);
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
        if (I8) {  // the 128s off, and the codes' unit and the sums' on
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][j] = SHIFTED ? (o[n][j] - o_off[j]) * (CODE_UNIT * AD_SUM) : o[n][j] * AD_SUM;
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
            float* const part = a.parts + ((uint64_t)blockIdx.x * 2 + (cur.unit == u0 ? 0 : 1)) * S::PART;
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
    join_kernel(const __grid_constant__ DecodeArgs a) {
    const DecodeParams& p = a.p;
    const uint32_t chunks_of_heads = a.chunks_of_heads;
    constexpr int PART = AD_HEADS * (DP + 2);
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_wait();
    const JoinRecord r = a.records[blockIdx.x];
    if (r.c1 == 0) return;
    const uint32_t d = p.c.d, group = p.q_heads / p.c.heads;
    const uint32_t kv_head = r.item / chunks_of_heads, head0 = kv_head * group + (r.item % chunks_of_heads) * AD_HEADS;
    if (warp >= min((uint32_t)AD_HEADS, (kv_head + 1) * group - head0)) return;
    auto slot = [&](uint32_t c) { return a.parts + ((uint64_t)c * 2 + (c == r.c0 ? r.slot : 0)) * PART; };
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
#pragma unroll 8
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

template <int DP, int KIND, bool WIDE>
cudaError_t launch(const DecodeArgs& a, uint32_t blocks, cudaStream_t stream) {
    using S = DecodeShape<DP, KIND, WIDE>;
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<DP, KIND, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    // (the second kernel keeps the first one's split of shared memory: changing it would drain the SMs twice a call)
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(join_kernel<DP>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    decode_kernel<DP, KIND, WIDE><<<blocks, AD_THREADS, S::SMEM, stream>>>(a);
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
    return cudaLaunchKernelEx(&cfg, join_kernel<DP>, a);
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
    const uint32_t unit = c.dtype == kInt8 ? DecodeShape<64, CK_INT8, false>::UNIT : DecodeShape<64, CK_F16, false>::UNIT;
    const uint64_t tokens = std::min<uint64_t>((uint64_t)table_width * c.page_size, INT32_MAX);
    const uint64_t items = (uint64_t)c.heads * ((q_heads / c.heads + AD_HEADS - 1) / AD_HEADS);
    return ((tokens + unit - 1) / unit + AD_ITEM_COST) * items <= (uint64_t)UINT32_MAX;
}

size_t attention_decode_workspace(uint32_t, uint32_t, uint32_t, uint32_t d, int num_sms) {
    return records_bytes(num_sms) + (size_t)num_sms * 2 * AD_HEADS * ((d > 64 ? 128 : 64) + 2) * sizeof(float);
}

cudaError_t launch_attention_decode(const DecodeParams& p, void* workspace, int num_sms, cudaStream_t stream) {
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    const DecodeArgs a{p, reinterpret_cast<float*>(ws + records_bytes(num_sms)), reinterpret_cast<JoinRecord*>(ws), 1.0 / num_sms,
                 (p.q_heads / p.c.heads + AD_HEADS - 1) / AD_HEADS, Divisor::of(p.c.page_size)};
    return p.c.d > 64 ? launch_kind<128>(a, num_sms, stream) : launch_kind<64>(a, num_sms, stream);
}

}  // namespace iq2
