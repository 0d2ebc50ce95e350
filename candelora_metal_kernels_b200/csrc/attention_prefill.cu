// Attention of packed prompts on the sm_100a tensor cores: for query i of a sequence with Lq queries and Lk keys
//     o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  j < Lk, and j <= i + Lk - Lq if causal.
//
// An item is two tiles of 128 rows of one key head. The rows of a tile are (token, head) pairs, the G query heads of the
// key head packed beside each other (TPT = 128 / G tokens a tile), so that each K and V tile that is loaded serves all of
// them and short prompts still fill the rows. Over tiles of 128 keys, with the running maximum and sum of a softmax:
//   S_i = Q_i K^T   tcgen05.mma, M = N = 128, into TMEM (f32)                          one MMA warp for both tiles
//   P_i = 2^(c S - m), rounded to the inputs' 16-bit type (by 2^-8 or 2^-11 of itself, as the output's own rounding; f16 see
//         below), written over S_i in TMEM; the sum is of the f32 values                a warpgroup a tile, a thread a row
//   O_i += P_i V    tcgen05.mma with A = P_i from TMEM, V as the N-major operand
// The two tiles alternate on the tensor core: while one warpgroup computes its exponentials the other's products run.
// K and V tiles arrive by TMA (128-byte swizzle, no multicast) in one ring, K_0 V_0 K_1 V_1 ..., across items.
//   * Work: one block an SM stays for the whole call. The items, each as long as its keys and AP_ITEM_COST more, form one
//     line, of which each block takes an equal contiguous part (short calls: whole items, see Work). A part that is
//     not a whole item leaves (o, m, l) in the workspace, unless it is the item's last one: that adds the parts up
//     (attention_parts.cuh), beside the other blocks' work and without a launch or a wait of its own.
//   * Lazy rescaling: the reference m of a row moves only when a score exceeds it by more than 2^8 (bf16) or 2^4 (f16), so
//     that O in TMEM is rescaled a few times a row instead of once a tile. f16 has no exponents to spare: where one token
//     takes nearly all of a row's weight, the output may be made of p far below it. So p is 2^11 at the reference (2^15 at
//     most) and keeps its eleven bits down to 2^-25 of the row's largest, 17.3 nats; below that its last bit is 2^-35 of the
//     largest. 512 tokens after 7001 in f16 take 274 us with this, 264 with 2^8 above 2^7, 282 with 2^2 above 2^13.
//   * Masked keys are replaced by -inf before the maximum (never added to), so that whatever K holds there cannot matter.
//     V needs more, since 0 * NaN is NaN: two guard warps look through the V tiles that hold keys some row does not see.
//     Rows past the last visible key (other sequences' tokens) become zeros; infinities and NaN of keys that only some
//     rows see become zeros too, and the epilogue adds them back to exactly the rows that see them.
// What bounds it: per pair of key tiles the four products take 2048 cycles of the tensor core; the step takes 3100 to 3400,
// since a row's softmax (load, maximum, 128 exponentials and their rounding, store: about 2000, of which the exponentials
// are 1500: 1024 at the exponential unit's own rate, which needs 2048 for both row tiles, as the tensor core does, and the
// rest latency and issue) and its products with their handshakes (about 1080) follow one another and the
// other tile fills only part of the gap. Two tiles of 128 rows and five K or V tiles of 32 KB are what shared memory and
// TMEM hold at 128 elements (at 64, TMEM has 128 columns to spare). Measured (32 query heads, 8 key heads, 128 elements, bf16, causal): 16384 tokens 1.73 to 1.89 ms, 1160 to 1270
// TFLOP/s, with the tensor pipe busy 62 % of the time; 2048 tokens 56 us, where an item's start and end (3 tiles' time) and
// the kernel's (about 4 us) are a third; a batch of nine prompts of up to 200 tokens 26.4 us, all of it such latencies.
// 64 elements: 8192 tokens 375 us, 730 TFLOP/s; 2048 tokens 45 us.
// Every wait is bounded by wall time (device_status); a block that gives up still drains its copies and frees its TMEM.
#include "attention_internal.h"
#include "attention_parts.cuh"
#include "iq2xxs_internal.h"
#include "tcgen05.cuh"

#include <cstring>

namespace iq2 {

namespace {

constexpr int AP_ROWS = 128, AP_KEYS = 128;
constexpr int AP_MMA_WARP = 8, AP_TMA_WARP = 9, AP_GUARD_WARP = 10, AP_THREADS = 12 * 32;  // warps 0-7: softmax
constexpr uint32_t AP_LOAD = 0x100u, AP_RELEASE = 0x200u, AP_PROB = 0x400u, AP_PRODUCT = 0x800u;  // status bits
// In powers of two: how far a score may exceed its row's reference, and p at the reference (f16: together below its 2^16).
template <bool BF>
constexpr float ap_lazy = BF ? 8.f : 4.f;
template <bool BF>
constexpr float ap_top = BF ? 0.f : 11.f;
constexpr int AP_FIRST = 6;      // of the eight steps of 16 keys of P V, those that begin before the rest of P is there
constexpr int AP_ITEM_ROWS = 2 * AP_ROWS;
// Keys' time that an item costs besides its keys, and that leaving and joining a part costs. Measured: 16384 tokens
// 1799 / 1722 / 1735 us with 2 / 3 / 4 tiles an item, 2048 tokens 59 us with each.
constexpr int32_t AP_ITEM_COST = 3 * AP_KEYS, AP_SPLIT_COST = 3 * AP_KEYS;
// setmaxnreg: 8 softmax warps and 4 others share what the launch holds, 12 x 32 x 168
constexpr int AP_REGS_SOFTMAX = 208, AP_REGS_OTHER = 88;
static_assert(8 * AP_REGS_SOFTMAX + 4 * AP_REGS_OTHER <= 12 * 168, "register shares");

constexpr int AP_PARTS = 4, AP_PART_BYTES = 80;  // parts of items on their way between the warps

template <int DP>
struct PrefillShape {
    static constexpr int TILE = 128 * DP * 2;           // bytes of 128 rows of q, k or v
    static constexpr int SLOTS = DP == 128 ? 5 : 8;     // K and V tiles in flight
    static constexpr int BARS = 2 + 2 * SLOTS + 15 + 2 * AP_PARTS;
    static constexpr int SMEM = (2 + SLOTS) * TILE + BARS * 8 + 16 + AP_PARTS * AP_PART_BYTES;
};

// A part of an item in the workspace: o [d / 4][256 rows][4], then the rows' references (in powers of two) and sums.
constexpr uint32_t part_floats(int dp) { return AP_ITEM_ROWS * (dp + 2); }

struct PrefillArgs {
    RowsView v;
    void* out;
    uint32_t* flags;  // see attention_parts.cuh
    float* parts;
    const int32_t *cu_q, *cu_k;
    unsigned int* status;
    uint64_t wait_ns;
    uint32_t stall;
    uint32_t seqs, q_tokens, k_tokens, q_heads, kv_heads, group, tpt, d;
    double inv_blocks;  // 1 / the blocks of the launch
    float c;            // scale log2(e)
    bool causal, out32;  // out32: the output's rows start on 32-byte boundaries
};

// Instruction descriptor, kind::f16: f32 accumulator, f16 or bf16 operands, M = 128; n: columns; B N-major for P V.
__device__ __forceinline__ uint32_t idesc16(bool bf, uint32_t n, bool b_nmajor) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((b_nmajor ? 1u : 0u) << 16) | ((n >> 3) << 17) | (8u << 24);
}

// Shared-memory matrix descriptors as two words, of which only the low one (the address in 16-byte units, and the stride
// between 64-column blocks) changes from step to step. Q and K: K-major rows of 128 bytes, groups of 8 rows 1024 bytes
// apart. V as the N-major operand: 64-column blocks of 128 keys x 128 bytes (16 KB apart), groups of 8 keys 1024 bytes
// apart. All with the 128-byte swizzle.
constexpr uint32_t AP_DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t kmajor_low(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t nmajor_low(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | ((16384u >> 4) << 16); }

// The MMA warp runs as a whole and one elected lane issues: in code that all lanes share the descriptors stay in uniform
// registers, where the instruction wants them (issued from a one-lane branch each product cost 110 to 150 cycles of
// register moves, more than the tensor core's own time).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_ss(uint32_t elected, uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(elected), "r"(AP_DESC_HIGH)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t elected, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 b, {%2, %6};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(elected), "r"(AP_DESC_HIGH)
        : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t elected, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(elected)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// 32 columns of this warp's 32 TMEM lanes; the values may be used after tmem_ld_wait, which the pins order them behind.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void pin32(float* v) {
    asm volatile(""
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                   "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
                   "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ void pin16(float* v) {
    asm volatile(""
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
        : "memory");
}

// 32 bytes, as one whole sector where the address allows.
__device__ __forceinline__ void store32(void* p, uint4 a, uint4 b, bool aligned) {
    if (aligned)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
                     "r"(b.y), "r"(b.z), "r"(b.w)
                     : "memory");
    else
        static_cast<uint4*>(p)[0] = a, static_cast<uint4*>(p)[1] = b;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two f32 values side by side (add, sub and fma of both in one instruction).
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float first_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float second_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// One test of a phase, without a time to sleep inside it: a sleep is longer than most waits here.
__device__ __forceinline__ bool try_bar(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}

// A bounded wait of the block: false when it ran out, or when another role of the block gave up. The waiting itself is a
// function of its own (as the steps from item to item are): the kernel waits in many places, and once its code no longer
// fits the instruction cache everything in it takes twice as long.
__device__ __forceinline__ bool wait_more(uint32_t bar, uint32_t parity, uint64_t limit, unsigned int* status, uint32_t code,
                                       volatile uint32_t* abort_flag) {
    const uint64_t t0 = global_ns();
#pragma unroll 1
    for (uint32_t tries = 1;; ++tries) {
        if (try_bar(bar, parity)) return true;
        if (tries % 64 != 0) continue;
        if (*abort_flag != 0u) return false;
        if (global_ns() - t0 > limit) {
            atomicOr(status, code);
            *abort_flag = 1u;
            return false;
        }
    }
}
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const PrefillArgs& p, uint32_t code, volatile uint32_t* abort_flag) {
    return try_bar(bar, parity) || wait_more(bar, parity, p.wait_ns, p.status, code, abort_flag);
}

// The line of work, from one point of it on, worked out by each warp for itself. Lengths are clamped to the tensors, so
// that no index leads outside them. Items are ordered by sequence, then token, then key head. An item is AP_ITEM_COST (its
// start and end) and then its visible keys long: sums over a sequence's items are sums of an arithmetic progression. A part
// [x, y) of an item has the key tiles from tile_at(x) to tile_at(y); every block's part is at least a tile long, so none of
// the blocks between an item's first and last is without a step of it. Splitting items costs a part written and joined,
// about AP_SPLIT_COST: where whole items, dealt by number, end no later by that measure, they stay whole (a batch of short
// prompts).
struct Work {
    // lane l: sequence b0 + l
    int32_t lane_q0, lane_lq, lane_k0, lane_lk;
    uint32_t b0;
    // the item, and the key tiles [j0, j1) of its n in this part
    uint32_t b, kv_head;
    int32_t tok0, n, j0, j1;
    int32_t pos, to;     // the part of the item's length
    uint64_t at, each;   // where the part begins in the line, and the blocks' share of it
    uint64_t left;    // of the block's part of the line, from this part on (whole items: their number)
    bool by_items;
    // its sequence and tiles
    int32_t q0, lq, k0, lk, least, most;  // least, most: visible keys of the item's first and last token
    int32_t tiles[2], masked;             // key tiles that tile i sees anything of; from `masked` on, some row sees part

    __device__ __forceinline__ void load_group(const PrefillArgs& p, uint32_t first) {
        b0 = first;
        const uint32_t s = first + threadIdx.x % 32;
        const int32_t tq = (int32_t)p.q_tokens, tk = (int32_t)p.k_tokens;
        lane_q0 = lane_lq = lane_k0 = lane_lk = 0;
        if (s < p.seqs) {
            const int32_t q_a = __ldg(p.cu_q + s), q_b = __ldg(p.cu_q + s + 1), k_a = __ldg(p.cu_k + s), k_b = __ldg(p.cu_k + s + 1);
            lane_q0 = min(max(q_a, 0), tq), lane_k0 = min(max(k_a, 0), tk);
            lane_lq = max(min(q_b, tq) - lane_q0, 0), lane_lk = max(min(k_b, tk) - lane_k0, 0);
        }
    }
    static __device__ __forceinline__ int32_t shown(const PrefillArgs& p, int32_t lq_, int32_t lk_, int32_t tok) {
        return p.causal ? max(min(lk_, tok + 1 + lk_ - lq_), 0) : lk_;
    }
    // Length of the items of one key head before block t of a sequence (t < its blocks).
    static __device__ __forceinline__ int64_t before(const PrefillArgs& p, int32_t lq_, int32_t lk_, int32_t t) {
        if (!p.causal) return (int64_t)t * (AP_ITEM_COST + lk_);
        const int32_t step = 2 * (int32_t)p.tpt, shift = lk_ - lq_;
        const int32_t z = shift < 0 ? min((int32_t)((uint32_t)-shift / (uint32_t)step), t) : 0;  // blocks that see no key
        const uint64_t steps = ((uint64_t)t * (uint32_t)(t + 1) - (uint64_t)z * (uint32_t)(z + 1)) >> 1;
        return (int64_t)t * AP_ITEM_COST + (int64_t)(steps * (uint32_t)step) + (int64_t)(t - z) * shift;
    }
    __device__ __forceinline__ int32_t tile_at(int32_t x) const {
        return x >= AP_ITEM_COST + most ? n : (max(x - AP_ITEM_COST, 0) + AP_KEYS - 1) / AP_KEYS;
    }
    __device__ __forceinline__ void enter_sequence() {
        const int s = (int)(b - b0);
        q0 = __shfl_sync(0xFFFFFFFFu, lane_q0, s), lq = __shfl_sync(0xFFFFFFFFu, lane_lq, s);
        k0 = __shfl_sync(0xFFFFFFFFu, lane_k0, s), lk = __shfl_sync(0xFFFFFFFFu, lane_lk, s);
    }
    __device__ __forceinline__ void enter_item(const PrefillArgs& p) {
        const int32_t tpt = (int32_t)p.tpt, last = min(tok0 + 2 * tpt, lq) - 1;
        least = shown(p, lq, lk, tok0), most = shown(p, lq, lk, last);
        tiles[0] = (shown(p, lq, lk, min(tok0 + tpt - 1, last)) + AP_KEYS - 1) / AP_KEYS;
        tiles[1] = tok0 + tpt < lq ? (most + AP_KEYS - 1) / AP_KEYS : 0;
        n = max(max(tiles[0], tiles[1]), 1);
        masked = least / AP_KEYS;
        const int32_t length = AP_ITEM_COST + most;
        to = by_items ? length : (int32_t)min((uint64_t)length, pos + left);
        j0 = tile_at(pos), j1 = tile_at(to);
    }
    __device__ __forceinline__ bool done() const { return left == 0; }
    __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == n; }
    // steps of tile i in this part: [j0, end(i))
    __device__ __forceinline__ int32_t end(int i) const { return min(j1, tiles[i]); }
    // The next part that has key tiles (the first or last bit of an item may have none).
    __device__ __forceinline__ void next(const PrefillArgs& p) {
        do {
            left -= by_items ? 1 : (uint64_t)(to - pos), at += (uint64_t)(to - pos);
            if (done()) return;
            pos = 0;
            if (++kv_head == p.kv_heads) {
                kv_head = 0;
                tok0 += 2 * (int32_t)p.tpt;
                if (tok0 >= lq) {
                    tok0 = 0;
                    do {
                        if (++b >= p.seqs) {  // (not reached while the lengths stay as they were)
                            left = 0;
                            return;
                        }
                        if (b - b0 == 32) load_group(p, b);
                        enter_sequence();
                    } while (lq == 0);
                }
            }
            enter_item(p);
        } while (j0 == j1);
    }
    // The blocks that have key tiles of the item, and the place of block c0's part: 1 where that block begins in an earlier
    // item (which then has place 0, if it has key tiles there).
    __device__ __forceinline__ void sharers(uint32_t* c0, uint32_t* c1, uint32_t* slot) const {
        *c0 = *c1 = blockIdx.x, *slot = 0;
        if (whole()) return;
        const uint64_t item = at - (uint64_t)pos, first = item + AP_ITEM_COST, last = first + (uint32_t)((n - 1) * AP_KEYS);
        while (*c0 * each > first) --*c0;
        while ((*c1 + 1) * each <= last) ++*c1;
        *slot = *c0 * each >= item ? 0 : 1;
    }
    // The block's part of the line; false if there is none. (Runs once, but from a cold instruction cache: without 64-bit
    // divisions it is a quarter of the code.) Every block but the last has `each` of the line.
    __device__ __noinline__ bool begin(const PrefillArgs& p) {
        const uint32_t lane = threadIdx.x % 32, step = 2 * p.tpt;
        uint64_t total = 0, sum = 0;
        uint32_t items = 0;
        int32_t longest = 0;
        auto group_length = [&]() {  // of one key head's items of each lane's sequence
            const int32_t blocks = (int32_t)(((uint32_t)lane_lq + step - 1) / step);
            return blocks > 0 ? (uint64_t)before(p, lane_lq, lane_lk, blocks - 1) + (uint32_t)(AP_ITEM_COST + lane_lk) : 0;
        };
#pragma unroll 1
        for (uint32_t s = 0; s < p.seqs; s += 32) {
            load_group(p, s);
            total += group_length();
            items += ((uint32_t)lane_lq + step - 1) / step, longest = max(longest, lane_lk);
        }
#pragma unroll 1
        for (int o = 16; o > 0; o /= 2) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        items = __reduce_add_sync(0xFFFFFFFFu, items) * p.kv_heads;
        longest = __reduce_max_sync(0xFFFFFFFFu, longest);
        total *= p.kv_heads;
        const uint32_t item_share = (items + gridDim.x - 1) / gridDim.x;
        const uint64_t share = (uint64_t)((double)total * p.inv_blocks) + 1;  // a little over its part of the line
        by_items = (uint64_t)item_share * (uint32_t)(AP_ITEM_COST + longest) <= share + AP_SPLIT_COST;
        each = by_items ? item_share : max(share, (uint64_t)AP_KEYS), at = blockIdx.x * each;
        const uint64_t all = by_items ? items : total, u0 = min(at, all);
        left = min(u0 + each, all) - u0;
        if (left == 0) return false;
#pragma unroll 1
        for (uint32_t s = 0;; s += 32) {
            if (s >= p.seqs) return false;  // (not reached while the lengths stay as they were)
            if (b0 != s) load_group(p, s);
            const uint64_t own = (by_items ? ((uint32_t)lane_lq + step - 1) / step : group_length()) * p.kv_heads;
            uint64_t upto = own;
#pragma unroll 1
            for (int o = 1; o < 32; o *= 2) {
                const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                if (lane >= (uint32_t)o) upto += x;
            }
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, sum + upto > u0);
            if (hit != 0) {
                const int at = __ffs(hit) - 1;
                b = s + at;
                sum += __shfl_sync(0xFFFFFFFFu, upto - own, at);
                break;
            }
            sum += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
        enter_sequence();
        uint64_t rest = u0 - sum;
        pos = 0;
        if (by_items) {
            tok0 = (int32_t)((uint32_t)rest / p.kv_heads * step), kv_head = (uint32_t)rest % p.kv_heads;
        } else {  // the last block t of tokens that begins at or before `rest`, 32 candidates at a time
            int32_t lo = 0, hi = (int32_t)(((uint32_t)lq + step - 1) / step);
#pragma unroll 1
            while (hi - lo > 1) {
                const int32_t stride = (hi - lo + 31) / 32, t = min(lo + (int32_t)lane * stride, hi - 1);
                const uint32_t in = __ballot_sync(0xFFFFFFFFu, before(p, lq, lk, t) * (int64_t)p.kv_heads <= (int64_t)rest);
                lo = min(lo + (__popc(in) - 1) * stride, hi - 1), hi = min(lo + stride, hi);
            }
            rest -= before(p, lq, lk, lo) * (int64_t)p.kv_heads;
            tok0 = lo * (int32_t)step;
            const uint32_t length = AP_ITEM_COST + shown(p, lq, lk, min(tok0 + (int32_t)step, lq) - 1);
            kv_head = (uint32_t)rest / length, pos = (int32_t)((uint32_t)rest % length);
        }
        enter_item(p);
        if (j0 == j1) next(p);
        return !done();
    }
};

// What the other warps need of a part of an item, handed on by the TMA warp, which alone walks the line.
struct Part {
    int32_t j0, j1, end0, end1;        // its key tiles; those of either tile of rows
    int32_t masked, least, most;       // see Work
    int32_t row0, tokens;              // the item's first token in the packed tensors; tokens of the sequence from it on
    int32_t seen0, keys;               // keys that the first token sees less one (before clamping to 0 .. keys)
    int32_t k0, kv_head, whole, more;  // more = 0: no further part
    uint32_t c0, c1, slot;             // see PartSet
};
static_assert(sizeof(Part) <= AP_PART_BYTES, "a part's place");

template <int DP, bool BF>
__global__ void __launch_bounds__(AP_THREADS, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PrefillArgs p) {
    using S = PrefillShape<DP>;
    constexpr int SLOTS = S::SLOTS, HALVES = DP / 64;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + 2 * S::TILE, bars = ring + SLOTS * S::TILE;
    volatile uint32_t* const words = reinterpret_cast<volatile uint32_t*>(smem + (2 + SLOTS) * S::TILE + S::BARS * 8);
    Part* const parts = reinterpret_cast<Part*>(smem + (2 + SLOTS) * S::TILE + S::BARS * 8 + 16);
    volatile uint32_t* const abort_flag = words + 1;
    volatile uint32_t* const odd_values = words + 2;  // the guard found infinities or NaN
    auto q_full = [&](int i) { return bars + i * 8; };
    auto full = [&](uint32_t s) { return bars + 16 + s * 8; };
    auto empty = [&](uint32_t s) { return bars + 16 + (SLOTS + s) * 8; };
    const uint32_t more = bars + 16 + 2 * SLOTS * 8;
    auto s_full = [&](int i) { return more + i * 8; };
    auto p_ready = [&](int i) { return more + 16 + i * 8; };  // the first AP_FIRST steps' P
    auto p_rest = [&](int i) { return more + 32 + i * 8; };
    auto o_full = [&](int i) { return more + 48 + i * 8; };
    auto o_empty = [&](int i) { return more + 64 + i * 8; };
    auto q_empty = [&](int i) { return more + 80 + i * 8; };
    const uint32_t v_landed = more + 96, v_safe = more + 104, drained = more + 112;
    auto part_full = [&](uint32_t s) { return more + 120 + s * 8; };
    auto part_empty = [&](uint32_t s) { return more + 120 + (AP_PARTS + s) * 8; };
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full(i), 1), mbar_init(q_empty(i), 1), mbar_init(s_full(i), 1), mbar_init(o_full(i), 1);
            mbar_init(p_ready(i), 4), mbar_init(p_rest(i), 4), mbar_init(o_empty(i), 4);
        }
        for (int s = 0; s < SLOTS; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
        for (int s = 0; s < AP_PARTS; ++s) mbar_init(part_full(s), 1), mbar_init(part_empty(s), 11);  // 8 softmax, 2 guard, MMA
        mbar_init(v_landed, 1), mbar_init(v_safe, 2), mbar_init(drained, 1);
        fence_barrier_init();
        *abort_flag = 0u;
        *odd_values = 0u;
    }
    if (warp == AP_MMA_WARP) tmem_alloc<false>(smem_u32(const_cast<uint32_t*>(words)), 512);
    pdl_wait();  // (the flags are down)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, words[0], 0);
    auto s_col = [&](int i) { return tmem + i * 128; };
    auto o_col = [&](int i) { return tmem + 256 + i * 128; };
    const int32_t tpt = (int32_t)p.tpt;

    // The next part, or false after the last one (or when a wait ran out); each reader gives its place back when done.
    uint32_t read = 0;
    auto next_part = [&](Part& part) {
        const uint32_t s = read % AP_PARTS;
        if (!__all_sync(0xFFFFFFFFu, wait_bar(part_full(s), (read / AP_PARTS) & 1, p, AP_LOAD, abort_flag))) return false;
        part = parts[s];
        __syncwarp();
        if (lane == 0) mbar_arrive(part_empty(s));
        ++read;
        return part.more != 0;
    };
    uint32_t issued = 0, q_issued[2] = {0, 0};  // K and V tiles, Q tiles (TMA warp)
    if (warp >= AP_MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AP_REGS_OTHER));
        if (warp == AP_TMA_WARP) {
            bool ok = true;
            uint32_t slot = 0, lap = 0, written = 0;
            Work w;
            if (!w.begin(p)) w.left = 0;
            auto load_kv = [&](const CUtensorMap* map, int32_t j) {
                if (lap > 0 && ok) ok = __all_sync(0xFFFFFFFFu, wait_bar(empty(slot), (lap - 1) & 1, p, AP_RELEASE, abort_flag));
                if (!ok) return;
                if (lane == 0) {
                    mbar_expect_tx(full(slot), S::TILE);
                    for (int h = 0; h < HALVES; ++h)
                        tma_load_3d(ring + slot * S::TILE + h * 16384, map, full(slot), h * 64, (int)w.kv_head, w.k0 + j * AP_KEYS);
                }
                ++issued;
                if (++slot == SLOTS) slot = 0, ++lap;
            };
            auto load_q = [&](int i) {
                if (!ok || w.j0 >= w.end(i)) return;
                if (q_issued[i] > 0) ok = __all_sync(0xFFFFFFFFu, wait_bar(q_empty(i), (q_issued[i] - 1) & 1, p, AP_RELEASE, abort_flag));
                if (!ok) return;
                if (lane == 0) {
                    mbar_expect_tx(q_full(i), HALVES * p.tpt * p.group * 128);
                    for (int h = 0; h < HALVES; ++h)
                        tma_load_4d(q_smem + i * S::TILE + h * 16384, &qmap, q_full(i), h * 64, 0, (int)w.kv_head, w.q0 + w.tok0 + i * tpt);
                }
                ++q_issued[i];
            };
#pragma unroll 1
            for (bool more_parts = true; ok && more_parts; ++written) {
                const uint32_t s = written % AP_PARTS;
                if (written >= AP_PARTS) ok = __all_sync(0xFFFFFFFFu, wait_bar(part_empty(s), (written / AP_PARTS - 1) & 1, p, AP_RELEASE, abort_flag));
                if (!ok) break;
                more_parts = !w.done();
                uint32_t c0 = 0, c1 = 0, first_slot = 0;
                if (more_parts) w.sharers(&c0, &c1, &first_slot);
                if (lane == 0) {
                    parts[s] = {w.j0, w.j1, w.end(0), w.end(1), w.masked, w.least, w.most, w.q0 + w.tok0, w.lq - w.tok0,
                                p.causal ? w.tok0 + w.lk - w.lq : w.lk - 1, w.lk, w.k0, (int32_t)w.kv_head, w.whole() ? 1 : 0, more_parts ? 1 : 0, c0, c1, first_slot};
                    mbar_arrive(part_full(s));
                }
                if (!more_parts) break;
                const int32_t last = max(w.end(0), w.end(1));
                load_q(0);
#pragma unroll 1
                for (int32_t j = w.j0; j < last && ok; ++j) {
#pragma unroll 1
                    for (int v = 0; v < 2; ++v) {
                        load_kv(v ? &vmap : &kmap, j);
                        if (j == w.j0 && v == 0) load_q(1);
                    }
                }
                w.next(p);
            }
        } else if (warp == AP_MMA_WARP) {
            const uint32_t elected = elect_one();
            const uint32_t id_s = idesc16(BF, AP_KEYS, false), id_o = idesc16(BF, p.d, true);
            bool ok = true;
            uint32_t ks = 0, k_lap = 0, vs = 1, v_lap = 0;         // ring slots of the K and V tiles next in line
            uint32_t items[2] = {0, 0}, steps[2] = {0, 0}, guards = 0;  // parts and steps of each tile so far, guarded V tiles
            auto wait = [&](uint32_t bar, uint32_t count, uint32_t code) {
                if (ok) ok = __all_sync(0xFFFFFFFFu, wait_bar(bar, count & 1, p, code, abort_flag));
            };
            const uint32_t q_low = kmajor_low(q_smem), ring_k = kmajor_low(ring), ring_v = nmajor_low(ring);
            auto products_s = [&](int i, bool last) {
                const uint32_t k_low = __shfl_sync(0xFFFFFFFFu, ring_k + ks * (S::TILE >> 4), 0);  // (uniform, and known to be)
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const uint32_t at = ((k / 4) * 16384 + (k % 4) * 32) >> 4;
                    if (k * 16 < (int)p.d) mma_ss(elected, s_col(i), q_low + i * (S::TILE >> 4) + at, k_low + at, id_s, k > 0);
                }
                commit_if(elected, s_full(i));
                if (last) commit_if(elected, q_empty(i));
            };
            auto k_done = [&]() {
                commit_if(elected, empty(ks));
                if ((ks += 2) >= SLOTS) ks -= SLOTS, ++k_lap;
            };
            Part w;
#pragma unroll 1
            while (ok && next_part(w)) {
                const int32_t j0 = w.j0, ends[2] = {w.end0, w.end1}, last = max(ends[0], ends[1]);
                if (j0 >= last) continue;  // an item without keys
                wait(full(ks), k_lap, AP_LOAD);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (j0 >= ends[i]) continue;
                    wait(q_full(i), items[i], AP_LOAD);
                    if (ok) products_s(i, j0 + 1 == ends[i]);
                }
                if (ok) k_done();
                // V tiles with masked keys go to the guard when they have landed: a step before they are wanted, if they have
                int32_t passed = max(j0, w.masked);
#pragma unroll 1
                for (int32_t j = j0; j < last && ok; ++j) {
                    wait(full(vs), v_lap, AP_LOAD);
                    if (passed == j && j < last) {
                        if (ok && lane == 0) mbar_arrive(v_landed);
                        ++passed;
                    }
                    if (j >= w.masked) wait(v_safe, guards++, AP_LOAD);
                    if (passed == j + 1 && j + 1 < last) {
                        const bool wraps = vs + 2 >= SLOTS;
                        if (__all_sync(0xFFFFFFFFu, try_bar(full(wraps ? vs + 2 - SLOTS : vs + 2), (v_lap + (wraps ? 1 : 0)) & 1))) {
                            if (lane == 0) mbar_arrive(v_landed);
                            ++passed;
                        }
                    }
                    if (j + 1 < last) wait(full(ks), k_lap, AP_LOAD);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (j >= ends[i]) continue;
                        if (j == j0 && items[i] > 0) wait(o_empty(i), items[i] - 1, AP_PROB);
                        wait(p_ready(i), steps[i], AP_PROB);
                        if (!ok) continue;
                        tc_fence_after();
                        const uint32_t v_low = __shfl_sync(0xFFFFFFFFu, ring_v + vs * (S::TILE >> 4), 0);
#pragma unroll
                        for (int k = 0; k < AP_FIRST; ++k)
                            mma_ts(elected, o_col(i), s_col(i) + k * 8, v_low + k * (2048 >> 4), id_o, (j > j0 || k > 0) ? 1u : 0u);
                        wait(p_rest(i), steps[i], AP_PROB);
                        if (!ok) continue;
                        tc_fence_after();
#pragma unroll
                        for (int k = AP_FIRST; k < AP_KEYS / 16; ++k)
                            mma_ts(elected, o_col(i), s_col(i) + k * 8, v_low + k * (2048 >> 4), id_o, 1u);
                        ++steps[i];
                        if (j + 1 < ends[i]) products_s(i, j + 2 == ends[i]);
                        else commit_if(elected, o_full(i)), ++items[i];
                    }
                    if (!ok) break;
                    commit_if(elected, empty(vs));
                    if ((vs += 2) >= SLOTS) vs -= SLOTS, ++v_lap;
                    if (j + 1 < last) k_done();
                }
            }
            if (!ok) {  // what was issued ends before the TMEM is freed
                commit_if(elected, drained);
                mbar_wait(drained, 0, p.status, AP_PRODUCT, p.wait_ns);
            }
        } else {
            const uint32_t tid = threadIdx.x - AP_GUARD_WARP * 32;
            // rows of no sequence (before the first or after the last one) are zeros
            const uint32_t first = (uint32_t)min(max(__ldg(p.cu_q), 0), (int32_t)p.q_tokens);
            const uint32_t last_end = (uint32_t)min(max(__ldg(p.cu_q + p.seqs), 0), (int32_t)p.q_tokens);
            const uint32_t row_chunks = p.q_heads * (p.d / 8);  // of 16 bytes
#pragma unroll 1
            for (uint32_t r = blockIdx.x; r < first + (p.q_tokens - last_end); r += gridDim.x) {
                uint4* const out = static_cast<uint4*>(p.out) + (int64_t)(r < first ? r : last_end + (r - first)) * row_chunks;
#pragma unroll 1
                for (uint32_t x = tid; x < row_chunks; x += 64) out[x] = make_uint4(0, 0, 0, 0);
            }
            uint32_t vs = 1, v_lap = 0, guards = 0;
            bool ok = true;
            Part w;
#pragma unroll 1
            while (ok && next_part(w)) {
                const int32_t last = max(w.end0, w.end1);
#pragma unroll 1
                for (int32_t j = w.j0; j < last && ok; ++j) {
                    if (j >= w.masked) {
                        // (the MMA warp passes each tile on: waiting on its load from here could meet the ring a lap away)
                        ok = __all_sync(0xFFFFFFFFu, wait_bar(v_landed, guards & 1, p, AP_LOAD, abort_flag));
                        if (!ok) break;
                        try_bar(full(vs), v_lap & 1);  // (complete: each lane observes what the copy wrote)
                        uint8_t* const tile = smem + (2 + vs) * S::TILE;
                        // an infinity or NaN has every exponent bit set: one unit more carries into the sign's place
                        constexpr uint32_t ONE = BF ? 0x00800080u : 0x04000400u, E = BF ? 0x7F80u : 0x7C00u;
#pragma unroll 1
                        for (uint32_t x = tid; x < AP_KEYS * HALVES; x += 64) {  // 128 bytes of a row, eight loads in flight
                            const int32_t key = j * AP_KEYS + (int32_t)(x % AP_KEYS);
                            if (key < w.least) continue;
                            uint8_t* const at = tile + x * 128;  // (half x / 128 of row x % 128)
                            uint4 v[8];
                            if (key >= w.most) {
#pragma unroll
                                for (uint32_t c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(at + ((c + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
                                continue;
                            }
#pragma unroll
                            for (uint32_t c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const uint4*>(at + ((c + lane) & 7) * 16);
                            uint32_t odd = 0;
                            auto look = [&](uint32_t u) { odd |= (u & 0x7FFF7FFFu) + ONE; };
#pragma unroll
                            for (uint32_t c = 0; c < 8; ++c) look(v[c].x), look(v[c].y), look(v[c].z), look(v[c].w);
                            if ((odd & 0x80008000u) != 0) {
                                *odd_values = 1u;
#pragma unroll 1
                                for (uint32_t c = 0; c < 64; ++c) {
                                    uint16_t* const e = reinterpret_cast<uint16_t*>(at) + c;
                                    if ((*e & E) == E) *e = 0;
                                }
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(v_safe);
                        ++guards;
                    }
                    if ((vs += 2) >= SLOTS) vs -= SLOTS, ++v_lap;
                }
            }
        }
    } else {
        // ---- softmax of tile i, thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AP_REGS_SOFTMAX));
        const int i = (int)warp / 4;
        const uint32_t row = threadIdx.x % 128, lanes = ((warp % 4) * 32) << 16;
        const int32_t row_tok = i * tpt + (int32_t)(row / p.group);
        const uint32_t row_head = row % p.group;
        const uint64_t scale2 = pair(p.c, p.c);
        uint32_t items = 0, steps = 0;
        bool ok = true;
        Part w;
#pragma unroll 1
        while (ok && next_part(w)) {
            const int32_t end = i == 0 ? w.end0 : w.end1;
            const bool valid = row < p.tpt * p.group && row_tok < w.tokens;
            const int32_t seen = !valid ? 0 : p.causal ? max(min(w.seen0 + row_tok + 1, w.keys), 0) : w.keys;
            float m = -INFINITY, l = 0.f;  // the reference of the row's exponents, and the sum of its p
#pragma unroll 1
            for (int32_t j = w.j0; j < end; ++j, ++steps) {
                ok = __all_sync(0xFFFFFFFFu, wait_bar(s_full(i), steps & 1, p, AP_PRODUCT, abort_flag));
                if (!ok) break;
                tc_fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32_async(s_col(i) + lanes + c * 32, s + c * 32);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 4; ++c) pin32(s + c * 32);
                if (j >= w.masked) {
                    const int32_t keep = seen - j * AP_KEYS;
#pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = c < keep ? s[c] : -INFINITY;
                }
                float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int c = 4; c < 124; c += 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) tops[x] = fmaxf(fmaxf(tops[x], s[c + x]), s[c + x + 4]);
                const float top = fmaxf(fmaxf(fmaxf(tops[0], s[124]), fmaxf(tops[1], s[125])), fmaxf(fmaxf(tops[2], s[126]), fmaxf(tops[3], s[127])));
                const bool move = (top - m) * p.c > ap_lazy<BF> || (m == -INFINITY && top > m);
                if (__any_sync(0xFFFFFFFFu, move)) {
                    const float next = fmaxf(m, top), keep = next == m ? 1.f : ex2((m - next) * p.c);
                    m = next;
                    l *= keep;
#pragma unroll 1
                    for (int c = 0; c < DP && j > w.j0; c += 16) {
                        float o[16];
                        uint32_t bits[16];
                        tmem_ld16_async(o_col(i) + lanes + c, o);
                        tmem_ld_wait();
                        pin16(o);
#pragma unroll
                        for (int x = 0; x < 16; ++x) bits[x] = __float_as_uint(o[x] * keep);
                        tmem_st16(o_col(i) + lanes + c, bits);
                    }
                }
                const float base = m == -INFINITY ? 0.f : m * p.c - ap_top<BF>;
                const uint64_t base2 = pair(-base, -base);
                uint64_t sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const uint64_t t2 = fma2(pair(s[c * 32 + 2 * x], s[c * 32 + 2 * x + 1]), scale2, base2);
                        const float e0 = ex2(first_of(t2)), e1 = ex2(second_of(t2));
                        sums[x % 2] = add2(sums[x % 2], pair(e0, e1));
                        packed[x] = pack2<BF>(e0, e1);
                    }
                    tmem_st16(s_col(i) + lanes + c * 16, packed);
                    if ((c + 1) * 2 == AP_FIRST || c == 3) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0 && !(p.stall == (uint32_t)j + 1 && i == 0)) mbar_arrive(c == 3 ? p_rest(i) : p_ready(i));
                    }
                }
                sums[0] = add2(sums[0], sums[1]);
                l += first_of(sums[0]) + second_of(sums[0]);
            }
            const bool any = w.j0 < end;  // whether this part has steps of the tile
            if (ok && any) {
                ok = __all_sync(0xFFFFFFFFu, wait_bar(o_full(i), items++ & 1, p, AP_PRODUCT, abort_flag));
                tc_fence_after();
            }
            if (!ok) break;
            // O / l to the output; or O, its reference and l to the workspace; or the sum of the item's parts to the output
            const bool whole = w.whole != 0, odd = any && *odd_values != 0u;
            const uint32_t item_row = i * AP_ROWS + row;
            uint16_t* const out = static_cast<uint16_t*>(p.out) +
                                  ((int64_t)(w.row0 + row_tok) * p.q_heads + w.kv_head * (int)p.group + (int)row_head) * p.d;
            const PartSet set{p.flags, w.c0, w.c1, w.slot, blockIdx.x, warp};
            auto part_at = [&](uint32_t c) { return p.parts + (uint64_t)set.part(c) * part_floats(DP) + item_row; };
            // (one loop for all three, since code that is not cached costs more than its branches)
            enum { WHOLE, LEAVE, JOIN };
            int what = whole ? WHOLE : set.others_done() ? JOIN : LEAVE;
            // A part that is left and then joined after all is taken from the workspace like the others': two warps that
            // finish together then write the same values, once each, the infinities of the guard among them.
            bool left = false;
            const float mine = m * p.c;
            for (;;) {
                float top = mine, sum = l;
                float* const part_o = p.parts + (uint64_t)set.part(set.self) * part_floats(DP);
                auto ref_of = [&](uint32_t c) { return c == set.self ? mine : __ldcg(part_at(c) + AP_ITEM_ROWS * DP); };
                if (what == LEAVE) part_o[AP_ITEM_ROWS * DP + item_row] = mine, part_o[AP_ITEM_ROWS * (DP + 1) + item_row] = l;
                if (what == JOIN) {
#pragma unroll 1
                    for (uint32_t c = set.c0; c <= set.c1; ++c) top = fmaxf(top, ref_of(c));
                    sum = 0.f;
#pragma unroll 1
                    for (uint32_t c = set.c0; c <= set.c1; ++c) {
                        const float mc = ref_of(c), lc = c == set.self ? l : __ldcg(part_at(c) + AP_ITEM_ROWS * (DP + 1));
                        sum += mc == -INFINITY ? lc : ex2(mc - top) * lc;  // (-inf: no key of the part is seen, or its scores are NaN)
                    }
                }
                // a row that sees no key: zeros (its O is 0, too); NaN scores throughout: the sum is NaN
                const float inv = top == -INFINITY && sum == 0.f ? 0.f : __fdividef(1.0f, sum);
                const uint64_t inv2 = pair(inv, inv);
                if (any || what != LEAVE) {  // (a part without steps of the tile has no O: its references are -inf)
#pragma unroll 1
                    for (int c = 0; c < DP; c += 32) {
                        float o[32];
                        if (any) {
                            tmem_ld32_async(o_col(i) + lanes + c, o);
                            tmem_ld_wait();
                            pin32(o);
                        } else {
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = 0.f;
                        }
                        if (what == LEAVE) {
#pragma unroll
                            for (int x = 0; x < 32; x += 4)
                                *reinterpret_cast<float4*>(part_o + ((c + x) / 4 * AP_ITEM_ROWS + item_row) * 4) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                        } else {
                            if (what == JOIN) {
                                float y[32];
#pragma unroll
                                for (int x = 0; x < 32; ++x) y[x] = 0.f;
#pragma unroll 1
                                for (uint32_t b = set.c0; b <= set.c1; ++b) {
                                    const float mc = ref_of(b);
                                    if (mc == -INFINITY) continue;
                                    const float wb = ex2(mc - top);
                                    const float* const src = part_at(b) - item_row + (c / 4 * AP_ITEM_ROWS + item_row) * 4;
#pragma unroll
                                    for (int x = 0; x < 32; x += 4) {
                                        const float4 z = b == set.self && !left ? make_float4(o[x], o[x + 1], o[x + 2], o[x + 3])
                                                                       : __ldcg(reinterpret_cast<const float4*>(src + x * AP_ITEM_ROWS));
                                        y[x] += z.x * wb, y[x + 1] += z.y * wb, y[x + 2] += z.z * wb, y[x + 3] += z.w * wb;
                                    }
                                }
#pragma unroll
                                for (int x = 0; x < 32; ++x) o[x] = y[x];
                            }
                            uint32_t v[16];
#pragma unroll
                            for (int x = 0; x < 16; ++x) {
                                const uint64_t y = mul2(pair(o[2 * x], o[2 * x + 1]), inv2);
                                v[x] = pack2<BF>(first_of(y), second_of(y));
                            }
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                if (valid && c + x * 16 < (int)p.d)
                                    store32(out + c + x * 16, make_uint4(v[8 * x], v[8 * x + 1], v[8 * x + 2], v[8 * x + 3]),
                                            make_uint4(v[8 * x + 4], v[8 * x + 5], v[8 * x + 6], v[8 * x + 7]), p.out32);
                        }
                        __syncwarp();
                    }
                }
                // infinities and NaN that the guard took out, back into the rows that see them
                if (odd && valid && !left) {
#pragma unroll 1
                    for (int32_t key = max(w.least, w.j0 * AP_KEYS); key < min(seen, w.j1 * AP_KEYS); ++key) {
                        const uint16_t* const v = static_cast<const uint16_t*>(p.v.p) + (int64_t)(w.k0 + key) * p.v.token_stride +
                                                  (int64_t)w.kv_head * p.v.head_stride;
#pragma unroll 1
                        for (int x = 0; x < (int)p.d; ++x) {
                            const float f = BF ? __uint_as_float((uint32_t)v[x] << 16) : half_bits_to_float(v[x]);
                            if (fabsf(f) < INFINITY) continue;
                            if (what == LEAVE) {
                                part_o[(x / 4 * AP_ITEM_ROWS + item_row) * 4 + x % 4] += f;
                            } else {
                                const float y = BF ? __uint_as_float((uint32_t)out[x] << 16) : half_bits_to_float(out[x]);
                                out[x] = (uint16_t)pack2<BF>(y + f, 0.f);
                            }
                        }
                    }
                }
                __syncwarp();
                if (what != LEAVE || !set.show()) break;
                what = JOIN, left = true;
            }
            if (any) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_empty(i));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == AP_MMA_WARP) tmem_dealloc<false>(tmem, 512);
    if (*abort_flag != 0u && warp == AP_TMA_WARP && lane == 0) {  // copies that nobody waited for land before the block ends
        for (int i = 0; i < 2; ++i)
            if (q_issued[i] > 0) mbar_wait(q_full(i), (q_issued[i] - 1) & 1, p.status, AP_LOAD, p.wait_ns);
        for (uint32_t x = issued > SLOTS ? issued - SLOTS : 0; x < issued; ++x)
            mbar_wait(full(x % SLOTS), (x / SLOTS) & 1, p.status, AP_LOAD, p.wait_ns);
    }
}

// Before every call's kernel, whose blocks start beside it and wait for its end.
constexpr int CLEAR_THREADS = 608;
__global__ void __launch_bounds__(CLEAR_THREADS) clear_flags(uint32_t* flags, uint32_t sixteens) {
    pdl_launch_dependents();
    for (uint32_t i = threadIdx.x; i < sixteens; i += CLEAR_THREADS) reinterpret_cast<uint4*>(flags)[i] = make_uint4(0, 0, 0, 0);
}

// The tensor map of [tokens][heads][d] rows as dims {d, inner, outer, tokens} (inner x outer = heads), box {64, bi, 1, bt}.
bool encode_rows(CUtensorMap* map, const RowsView& r, uint32_t d, uint32_t inner, uint32_t outer, uint32_t tokens, bool bf,
                 uint32_t bi, uint32_t bt, bool four) {
    // (a dimension of size 1 may carry any stride; a tensor map wants a positive multiple of 16 bytes)
    const cuuint64_t heads = inner * outer > 1 ? (cuuint64_t)r.head_stride * 2 : d * 2;
    const cuuint64_t toks = tokens > 1 ? (cuuint64_t)r.token_stride * 2 : d * 2;
    const CUtensorMapDataType type = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint32_t es[4] = {1, 1, 1, 1};
    CUresult e;
    if (four) {
        const cuuint64_t dims[4] = {d, inner, outer, tokens}, strides[3] = {heads, heads * inner, toks};
        const cuuint32_t box[4] = {64, bi, 1, bt};
        e = encode_fn()(map, type, 4, const_cast<void*>(r.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    } else {
        const cuuint64_t dims[3] = {d, outer, tokens}, strides[2] = {heads, toks};
        const cuuint32_t box[3] = {64, 1, bt};
        e = encode_fn()(map, type, 3, const_cast<void*>(r.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    return e == CUDA_SUCCESS;
}


template <int DP, bool BF>
cudaError_t launch(const PrefillParams& p, uint8_t* workspace, unsigned blocks, cudaStream_t stream) {
    using S = PrefillShape<DP>;
    PrefillArgs a{};
    cudaError_t e = device_status(&a.status, &a.wait_ns, &a.stall);
    if (e != cudaSuccess) return e;
    if (encode_fn() == nullptr) return cudaErrorNotSupported;
    a.v = p.v, a.out = p.out, a.cu_q = p.cu_q, a.cu_k = p.cu_k;
    a.flags = reinterpret_cast<uint32_t*>(workspace);
    a.parts = reinterpret_cast<float*>(workspace + part_flags_bytes(blocks));
    a.seqs = p.seqs, a.q_tokens = p.q_tokens, a.k_tokens = p.k_tokens, a.q_heads = p.q_heads, a.kv_heads = p.kv_heads;
    a.group = p.q_heads / p.kv_heads, a.tpt = AP_ROWS / a.group, a.d = p.d;
    a.inv_blocks = 1.0 / blocks;
    a.c = p.scale * 1.44269504f, a.causal = p.causal, a.out32 = reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
    CUtensorMap qm, km, vm;
    std::memset(&km, 0, sizeof(km));
    std::memset(&vm, 0, sizeof(vm));
    if (!encode_rows(&qm, p.q, p.d, a.group, p.kv_heads, p.q_tokens, BF, a.group, a.tpt, true)) return cudaErrorInvalidValue;
    if (p.k_tokens > 0 && (!encode_rows(&km, p.k, p.d, 1, p.kv_heads, p.k_tokens, BF, 1, AP_KEYS, false) ||
                           !encode_rows(&vm, p.v, p.d, 1, p.kv_heads, p.k_tokens, BF, 1, AP_KEYS, false)))
        return cudaErrorInvalidValue;
    e = cudaFuncSetAttribute(prefill_kernel<DP, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return e;
    // (one split of shared memory for both: changing it would drain an SM)
    e = cudaFuncSetAttribute(clear_flags, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    clear_flags<<<1, CLEAR_THREADS, 0, stream>>>(a.flags, (uint32_t)(part_flags_bytes(blocks) / 16));
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(AP_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prefill_kernel<DP, BF>, qm, km, vm, a);
}

}  // namespace

size_t attention_prefill_workspace(const PrefillParams& p, int num_sms) {
    return part_flags_bytes(num_sms) + (size_t)num_sms * 2 * part_floats(p.d > 64 ? 128 : 64) * sizeof(float);
}

cudaError_t launch_attention_prefill(const PrefillParams& p, void* workspace, int num_sms, cudaStream_t stream) {
    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    const unsigned blocks = (unsigned)num_sms;
    if (p.d > 64) return p.dtype == kBf16 ? launch<128, true>(p, ws, blocks, stream) : launch<128, false>(p, ws, blocks, stream);
    return p.dtype == kBf16 ? launch<64, true>(p, ws, blocks, stream) : launch<64, false>(p, ws, blocks, stream);
}

}  // namespace iq2
