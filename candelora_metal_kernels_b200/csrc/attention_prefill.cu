// Attention of packed prompts on the sm_100a tensor cores: for query i of a sequence with Lq queries and Lk keys
//     o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  j < Lk, and j <= i + Lk - Lq if causal.
//
// A block takes two tiles of 128 rows. The rows of a tile are (token, head) pairs, the G query heads of one key head
// packed beside each other (TPT = 128 / G tokens a tile), so that each K and V tile that is loaded serves all of them and
// short prompts still fill the rows. Over tiles of 128 keys, with the running maximum and sum of a softmax:
//   S_i = Q_i K^T   tcgen05.mma, M = N = 128, into TMEM (f32)                          one MMA thread for both tiles
//   P_i = 2^(c S - m), rounded to the inputs' 16-bit type (one unit of 2^-8 or 2^-11, as the output's own rounding),
//         written over S_i in TMEM; the sum is of the f32 values                        a warpgroup a tile, a thread a row
//   O_i += P_i V    tcgen05.mma with A = P_i from TMEM, V as the N-major operand
// The two tiles alternate on the tensor core: while one warpgroup computes its exponentials the other's products run.
// K and V tiles arrive by TMA (128-byte swizzle, no multicast) in one ring, K_0 V_0 K_1 V_1 ...
//   * Lazy rescaling: the reference m of a row moves only when a score exceeds it by more than 2^8 (p stays below 256,
//     far inside both types' range), so O in TMEM is rescaled a few times a row instead of once a tile.
//   * Masked keys are replaced by -inf before the maximum (never added to), so that whatever K holds there cannot matter.
//     V needs more, since 0 * NaN is NaN: two guard warps look through the V tiles that hold keys some row does not see.
//     Rows past the last visible key (other sequences' tokens) become zeros; infinities and NaN of keys that only some
//     rows see become zeros too, and the epilogue adds them back to exactly the rows that see them.
// Every wait is bounded by wall time (device_status); a block that gives up still drains its copies and frees its TMEM.
#include "attention_internal.h"
#include "iq2xxs_internal.h"
#include "tcgen05.cuh"

#include <cstring>

namespace iq2 {

namespace {

constexpr int AP_ROWS = 128, AP_KEYS = 128;
constexpr int AP_MMA_WARP = 8, AP_TMA_WARP = 9, AP_GUARD_WARP = 10;  // warps 0-7: the two softmax warpgroups
constexpr int AP_THREADS = 12 * 32;
constexpr uint32_t AP_LOAD = 0x100u, AP_RELEASE = 0x200u, AP_PROB = 0x400u, AP_PRODUCT = 0x800u;  // status bits
constexpr float AP_LAZY = 8.0f;  // how far (in powers of two) a score may exceed its row's reference

template <int DP>
struct PrefillShape {
    static constexpr int TILE = 128 * DP * 2;           // bytes of 128 rows of q, k or v
    static constexpr int SLOTS = DP == 128 ? 5 : 8;     // K and V tiles in flight
    static constexpr int BARS = 2 + 2 * SLOTS + 9;
    static constexpr int SMEM = 1024 + 2 * TILE + SLOTS * TILE + BARS * 8 + 16;
};

struct PrefillArgs {
    RowsView v;
    void* out;
    const int32_t *cu_q, *cu_k;
    unsigned int* status;
    uint64_t wait_ns;
    uint32_t stall;
    uint32_t seqs, q_tokens, k_tokens, q_heads, kv_heads, group, tpt, d;
    float c;  // scale log2(e)
    bool causal;
};

// Instruction descriptor, kind::f16: f32 accumulator, f16 or bf16 operands, M = 128; n: columns; B N-major for P V.
__device__ __forceinline__ uint32_t idesc16(bool bf, uint32_t n, bool b_nmajor) {
    return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((b_nmajor ? 1u : 0u) << 16) | ((n >> 3) << 17) | (8u << 24);
}

// V as the N-major operand: 64-column blocks of 128 keys x 128 bytes (16 KB apart), groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t nmajor_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(16384u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

__device__ __forceinline__ void mma_a_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"f"(v[0]),
        "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
        "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]),
        "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]),
        "f"(v[29]), "f"(v[30]), "f"(v[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// A bounded wait of the block: false when it ran out, or when another role of the block gave up.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const PrefillArgs& p, uint32_t code, volatile uint32_t* abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
        for (int i = 0; i < 32; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag != 0u) return false;
        if (global_ns() - t0 > p.wait_ns) {
            atomicOr(p.status, code);
            *abort_flag = 1u;
            return false;
        }
    }
}

// The sequence whose blocks (of `step` tokens) hold block `index` counted from the last one: lanes take 32 sequences at a
// time. Returns false past the blocks' end. Lengths are clamped to the tensors, so that no index leads outside them.
struct BlockWork {
    int32_t q0, lq, k0, lk, tok0;
};
__device__ __forceinline__ bool find_work(const PrefillArgs& p, uint32_t index, uint32_t step, BlockWork* w) {
    const uint32_t lane = threadIdx.x % 32;
    const int32_t tq = (int32_t)p.q_tokens, tk = (int32_t)p.k_tokens;
    auto len = [&](uint32_t b) {
        if (b >= p.seqs) return 0;
        const int32_t a = min(max(__ldg(p.cu_q + b), 0), tq);
        return max(min(__ldg(p.cu_q + b + 1), tq) - a, 0);
    };
    uint32_t total = 0;
    for (uint32_t b0 = 0; b0 < p.seqs; b0 += 32) total += __reduce_add_sync(0xFFFFFFFFu, ((uint32_t)len(b0 + lane) + step - 1) / step);
    if (index >= total) return false;
    const uint32_t want = total - 1 - index;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < p.seqs; b0 += 32) {
        const uint32_t own = ((uint32_t)len(b0 + lane) + step - 1) / step;
        uint32_t upto = own;
        for (int o = 1; o < 32; o *= 2) {
            const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= (uint32_t)o) upto += x;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, before + upto > want);
        if (hit != 0) {
            const int first = __ffs(hit) - 1;
            const uint32_t b = b0 + first, start = before + __shfl_sync(0xFFFFFFFFu, upto - own, first);
            w->q0 = min(max(__ldg(p.cu_q + b), 0), tq);
            w->lq = len(b);
            w->k0 = min(max(__ldg(p.cu_k + b), 0), tk);
            w->lk = max(min(__ldg(p.cu_k + b + 1), tk) - w->k0, 0);
            w->tok0 = (int32_t)((want - start) * step);
            return true;
        }
        before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    return false;
}

template <int DP, bool BF>
__global__ void __launch_bounds__(AP_THREADS, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PrefillArgs p) {
    using S = PrefillShape<DP>;
    constexpr int SLOTS = S::SLOTS, HALVES = DP / 64;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + 2 * S::TILE, bars = ring + SLOTS * S::TILE;
    volatile uint32_t* const words = reinterpret_cast<volatile uint32_t*>(smem + (2 + SLOTS) * S::TILE + S::BARS * 8);
    volatile uint32_t* const abort_flag = words + 1;
    volatile uint32_t* const odd_values = words + 2;  // the guard found infinities or NaN
    auto q_full = [&](int i) { return bars + i * 8; };
    auto full = [&](uint32_t s) { return bars + 16 + s * 8; };
    auto empty = [&](uint32_t s) { return bars + 16 + (SLOTS + s) * 8; };
    auto s_full = [&](int i) { return bars + 16 + (2 * SLOTS + i) * 8; };
    auto p_ready = [&](int i) { return bars + 16 + (2 * SLOTS + 2 + i) * 8; };
    auto o_full = [&](int i) { return bars + 16 + (2 * SLOTS + 4 + i) * 8; };
    const uint32_t v_safe = bars + 16 + (2 * SLOTS + 6) * 8, drained = v_safe + 8, v_landed = v_safe + 16;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    const uint32_t kv_head = blockIdx.x % p.kv_heads;
    BlockWork w;
    if (!find_work(p, blockIdx.x / p.kv_heads, 2 * p.tpt, &w)) return;
    const int32_t shift = w.lk - w.lq;
    // keys that the query at `tok` of the sequence sees
    auto shown = [&](int32_t tok) { return p.causal ? max(min(w.lk, tok + 1 + shift), 0) : w.lk; };
    const int32_t tpt = (int32_t)p.tpt;
    const int32_t last = min(w.tok0 + 2 * tpt, w.lq) - 1;       // the block's last token
    const int32_t least = shown(w.tok0), most = shown(last);    // visible keys of its first and last rows
    int32_t n_tiles[2];
    n_tiles[0] = (shown(min(w.tok0 + tpt - 1, last)) + AP_KEYS - 1) / AP_KEYS;
    n_tiles[1] = w.tok0 + tpt < w.lq ? (most + AP_KEYS - 1) / AP_KEYS : 0;
    const int32_t n = max(n_tiles[0], n_tiles[1]), masked0 = least / AP_KEYS;  // from masked0 on some row sees less than a tile

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(q_full(i), 1);
        for (int s = 0; s < SLOTS; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
        for (int i = 0; i < 2; ++i) mbar_init(s_full(i), 1), mbar_init(p_ready(i), 4), mbar_init(o_full(i), 1);
        mbar_init(v_safe, 2);
        mbar_init(drained, 1);
        mbar_init(v_landed, 1);
        fence_barrier_init();
        *abort_flag = 0u;
        *odd_values = 0u;
    }
    if (warp == AP_MMA_WARP) tmem_alloc<false>(smem_u32(const_cast<uint32_t*>(words)), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = words[0];
    auto s_col = [&](int i) { return tmem + i * 128; };
    auto o_col = [&](int i) { return tmem + 256 + i * 128; };

    uint32_t issued = 0;  // K and V tiles (TMA thread)
    if (warp == AP_TMA_WARP) {
        if (lane == 0 && n > 0) {
            const int hk = (int)kv_head;
            bool ok = true;
            auto load_kv = [&](const CUtensorMap* map, int32_t j) {
                const uint32_t s = issued % SLOTS;
                if (issued >= SLOTS) ok = wait_bar(empty(s), (issued / SLOTS - 1) & 1, p, AP_RELEASE, abort_flag);
                if (!ok) return;
                mbar_expect_tx(full(s), S::TILE);
                for (int h = 0; h < HALVES; ++h)
                    tma_load_3d(ring + s * S::TILE + h * 16384, map, full(s), h * 64, hk, w.k0 + j * AP_KEYS);
                ++issued;
            };
            auto load_q = [&](int i) {
                if (n_tiles[i] == 0) return;
                mbar_expect_tx(q_full(i), HALVES * p.tpt * p.group * 128);
                for (int h = 0; h < HALVES; ++h)
                    tma_load_4d(q_smem + i * S::TILE + h * 16384, &qmap, q_full(i), h * 64, 0, hk, w.q0 + w.tok0 + i * tpt);
            };
            load_q(0);
            load_kv(&kmap, 0);
            load_q(1);
            for (int32_t j = 0; j < n && ok; ++j) {
                if (j > 0) load_kv(&kmap, j);
                if (ok) load_kv(&vmap, j);
            }
        }
    } else if (warp == AP_MMA_WARP) {
        if (lane == 0 && n > 0) {
            const uint32_t id_s = idesc16(BF, AP_KEYS, false), id_o = idesc16(BF, p.d, true);
            const int ksteps = (int)p.d / 16;
            auto products_s = [&](int i, uint32_t slot) {
                for (int k = 0; k < ksteps; ++k) {
                    const uint32_t at = (k / 4) * 16384 + (k % 4) * 32;
                    tc_mma(s_col(i), sw128_desc(q_smem + i * S::TILE + at), sw128_desc(ring + slot * S::TILE + at), id_s, k > 0);
                }
                tc_commit(s_full(i));
            };
            bool ok = wait_bar(full(0), 0, p, AP_LOAD, abort_flag);
            for (int i = 0; i < 2 && ok; ++i) {
                if (n_tiles[i] == 0) continue;
                ok = wait_bar(q_full(i), 0, p, AP_LOAD, abort_flag);
                if (ok) products_s(i, 0);
            }
            if (ok) tc_commit(empty(0));
            for (int32_t j = 0; j < n && ok; ++j) {
                const uint32_t vi = 2 * j + 1, vs = vi % SLOTS, ki = 2 * j + 2, ks = ki % SLOTS;
                ok = wait_bar(full(vs), (vi / SLOTS) & 1, p, AP_LOAD, abort_flag);
                if (ok && j >= masked0) mbar_arrive(v_landed);
                if (ok && j >= masked0) ok = wait_bar(v_safe, (j - masked0) & 1, p, AP_LOAD, abort_flag);
                if (ok && j + 1 < n) ok = wait_bar(full(ks), (ki / SLOTS) & 1, p, AP_LOAD, abort_flag);
                for (int i = 0; i < 2 && ok; ++i) {
                    if (j >= n_tiles[i]) continue;
                    if (!(ok = wait_bar(p_ready(i), j & 1, p, AP_PROB, abort_flag))) break;
                    tc_fence_after();
                    for (int k = 0; k < AP_KEYS / 16; ++k)
                        mma_a_tmem(o_col(i), s_col(i) + k * 8, nmajor_desc(ring + vs * S::TILE + k * 2048), id_o, (j > 0 || k > 0) ? 1u : 0u);
                    if (j + 1 < n_tiles[i]) products_s(i, ks);
                    else tc_commit(o_full(i));
                }
                if (!ok) break;
                tc_commit(empty(vs));
                if (j + 1 < n) tc_commit(empty(ks));
            }
            if (!ok) {  // what was issued ends before the TMEM is freed
                tc_commit(drained);
                mbar_wait(drained, 0, p.status, AP_PRODUCT, p.wait_ns);
            }
        }
    } else if (warp >= AP_GUARD_WARP) {
        const uint32_t tid = threadIdx.x - AP_GUARD_WARP * 32;
        for (int32_t j = masked0; j < n; ++j) {
            const uint32_t vi = 2 * j + 1, vs = vi % SLOTS;
            bool ok = true;
            // (the MMA thread passes each tile on: waiting on its load from here could meet the ring a lap away)
            if (lane == 0) ok = wait_bar(v_landed, (j - masked0) & 1, p, AP_LOAD, abort_flag);
            if (!__shfl_sync(0xFFFFFFFFu, (int)ok, 0)) break;
            // (every lane observes the barrier itself before it reads what the copy wrote)
            mbar_try_wait(full(vs), (vi / SLOTS) & 1);
            uint8_t* const tile = smem + (2 + vs) * S::TILE;
            for (uint32_t r = tid; r < AP_KEYS; r += 64) {
                const int32_t key = j * AP_KEYS + (int32_t)r;
                if (key < least) continue;
                for (int h = 0; h < HALVES; ++h)
                    for (uint32_t c = 0; c < 8; ++c) {
                        uint4* const at = reinterpret_cast<uint4*>(tile + h * 16384 + r * 128 + ((c + lane) & 7) * 16);
                        if (key >= most) {
                            *at = make_uint4(0, 0, 0, 0);
                            continue;
                        }
                        constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;  // exponent bits of an infinity or NaN
                        uint4 x = *at;
                        bool odd = false;
                        auto clean = [&](uint32_t& v) {
                            if ((v & E) == E) v &= 0xFFFF0000u, odd = true;
                            if (((v >> 16) & E) == E) v &= 0xFFFFu, odd = true;
                        };
                        clean(x.x), clean(x.y), clean(x.z), clean(x.w);
                        if (odd) *at = x, *odd_values = 1u;
                    }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_safe);
        }
    } else {
        // ---- softmax of tile i, thread = row ----
        const int i = (int)warp / 4;
        const uint32_t row = threadIdx.x % 128, lanes = ((warp % 4) * 32) << 16;
        const int32_t tok = w.tok0 + i * tpt + (int32_t)(row / p.group);
        const bool valid = row < p.tpt * p.group && tok < w.lq;
        const int32_t seen = valid ? shown(tok) : 0;
        float m = -INFINITY, l = 0.f;  // the reference of the row's exponents, and the sum of its p
        bool ok = true;
        for (int32_t j = 0; j < n_tiles[i] && ok; ++j) {
            ok = wait_bar(s_full(i), j & 1, p, AP_PRODUCT, abort_flag);
            if (!(ok = __all_sync(0xFFFFFFFFu, ok))) break;
            tc_fence_after();
            float s[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_async(s_col(i) + lanes + c * 32, s + c * 32);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 4; ++c) pin32(s + c * 32);
            if (j >= masked0) {
                const int32_t keep = seen - j * AP_KEYS;
#pragma unroll
                for (int c = 0; c < 128; ++c) s[c] = c < keep ? s[c] : -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int c = 1; c < 128; ++c) top = fmaxf(top, s[c]);
            const bool move = (top - m) * p.c > AP_LAZY || (m == -INFINITY && top > m);
            if (__any_sync(0xFFFFFFFFu, move)) {
                const float next = fmaxf(m, top), keep = next == m ? 1.f : ex2((m - next) * p.c);
                m = next;
                l *= keep;
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < DP; c += 32) {
                        float o[32];
                        tmem_ld32_async(o_col(i) + lanes + c, o);
                        tmem_ld_wait();
                        pin32(o);
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] *= keep;
                        tmem_st32(o_col(i) + lanes + c, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m * p.c;
            float sum[4] = {};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t packed[16];
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                    const float a = ex2(fmaf(s[c * 32 + x], p.c, -base)), b = ex2(fmaf(s[c * 32 + x + 1], p.c, -base));
                    sum[x & 2] += a;
                    sum[(x & 2) + 1] += b;
                    packed[x / 2] = pack2<BF>(a, b);
                }
                tmem_st16(s_col(i) + lanes + c * 16, packed);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && !(p.stall == (uint32_t)j + 1 && i == 0)) mbar_arrive(p_ready(i));
        }
        if (ok && n_tiles[i] > 0) {
            ok = wait_bar(o_full(i), 0, p, AP_PRODUCT, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after();
        }
        if (ok) {
            // O / l, through the tile's Q rows in shared memory (no longer needed) to whole rows of the output
            uint8_t* const mine = smem + i * S::TILE + (warp % 4) * 32 * DP * 2;
            const float inv = seen > 0 ? 1.0f / l : 0.f;
            const bool odd = n_tiles[i] > 0 && *odd_values != 0u;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                float o[32];
                if (n_tiles[i] > 0) {
                    tmem_ld32_async(o_col(i) + lanes + c, o);
                    tmem_ld_wait();
                    pin32(o);
                }
                if (odd)
                    for (int32_t key = least; key < seen; ++key)
                        for (int x = 0; x < 32 && c + x < (int)p.d; ++x) {
                            const int64_t at = (int64_t)(w.k0 + key) * p.v.token_stride + (int64_t)kv_head * p.v.head_stride + c + x;
                            const uint16_t b = static_cast<const uint16_t*>(p.v.p)[at];
                            const float f = BF ? __uint_as_float((uint32_t)b << 16) : half_bits_to_float(b);
                            if (!(fabsf(f) < INFINITY))
#pragma unroll
                                for (int y = 0; y < 32; ++y)
                                    if (y == x) o[y] += f;
                        }
#pragma unroll
                for (int x = 0; x < 32; x += 8) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (seen > 0)
                        v = make_uint4(pack2<BF>(o[x] * inv, o[x + 1] * inv), pack2<BF>(o[x + 2] * inv, o[x + 3] * inv),
                                       pack2<BF>(o[x + 4] * inv, o[x + 5] * inv), pack2<BF>(o[x + 6] * inv, o[x + 7] * inv));
                    *reinterpret_cast<uint4*>(mine + lane * DP * 2 + ((((c + x) / 8) ^ (lane & 7)) * 16)) = v;
                }
            }
            __syncwarp();
            constexpr int CH = DP / 8;  // 16-byte chunks of a row; a warp writes 32 / CH rows at a time
            for (int r0 = 0; r0 < 32; r0 += 32 / CH) {
                const uint32_t r = r0 + lane / CH, c = lane % CH, tile_row = (warp % 4) * 32 + r;
                const int32_t t = w.tok0 + i * tpt + (int32_t)(tile_row / p.group);
                if (tile_row < p.tpt * p.group && t < w.lq && c * 8 < p.d) {
                    const int64_t at = ((int64_t)(w.q0 + t) * p.q_heads + kv_head * p.group + tile_row % p.group) * p.d + c * 8;
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) =
                        *reinterpret_cast<const uint4*>(mine + r * DP * 2 + ((c ^ (r & 7)) * 16));
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == AP_MMA_WARP) tmem_dealloc<false>(tmem, 512);
    if (*abort_flag != 0u && issued > 0) {  // copies that nobody waited for land before the block ends
        for (int i = 0; i < 2; ++i)
            if (n_tiles[i] > 0) mbar_wait(q_full(i), 0, p.status, AP_LOAD, p.wait_ns);
        for (uint32_t x = issued > SLOTS ? issued - SLOTS : 0; x < issued; ++x)
            mbar_wait(full(x % SLOTS), (x / SLOTS) & 1, p.status, AP_LOAD, p.wait_ns);
    }
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
cudaError_t launch(const PrefillParams& p, cudaStream_t stream) {
    using S = PrefillShape<DP>;
    PrefillArgs a{};
    cudaError_t e = device_status(&a.status, &a.wait_ns, &a.stall);
    if (e != cudaSuccess) return e;
    if (encode_fn() == nullptr) return cudaErrorNotSupported;
    a.v = p.v, a.out = p.out, a.cu_q = p.cu_q, a.cu_k = p.cu_k;
    a.seqs = p.seqs, a.q_tokens = p.q_tokens, a.k_tokens = p.k_tokens, a.q_heads = p.q_heads, a.kv_heads = p.kv_heads;
    a.group = p.q_heads / p.kv_heads, a.tpt = AP_ROWS / a.group, a.d = p.d;
    a.c = p.scale * 1.44269504f, a.causal = p.causal;
    CUtensorMap qm, km, vm;
    std::memset(&km, 0, sizeof(km));
    std::memset(&vm, 0, sizeof(vm));
    if (!encode_rows(&qm, p.q, p.d, a.group, p.kv_heads, p.q_tokens, BF, a.group, a.tpt, true)) return cudaErrorInvalidValue;
    if (p.k_tokens > 0 && (!encode_rows(&km, p.k, p.d, 1, p.kv_heads, p.k_tokens, BF, 1, AP_KEYS, false) ||
                           !encode_rows(&vm, p.v, p.d, 1, p.kv_heads, p.k_tokens, BF, 1, AP_KEYS, false)))
        return cudaErrorInvalidValue;
    e = cudaFuncSetAttribute(prefill_kernel<DP, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return e;
    // every sequence's last block may be part full
    const uint64_t step = 2 * a.tpt, blocks = ((uint64_t)p.q_tokens + step - 1) / step + p.seqs;
    prefill_kernel<DP, BF><<<(unsigned)(blocks * p.kv_heads), AP_THREADS, S::SMEM, stream>>>(qm, km, vm, a);
    return cudaGetLastError();
}

}  // namespace

size_t attention_prefill_workspace(const PrefillParams&, int) { return 0; }

cudaError_t launch_attention_prefill(const PrefillParams& p, void*, int, cudaStream_t stream) {
    if (p.d > 64) return p.dtype == kBf16 ? launch<128, true>(p, stream) : launch<128, false>(p, stream);
    return p.dtype == kBf16 ? launch<64, true>(p, stream) : launch<64, false>(p, stream);
}

}  // namespace iq2
