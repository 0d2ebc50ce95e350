// The dealing of the decode attentions' work (Cursor in attention_decode.cuh) run on the host. Reads calls, one a line:
//     kind (1: 4-bit caches, 0: others of 128 tokens a unit)  blocks  items  sequences  length ...
// and prints for each, a line an entry: "part WARP B ITEM T0 T1 WHOLE FIRST" for what a warp (a block, for kind 0) takes, "join B ITEM C0
// C1 SLOT" for what a block joins, after "block N", and "end".
#include "attention_decode.cuh"

#include <cstdio>
#include <vector>

namespace {

template <uint32_t UNIT, uint32_t COST, bool EVEN>
void deal(uint32_t blocks, uint32_t per_block, uint32_t items, std::vector<int32_t>& lens) {
    using Cursor = iq2::Cursor<UNIT, COST, EVEN>;
    iq2::DecodeParams p{};
    p.seq_lens = lens.data(), p.batch = (uint32_t)lens.size(), p.table_width = 1u << 26, p.c.page_size = 64;
    uint64_t units = 0;
    for (uint32_t b = 0; b < p.batch; ++b) units += Cursor::units_of(iq2::seq_len(p, b));
    units *= items;
    const double inv = 1.0 / blocks * (1.0 / per_block);
    const typename Cursor::Parts line = Cursor::Parts::of(units, blocks * per_block, inv);
    for (uint32_t block = 0; block < blocks; ++block) {
        std::printf("block %u\n", block);
        for (uint32_t warp = 0; warp < per_block; ++warp) {
            const uint32_t part = block * per_block + warp;
            const uint64_t u0 = line.begin(part), u1 = line.begin(part + 1);
            Cursor cur{};
            uint64_t before = 0;
            for (uint32_t b = 0; u0 < u1 && b < p.batch; ++b) {
                const uint32_t own = Cursor::units_of(iq2::seq_len(p, b));
                if (before + (uint64_t)own * items > u0) {
                    cur = Cursor::at(u0, u1, b, iq2::seq_len(p, b), own, before);
                    break;
                }
                before += (uint64_t)own * items;
            }
            if (warp == 0) {
                const iq2::JoinRecord r = cur.record(line, block, part, per_block);
                if (r.c1 != 0) std::printf("join %u %u %u %u %u\n", r.b, r.item, r.c0, r.c1, r.slot);
            }
            if (EVEN && cur.t0 == cur.t1) cur.unit = cur.end;
            for (; !cur.done(); cur.next(p, items))
                if (cur.t0 != cur.t1) std::printf("part %u %u %u %u %u %u %u\n", warp, cur.b, cur.item, cur.t0, cur.t1, (unsigned)cur.whole(),
                                                  (unsigned)cur.first_of(line.begin(block * per_block)));
        }
    }
    std::printf("end\n");
}

}  // namespace

int main() {
    std::printf("%u %u %d %u\n", iq2::AD_I4_UNIT, iq2::AD_I4_ITEM_COST, iq2::AD_I4_WARPS, iq2::AD_ITEM_COST);
    uint32_t kind, blocks, items, n;
    while (std::scanf("%u %u %u %u", &kind, &blocks, &items, &n) == 4) {
        std::vector<int32_t> lens(n);
        for (int32_t& x : lens)
            if (std::scanf("%d", &x) != 1) return 1;
        if (kind == 1) deal<iq2::AD_I4_UNIT, iq2::AD_I4_ITEM_COST, true>(blocks, iq2::AD_I4_WARPS, items, lens);
        else deal<128, iq2::AD_ITEM_COST, false>(blocks, 1, items, lens);
    }
}
