"""How the decode attention over 4-bit caches deals its work to warps, modelled on the CPU: the parts of the line that begin at
multiples of a fraction (Cursor with EVEN in attention_decode.cuh), the pieces that a block's warps leave and add up
(attention_decode_int4.cu), and the blocks' parts that a record joins. Every token of every item is taken once and in order, no
place is used twice, and what is joined is what there is."""
import random

import pytest

UNIT, COST, WARPS = 32, 1, 12


def line_of(lens, items):
    """[(sequence, item, first unit, units)] of the line."""
    out, at = [], 0
    for b, n in enumerate(lens):
        units = 0 if n == 0 else -(-n // UNIT) + COST
        for item in range(items if n else 0):
            out.append((b, item, at, units))
            at += units
    return out, at


def model(lens, items, blocks):
    line, units = line_of(lens, items)
    parts = blocks * WARPS
    share = max(float(units) * (1.0 / blocks) * (1.0 / WARPS), 1.0)

    def begin(part):
        return units if part >= parts else min(int(part * share), units)

    def walk(u0, u1):
        """[(entry of the line, first unit of it in the part, t0, t1)], as Cursor goes."""
        out, unit = [], u0
        while unit < u1:
            entry = next(e for e in line if e[2] <= unit < e[2] + e[3])
            k = unit - entry[2]
            n = min(entry[3] - k, u1 - unit)
            t0, t1 = (max(k, COST) - COST) * UNIT, min((max(k + n, COST) - COST) * UNIT, lens[entry[0]])
            if t0 == t1:
                break
            out.append((entry, unit, t0, t1))
            unit += n
        return out

    outputs, places, records = {}, {}, []
    for block in range(blocks):
        part0 = block * WARPS
        first_unit = begin(part0)
        pieces = []  # in the order of the warps: (entry, t0, t1, whether it is a warp's first piece)
        for warp in range(WARPS):
            for i, (entry, unit, t0, t1) in enumerate(walk(begin(part0 + warp), begin(part0 + warp + 1))):
                if t0 == 0 and t1 == lens[entry[0]]:
                    assert entry[:2] not in outputs
                    outputs[entry[:2]] = [(t0, t1)]
                else:
                    pieces.append((entry, t0, t1, warp, i == 0))
        for warp in range(WARPS):  # a warp keeps two places
            assert sum(p[3] == warp and p[4] for p in pieces) <= 1 and sum(p[3] == warp and not p[4] for p in pieces) <= 1
        while pieces:
            entry = pieces[0][0]
            same = [p for p in pieces if p[0] == entry]
            assert pieces[:len(same)] == same  # those of an item follow one another
            pieces = pieces[len(same):]
            assert all(a[2] == b[1] for a, b in zip(same, same[1:]))
            span = (same[0][1], same[-1][2])
            if span == (0, lens[entry[0]]):
                assert entry[:2] not in outputs
                outputs[entry[:2]] = [span]
            else:
                slot = (block, 0 if entry[2] <= first_unit else 1)
                assert slot not in places
                places[slot] = (entry, span)
        mine = walk(first_unit, begin(part0 + 1)) if begin(part0) < begin(part0 + 1) else []
        if mine and mine[0][2] > 0:
            entry = mine[0][0]
            before = begin(part0 - WARPS)
            if before <= entry[2] + COST:
                last = block
                while begin((last + 1) * WARPS) < entry[2] + entry[3]:
                    last += 1
                records.append((entry, block - 1, last, 0 if before >= entry[2] else 1))
    for entry, c0, c1, slot in records:
        got = [places.pop((c, slot if c == c0 else 0)) for c in range(c0, c1 + 1)]
        assert all(e == entry for e, _ in got) and entry[:2] not in outputs
        outputs[entry[:2]] = [span for _, span in got]
    assert not places
    assert sorted(outputs) == sorted(e[:2] for e in line)
    for (b, _), spans in outputs.items():
        assert spans[0][0] == 0 and spans[-1][1] == lens[b] and all(a[1] == c[0] for a, c in zip(spans, spans[1:]))


@pytest.mark.parametrize("blocks", [1, 2, 7, 148])
def test_every_token_once(blocks):
    rng = random.Random(blocks)
    for _ in range(60):
        n = rng.choice([1, 1, 2, 5, 30])
        most = rng.choice([1, 31, 33, 200, 3000, 40000 if n < 3 else 500])
        lens = [rng.choice([0, 1, 32, most, rng.randint(1, most)]) for _ in range(n)]
        if any(lens):
            model(lens, rng.choice([1, 2, 8]), blocks)


def test_lines_of_about_a_unit_a_warp():
    for units in range(1, 60):
        for blocks in (1, 2, 3, 4):
            model([32 * units], 1, blocks)
            model([32] * units, 2, blocks)
