"""How the two attentions deal their work to blocks, modelled on the CPU: the walks of attention_prefill.cu (Work) and
attention_decode.cu (Cursor) restated step by step, over many batches. Every item's key tiles (or tokens) are covered once
and in order, the blocks that share an item agree on who they are and where their parts lie, and no place is used twice."""
import random

import pytest

KEYS = 128


def prefill_parts(seqs, kv_heads, tpt, causal, blocks, item_cost=3 * KEYS, split_cost=3 * KEYS):
    """[(block, item, j0, j1, n, sharers or None)] in the order of the blocks' walks."""
    step = 2 * tpt

    def shown(lq, lk, tok):
        return max(min(lk, tok + 1 + lk - lq), 0) if causal else lk

    def before(lq, lk, t):
        if not causal:
            return t * (item_cost + lk)
        shift = lk - lq
        z = min(-shift // step, t) if shift < 0 else 0
        return t * item_cost + step * ((t * (t + 1) - z * (z + 1)) // 2) + (t - z) * shift

    n_blocks = [-(-lq // step) for lq, _ in seqs]
    length = [before(lq, lk, nb - 1) + item_cost + lk if nb else 0 for (lq, lk), nb in zip(seqs, n_blocks)]
    total, items = sum(length) * kv_heads, sum(n_blocks) * kv_heads
    item_share, share = -(-items // blocks), int(total * (1.0 / blocks)) + 1
    by_items = item_share * (item_cost + max(lk for _, lk in seqs)) <= share + split_cost
    each, everything = (item_share, items) if by_items else (max(share, KEYS), total)
    out = []
    for block in range(blocks):
        u0 = min(block * each, everything)
        left, at = min(u0 + each, everything) - u0, block * each
        if left == 0:
            continue
        acc = 0
        for b, (lq, lk) in enumerate(seqs):
            own = (n_blocks[b] if by_items else length[b]) * kv_heads
            if acc + own > u0:
                break
            acc += own
        rest, pos = u0 - acc, 0
        if by_items:
            tok0, head = rest // kv_heads * step, rest % kv_heads
        else:
            t = max(x for x in range(n_blocks[b]) if before(lq, lk, x) * kv_heads <= rest)
            rest -= before(lq, lk, t) * kv_heads
            tok0 = t * step
            size = item_cost + shown(lq, lk, min(tok0 + step, lq) - 1)
            head, pos = rest // size, rest % size
        while left > 0:
            lq, lk = seqs[b]
            last = min(tok0 + 2 * tpt, lq) - 1
            most = shown(lq, lk, last)
            tiles = [-(-shown(lq, lk, min(tok0 + tpt - 1, last)) // KEYS), -(-most // KEYS) if tok0 + tpt < lq else 0]
            n = max(tiles + [1])
            size = item_cost + most

            def tile_at(x):
                return n if x >= size else -(-max(x - item_cost, 0) // KEYS)

            to = size if by_items else min(size, pos + left)
            j0, j1 = tile_at(pos), tile_at(to)
            if j0 < j1:
                sharers = None
                if (j0, j1) != (0, n):
                    item = at - pos
                    first, final = item + item_cost, item + item_cost + (n - 1) * KEYS
                    c0 = c1 = block
                    while c0 * each > first:
                        c0 -= 1
                    while (c1 + 1) * each <= final:
                        c1 += 1
                    sharers = (c0, c1, 0 if c0 * each >= item else 1)
                out.append((block, (b, tok0, head), j0, j1, n, sharers))
            left -= 1 if by_items else to - pos
            at += to - pos
            pos = 0
            head += 1
            if head == kv_heads:
                head, tok0 = 0, tok0 + step
                if tok0 >= lq:
                    tok0, b = 0, b + 1
                    while b < len(seqs) and seqs[b][0] == 0:
                        b += 1
            if left > 0:
                assert b < len(seqs)
    return out


def decode_parts(lens, items, unit, blocks, cost=3):
    """[(block, item, first token, end, length, sharers or None)]."""
    size = [0 if n == 0 else -(-n // unit) + cost for n in lens]
    total = sum(size) * items
    each = -(-total // blocks)
    out = []
    for block in range(blocks):
        u0, u1 = min(block * each, total), min(block * each + each, total)
        u = u0
        while u < u1:
            acc = 0
            for b in range(len(lens)):
                if acc + size[b] * items > u:
                    break
                acc += size[b] * items
            item, k = divmod(u - acc, size[b])
            n = min(size[b] - k, u1 - u)
            t0, t1 = (max(k, cost) - cost) * unit, min((max(k + n, cost) - cost) * unit, lens[b])
            if t0 < t1:
                sharers = None
                if (t0, t1) != (0, lens[b]):
                    c0 = c1 = block
                    while c0 * each > u - k + cost:
                        c0 -= 1
                    while (c1 + 1) * each <= u - k + size[b] - 1:
                        c1 += 1
                    sharers = (c0, c1, 0 if c0 * each >= u - k else 1)
                out.append((block, (b, item), t0, t1, lens[b], sharers))
            u += n
    return out


def check(parts, wanted):
    covered, shared, places = {}, {}, set()
    for block, item, first, end, n, sharers in parts:
        assert covered.get(item, 0) == first, (item, first)
        covered[item] = end
        assert end <= n
        if sharers is not None:
            c0, c1, slot = sharers
            assert c0 <= block <= c1 and c0 < c1
            assert shared.setdefault(item, (sharers, []))[0] == sharers
            shared[item][1].append(block)
            place = (block, slot if block == c0 else 0)
            assert place not in places
            places.add(place)
    assert covered == wanted
    for (c0, c1, _), blocks in shared.values():
        assert blocks == list(range(c0, c1 + 1))


@pytest.mark.parametrize("seed", range(60))
def test_prefill_work(seed):
    r = random.Random(seed)
    group, kv_heads, blocks = r.choice([1, 2, 4, 7, 8, 16, 100]), r.choice([1, 2, 8]), r.choice([148, 148, 132, 3])
    tpt, causal = 128 // group, r.random() < 0.8
    seqs = []
    for _ in range(r.choice([1, 1, 3, 40])):
        lq = r.choice([0, 1, r.randrange(1, 300), int(2 ** r.uniform(0, 11))])
        seqs.append((lq, r.choice([lq, lq, lq + int(2 ** r.uniform(0, 14)), r.randrange(0, lq + 1)])))
    if not any(lq for lq, _ in seqs):
        seqs.append((5, 5))
    wanted = {}
    for b, (lq, lk) in enumerate(seqs):
        for tok0 in range(0, lq, 2 * tpt):
            last = min(tok0 + 2 * tpt, lq) - 1
            most = max(min(lk, last + 1 + lk - lq), 0) if causal else lk
            for head in range(kv_heads):
                wanted[(b, tok0, head)] = max(-(-most // KEYS), 1)
    check(prefill_parts(seqs, kv_heads, tpt, causal, blocks), wanted)


@pytest.mark.parametrize("seed", range(60))
def test_decode_work(seed):
    r = random.Random(seed)
    lens = [r.choice([0, 1, r.randrange(1, 200), int(2 ** r.uniform(0, 16))]) for _ in range(r.choice([1, 1, 3, 16, 200]))]
    items, unit = r.choice([1, 2, 8, 16]), r.choice([64, 128])
    check(decode_parts(lens, items, unit, r.choice([148, 148, 7])), {(b, i): n for b, n in enumerate(lens) if n for i in range(items)})
