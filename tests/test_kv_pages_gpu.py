"""The step of the sequences' pages on the GPU against the same step taken one token at a time on the CPU: all of it is whole
numbers, so that state and outputs are compared exactly."""
import random

import pytest
import torch

import candelora_metal_kernels_b200 as c
import kv_step_reference as ref

pytestmark = pytest.mark.gpu
I32 = torch.int32


def i32(x):
    return torch.tensor(x, dtype=I32).cuda()


def empty(pages, page, sequences, width):
    """A KvPages without tokens, and the same as lists."""
    got = c.KvPages.empty(pages, page, sequences, width)
    return got, {"table": [[0] * width for _ in range(sequences)], "lens": [0] * sequences, "free": list(range(pages))[::-1],
                 "count": pages}


def check(pages, state, step, want):
    assert step.slots.tolist() == want[0]
    assert step.positions.tolist() == want[1]
    assert step.cu_seqlens_q.tolist() == want[2]
    assert step.cu_seqlens_k.tolist() == want[3]
    assert step.granted.tolist() == want[4]
    assert pages.seq_lens.tolist() == state["lens"] and pages.free_count.tolist() == [state["count"]]
    assert pages.block_table.tolist() == state["table"] and pages.free_pages.tolist() == state["free"]


def walk(pages, state, page, steps, reuse=False):
    out = None
    for new, total, keep in steps:
        want = ref.pages_step(state, page, new, total, keep)
        if reuse and (out is None or out.slots.shape[0] != total):
            out = c.KvStep.empty(pages, total)
        got = c.kv_pages_step(pages, i32(new), total, keep=None if keep is None else i32(keep), out=out if reuse else None)
        check(pages, state, got, want)


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("sequences,most", [(1, 1), (3, 40), (33, 200), (200, 30)])
def test_steps_of_prompts_tokens_and_cuts(sequences, most, page):
    """Prompts, then steps of a few tokens with sequences that are cut by some, ended, or left alone, padded or not."""
    rng = random.Random(sequences * 100 + page)
    width = -(-3 * most // page) + 1
    pages, state = empty(sequences * width * 2 // 3 + 1, page, sequences, width)
    steps, first = [], [rng.choice([0, 1, page, rng.randint(0, most)]) for _ in range(sequences)]
    steps.append((first, sum(first) + 3, None))
    for _ in range(8):
        new = [rng.choice([0, 1, 1, 2, 5, rng.randint(0, most)]) for _ in range(sequences)]
        keep = [rng.choice([0, 2 ** 31 - 1, rng.randint(0, 2 * most), page]) for _ in range(sequences)]
        steps.append((new, sum(new) + rng.choice([0, 1, 17]), rng.choice([keep, keep, None])))
    walk(pages, state, page, steps, reuse=page == 16)


@pytest.mark.parametrize("page", [16, 5])
def test_large_steps_take_a_cluster_of_blocks(page):
    """More sequences than a block's threads and more tokens than one block takes, again and again over the same pages."""
    rng, n = random.Random(5), 2500
    pages, state = empty(9000 if page == 16 else 20000, page, n, 12 if page == 16 else 30)
    steps = []
    for i in range(4):
        new = [rng.choice([0, 1, 3, 20, 60]) for _ in range(n)]
        steps.append((new, sum(new) + 5, None if i == 0 else [rng.choice([0, 2 ** 31 - 1, 30]) for _ in range(n)]))
    walk(pages, state, page, steps)


@pytest.mark.parametrize("n,width,long", [(8192, 70, 60), (3, 70000, 66000)])
def test_the_most_sequences_and_long_ones(n, width, long):
    pages, state = empty(n + 140000, 1, n, width)
    new = [1] * n
    new[1], new[n - 1] = long, long // 3
    walk(pages, state, 1, [(new, sum(new), None), ([1] * n, n, [0 if b % 3 == 1 else 2 for b in range(n)])])


def test_too_few_pages_rows_or_columns():
    """From the first sequence on that asks for more than is left, those that need a page get nothing; the others do."""
    pages, state = empty(5, 4, 5, 3)
    walk(pages, state, 4, [
        ([3, 0, 4, 2, 1], 10, None),             # four pages of five
        ([1, 4, 4, 2, 1], 12, None),             # 0: the page it has; 1: the last one; 2: none left; 3 and 4: theirs
        ([9, 1, 1, 1, 1], 13, [0, 0, 0, 0, 0]),  # all ended: 0 takes three pages, 1 and 2 the others, 3 and 4 get none
        ([4, 0, 0, 0, 1], 9, None),              # 0 would pass its table's width
        ([1, 1, 1, 1, 1], 3, [0] * 5),           # rows for three only
        ([1, 1, 1, 1, 1], 0, None),
        ([0, 0, 0, 0, 0], 4, [0] * 5),
    ])


def test_counts_below_zero_and_lengths_past_the_table():
    pages, state = empty(12, 4, 3, 4)
    walk(pages, state, 4, [([5, 9, 1], 15, None), ([-3, 2, -2 ** 31], 2, [-1, 4, -2 ** 31])])
    pages.seq_lens.copy_(i32([2 ** 31 - 1, -7, 3])), pages.block_table[0].copy_(i32([8, 9, 10, 11]))
    pages.free_count.fill_(0)
    state["table"][0], state["lens"], state["count"] = [8, 9, 10, 11], [2 ** 31 - 1, -7, 3], 0
    state["table"][1:] = pages.block_table[1:].tolist()
    walk(pages, state, 4, [([0, 1, 1], 2, [3, 0, 3])])


def test_pages_outside_the_pool_have_no_slots():
    """A table with numbers outside the pool: their tokens get slot -1, and a stack past its end is not written."""
    pages, _ = empty(4, 2, 2, 3)
    pages.block_table.copy_(i32([[9, -5, 0], [1, 2, 0]])), pages.seq_lens.copy_(i32([1, 3])), pages.free_count.fill_(1)
    got = c.kv_pages_step(pages, i32([1, 1]), 2)
    assert got.slots.tolist() == [-1, 5] and got.positions.tolist() == [1, 3]
    pages.free_count.fill_(3)
    c.kv_pages_step(pages, i32([0, 0]), 0, keep=i32([0, 0]))  # three pages come back to three free ones of four
    assert pages.free_count.tolist() == [4] and pages.free_pages.tolist()[3] == 9
    pages.free_count.fill_(99)
    got = c.kv_pages_step(pages, i32([2, 0]), 2)
    assert pages.free_count.tolist() == [3] and got.slots.tolist() == [-1, -1]  # (the page taken is 9)


def test_captured_steps_replay_with_other_counts():
    """Two steps of fixed sizes in one graph, replayed as the sequences go on."""
    n, total, page = 40, 200, 16
    pages, state = empty(300, page, n, 30)
    new, keep = torch.zeros((2, n), dtype=I32).cuda(), torch.zeros((2, n), dtype=I32).cuda()
    outs = [c.KvStep.empty(pages, total) for _ in range(2)]
    c.kv_pages_step(pages, new[0], total, keep=keep[0], out=outs[0])  # (all empty)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(2):
            c.kv_pages_step(pages, new[i], total, keep=keep[i], out=outs[i])
    rng = random.Random(2)
    for _ in range(6):
        steps = [([rng.randint(0, 5) for _ in range(n)], [rng.choice([2 ** 31 - 1, 0, 20]) for _ in range(n)]) for _ in range(2)]
        for i, (x, k) in enumerate(steps):
            new[i].copy_(i32(x)), keep[i].copy_(i32(k))
        graph.replay()
        want = ref.pages_step(state, page, steps[0][0], total, steps[0][1])
        assert outs[0].slots.tolist() == want[0] and outs[0].cu_seqlens_k.tolist() == want[3]
        check(pages, state, outs[1], ref.pages_step(state, page, steps[1][0], total, steps[1][1]))


def test_other_streams_aliased_counts_and_strided_ones():
    pages, state = empty(50, 4, 6, 10)
    side = torch.cuda.Stream()
    new = i32([[3, 9], [1, 9], [0, 9], [7, 9], [2, 9], [5, 9]])[:, 0]  # (copied: not contiguous)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = c.kv_pages_step(pages, new, 20)
    side.synchronize()
    check(pages, state, got, ref.pages_step(state, 4, new.tolist(), 20))
    before = list(state["lens"])
    got = c.kv_pages_step(pages, pages.seq_lens, 20, keep=pages.seq_lens)  # every sequence twice as long
    check(pages, state, got, ref.pages_step(state, 4, before, 20, before))


def test_refusals():
    pages = c.KvPages.empty(8, 4, 3, 2)
    new = i32([1, 1, 1])

    def refused(match, fn, *args, **kw):
        with pytest.raises(c.Iq2Error, match=match):
            fn(*args, **kw)

    t, lens, free, count = pages.block_table, pages.seq_lens, pages.free_pages, pages.free_count
    refused("int32 tensor of rank 1", c.kv_pages_step, pages, new.long(), 3)
    refused("new_lens 2", c.kv_pages_step, pages, new[:2], 3)
    refused("keep 2", c.kv_pages_step, pages, new, 3, keep=new[:2])
    refused("device mismatch", c.kv_pages_step, pages, new.cpu(), 3)
    refused("negative or too large", c.kv_pages_step, pages, new, -1)
    refused("negative or too large", c.kv_pages_step, pages, new, 2 ** 31 - 1)
    refused("out has 4 rows", c.kv_pages_step, pages, new, 3, out=c.KvStep.empty(pages, 4))
    refused("non-zero dimensions", c.kv_pages_step, c.KvPages(t[:0], lens[:0], free, count, 4), new[:0], 3)
    refused("non-zero dimensions", c.KvPages, t, lens, free, count, 0)
    refused("too large", c.kv_pages_step, c.KvPages(t, lens, free, count, 2 ** 29), new, 3)
    refused("more than 8192", c.kv_pages_step, c.KvPages.empty(1, 1, 8193, 1), torch.zeros(8193, dtype=I32).cuda(), 3)
    refused("rank 2", c.KvPages, lens, lens, free, count, 4)
    refused("free_count 2", c.KvPages, t, lens, free, free[:2], 4)
    refused("seq_lens 2", c.KvPages, t, lens[:2], free, count, 4)
    refused("contiguous", c.KvPages, t.t(), lens[:2], free, count, 4)
    refused("device mismatch", c.KvPages, t, lens.cpu(), free, count, 4)
    with pytest.raises(AttributeError):
        pages.seq_lens = lens
    pages.seq_lens.data = lens.clone()
    refused("have moved", c.kv_pages_step, pages, new, 3)
