"""A serving step's operators together: pages, norms with rotation and cache write, and the attentions over what they left."""
import sys
from pathlib import Path

import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
import kv_step_reference as step_ref
from test_kv_cache_gpu import randn, tables

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8, I4 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.uint8
HQ, HKV, D, PAGE, SEQS, WIDTH = 8, 2, 64, 16, 6, 12


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Layer:
    """A cache and its sequences' pages, with the tokens that each sequence should hold, in 64 bits."""

    def __init__(self, cache_dtype, pages=SEQS * WIDTH):
        self.cache, self.pages = c.KvCache.empty(pages, HKV, PAGE, D, cache_dtype), c.KvPages.empty(pages, PAGE, SEQS, WIDTH)
        self.cos, self.sin = tables(PAGE * WIDTH, D)
        self.wq, self.wk = (1 + 0.3 * randn((D,), i) for i in (1, 2))
        self.dev = [x.cuda() for x in (self.cos, self.sin, self.wq, self.wk)]
        self.held = [[] for _ in range(SEQS)]

    def write(self, q, k, v, step):
        cos, sin, wq, wk = self.dev
        return c.kv_cache_write(self.cache, k, v, step.slots, q=q, positions=step.positions, cos=cos, sin=sin, q_norm=wq, k_norm=wk)

    def step(self, q, k, v, new, keep=None, total=None, out=None):
        step = c.kv_pages_step(self.pages, i32(new), total or sum(new), keep=None if keep is None else i32(keep), out=out)
        return step, self.write(q, k, v, step)

    def remember(self, k, v, new, keep=None):
        """What the step should have left, as the cache holds it."""
        k64, row = step_ref.normed(k, self.wk, 1e-6), 0
        for b in range(SEQS):
            del self.held[b][len(self.held[b]) if keep is None else keep[b]:]
            for i in range(new[b]):
                pos = torch.tensor([len(self.held[b])])
                self.held[b].append((ref.rotated(k64[row:row + 1], pos, self.cos, self.sin, False)[0], v[row].float()))
                row += 1

    def stored(self, b):
        """K and V [tokens, heads, d] in 64 bits that sequence b should have: rounded or quantised as the cache does."""
        rows = [torch.stack(x) if x else torch.zeros((0, HKV, D)) for x in (zip(*self.held[b]) if self.held[b] else ((), ()))]
        if self.cache.dtype == I4:
            return [step_ref.values4(*step_ref.quantised4(x)) for x in rows]
        if self.cache.dtype == I8:
            return [codes.double() * scale.double()[..., None] for codes, scale in (ref.quantised(x) for x in rows)]
        return [x.to(self.cache.dtype).double() for x in rows]

    def check_decode(self, q, got, tolerance):
        for b in range(SEQS):
            k, v = self.stored(b)
            n = k.shape[0]
            for h in range(HQ):
                o, size = ref.attend(q[b, h:h + 1].double().cpu(), k[:, h // (HQ // HKV)], v[:, h // (HQ // HKV)], [n], D ** -0.5)
                assert ((got[b, h].double().cpu() - o[0]).abs() <= tolerance * size[0] + ref.UNIT[got.dtype] * o[0].abs()).all(), (b, h)


@pytest.mark.parametrize("cache_dtype", [I4, I8, BF16])
def test_prompts_drafts_and_ends(cache_dtype):
    """Prompts; steps of several tokens of which some are taken back; sequences that end and begin anew: the attention of the last
    step's tokens over the cache is that of the tokens which should be there.

    Tolerance: of decode attention for f32 q (bf16 caches 2^-12, others 2^-15 of sum p |v|; normed q and k have scores of 13 at
    most as in test_kv_int4_gpu.py)."""
    layer = Layer(cache_dtype)
    plan = [([40, 3, 0, 100, 17, 64], None), ([1] * 6, None), ([4, 4, 4, 0, 4, 4], None), ([3, 5, 1, 2, 1, 1], [41, 6, 0, 60, 18, 66]),
            ([1, 30, 1, 1, 1, 1], [2 ** 31 - 1, 0, 4, 2 ** 31 - 1, 0, 2 ** 31 - 1]), ([1] * 6, None)]
    for turn, (new, keep) in enumerate(plan):
        rows = sum(new)
        q, k, v = (randn((rows, h, D), 10 * turn + i) for i, h in enumerate((HQ, HKV, HKV)))
        step, got_q = layer.step(q.cuda(), k.cuda(), v.cuda(), new, keep)
        layer.remember(k, v, new, keep)
        assert layer.pages.seq_lens.tolist() == [len(x) for x in layer.held] and step.granted.tolist() == new
        if min(new) > 0:
            last = got_q[step.cu_seqlens_q[1:].long() - 1]
            got = c.attention_decode(last, layer.cache, layer.pages.block_table, layer.pages.seq_lens)
            layer.check_decode(last, got, 2.0 ** -12 if cache_dtype == BF16 else 2.0 ** -15)
        total = sum(len(x) for x in layer.held)
        ks, vs = c.kv_cache_read(layer.cache, layer.pages.block_table, step.cu_seqlens_k, total, dtype=F32)
        want = [torch.cat(x) for x in zip(*(layer.stored(b) for b in range(SEQS)))]
        assert torch.equal(ks.cpu(), want[0].float()) and torch.equal(vs.cpu(), want[1].float())


def test_prompt_attention_over_a_4_bit_cache_in_chunks():
    """A prompt in three chunks through pages, write, read and attention_prefill: each chunk's attention is the 64-bit one over the
    stored tokens (3 roundings of bf16, as in test_attention_gpu.py)."""
    layer = Layer(I4)
    for turn, new in enumerate(([50, 0, 7, 1, 0, 33], [20, 16, 1, 0, 0, 60], [1, 40, 90, 3, 0, 1])):
        q, k, v = (randn((sum(new), h, D), 20 * turn + i) for i, h in enumerate((HQ, HKV, HKV)))
        step, got_q = layer.step(q.cuda(), k.cuda(), v.cuda(), new)
        layer.remember(k, v, new)
        cu_k = step.cu_seqlens_k
        ks, vs = c.kv_cache_read(layer.cache, layer.pages.block_table, cu_k, int(cu_k[-1]))  # bf16, exactly what is stored
        got = c.attention_prefill(got_q.bfloat16(), ks, vs, step.cu_seqlens_q, cu_k)
        stored = [torch.cat(x) for x in zip(*(layer.stored(b) for b in range(SEQS)))]
        want, size = ref.prefill(got_q.bfloat16(), *stored, step.cu_seqlens_q.tolist(), cu_k.tolist())
        assert ((got.double().cpu() - want).abs() <= 3 * 2.0 ** -8 * size).all()


@pytest.mark.parametrize("cache_dtype", [I4, BF16])
def test_captured_step_replays_as_the_sequences_go_on(cache_dtype):
    """Pages, write and attention of a step in one graph, padded to its rows, replayed with other tokens, cuts and ends, give what
    the calls give one by one in another layer."""
    rows = 2 * SEQS
    layers = [Layer(cache_dtype) for _ in range(2)]
    q, k, v = (randn((rows, h, D), i).cuda() for i, h in enumerate((HQ, HKV, HKV)))
    new, keep = torch.zeros(SEQS, dtype=torch.int32).cuda(), torch.full((SEQS,), 2 ** 31 - 1, dtype=torch.int32).cuda()
    out = c.KvStep.empty(layers[0].pages, rows)
    at = torch.zeros(SEQS, dtype=torch.int64).cuda()  # the row of each sequence's last new token (any, where it has none)

    def run(layer, out=None):
        step = c.kv_pages_step(layer.pages, new, rows, keep=keep, out=out)
        got_q = layer.write(q, k, v, step)
        last = got_q.index_select(0, at)
        return step, c.attention_decode(last, layer.cache, layer.pages.block_table, layer.pages.seq_lens)

    run(layers[0], out), run(layers[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, captured = run(layers[0], out)
    for turn in range(25):
        gen = torch.Generator().manual_seed(turn)
        new.copy_(torch.randint(0, 3, (SEQS,), generator=gen).int())
        keep.copy_(torch.where(torch.rand(SEQS, generator=gen) < 0.2, torch.randint(0, 20, (SEQS,), generator=gen), 2 ** 31 - 1).int())
        at.copy_((new.cumsum(0) - 1).clamp(min=0))
        for i, x in enumerate((q, k, v)):
            x.copy_(randn(x.shape, 100 * turn + i))
        graph.replay()
        step, want = run(layers[1])
        assert torch.equal(captured, want) and torch.equal(out.slots, step.slots) and torch.equal(out.cu_seqlens_k, step.cu_seqlens_k)
        assert torch.equal(layers[0].pages.block_table, layers[1].pages.block_table)
        assert torch.equal(layers[0].cache.k, layers[1].cache.k)


@pytest.mark.parametrize("cache_dtype,norms", [(I4, True), (I4, False), (BF16, True)])
def test_example_with_norms_and_a_4_bit_cache(cache_dtype, norms):
    """The example's tokens and chunks against its whole prompts. bf16 roundings move a key or value by up to 2^-8 of itself; of 4-bit
    codes, whose steps are up to a seventh of a group's largest, one in a hundred then falls to its neighbour, which is a few
    hundredths of the values' size in all. A token at the wrong place, or of another sequence, is an error of about 1."""
    from attention_block import Shape, run
    worst, _, _ = run(Shape(hidden=512, heads=8, kv_heads=2, head_dim=128, head_norms=norms), lengths=(70, 1, 260), steps=3, cache_dtype=cache_dtype)
    assert worst <= (0.2 if cache_dtype == I4 else 5 * 2.0 ** -8)
