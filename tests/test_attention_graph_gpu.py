"""The attention operators in CUDA graphs: a captured layer replayed with other inputs and lengths, calls that share a workspace,
and what a workspace held before. Same inputs give the same bits, captured or not, so that results are compared exactly."""
import pytest
import torch

import candelora_metal_kernels_b200 as c

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
HQ, HKV, D, PAGE = 8, 2, 64, 16


def randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def prompts(lens, keys, tokens, key_tokens, seed, dtype=BF16):
    """q, k, v of fixed sizes, of which sequences of `lens` queries and `keys` keys take the first part."""
    q, k, v = (randn((n, h, D), seed + i, dtype) for i, (n, h) in enumerate([(tokens, HQ), (key_tokens, HKV), (key_tokens, HKV)]))
    return q, k, v, i32([0] + lens).cumsum(0).int(), i32([0] + keys).cumsum(0).int()


def prefill_workspace(q, k, cu):
    from candelora_metal_kernels_b200 import _lib
    args = _lib.ATTENTION_PROMPTS.pack(*[0] * 9, 2, cu.shape[0] - 1, q.shape[0], k.shape[0], HQ, HKV, D, 0, 0, 1, 0.0, 0)
    return torch.empty(_lib.load().iq2_attention_prefill_workspace_size(args), dtype=torch.uint8, device="cuda")


SHAPES = [([700], [700]), ([64], [9000]), ([333, 0, 901], [333, 5, 901]), ([601, 7], [1202, 3000])]


@pytest.mark.parametrize("left", [1, -1, 0x3F800000])
@pytest.mark.parametrize("lens,keys", SHAPES)
def test_what_the_workspace_held_does_not_matter(lens, keys, left):
    """Items cut between blocks, over a workspace in which every word may look like a flag of a part that is there."""
    q, k, v, cu_q, cu_k = prompts(lens, keys, sum(lens), sum(keys), 1)
    ws = prefill_workspace(q, k, cu_q)
    ws.zero_()
    want = c.attention_prefill(q, k, v, cu_q, cu_k, workspace=ws)
    for _ in range(5):
        ws.view(torch.int32).fill_(left)
        assert torch.equal(c.attention_prefill(q, k, v, cu_q, cu_k, workspace=ws), want)
        assert torch.equal(c.attention_prefill(q, k, v, cu_q, cu_k, workspace=ws), want)  # over the call's own leavings


def test_captured_prefills_over_one_workspace():
    """Two captured calls in one graph and a third in another, all over one workspace, replayed in turn with new inputs."""
    sizes = [SHAPES[0], SHAPES[2], SHAPES[1]]
    inputs = [prompts(*s, sum(s[0]), sum(s[1]), 10 * i) for i, s in enumerate(sizes)]
    outs = [torch.empty_like(x[0]) for x in inputs]
    ws = max((prefill_workspace(x[0], x[1], x[3]) for x in inputs), key=lambda t: t.numel())
    for x, out in zip(inputs, outs):
        c.attention_prefill(*x, out=out, workspace=ws)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, members in zip(graphs, ([0, 1], [2])):
        with torch.cuda.graph(graph):
            for i in members:
                c.attention_prefill(*inputs[i], out=outs[i], workspace=ws)
    for turn in range(6):
        for i, x in enumerate(inputs):
            for j in range(3):
                x[j].copy_(randn(x[j].shape, 100 * turn + 10 * i + j, BF16))
            outs[i].fill_(float("nan"))
        for graph in (graphs if turn % 2 else graphs[::-1]):
            graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(inputs, outs):
            assert torch.equal(out, c.attention_prefill(*x))


@pytest.mark.parametrize("cache_dtype", [BF16, F16, I8])
def test_captured_layer_replays_with_new_inputs_and_lengths(cache_dtype):
    """Write, read and prefill of a batch of prompts, then the write and decode of their next tokens, captured once at fixed
    sizes: replays with other values and lengths (one of them empty) give what eager calls give."""
    seqs, most, tokens = 3, 640, 1000
    pages = seqs * most // PAGE
    dtype = F16 if cache_dtype == F16 else BF16
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).to(torch.int32).view(seqs, -1).cuda()
    cos, sin = randn((most, D // 2), 1), randn((most, D // 2), 2)
    b = {"q": randn((tokens, HQ, D), 3), "k": randn((tokens, HKV, D), 4), "v": randn((tokens, HKV, D), 5),
         "q1": randn((seqs, HQ, D), 6), "k1": randn((seqs, HKV, D), 7), "v1": randn((seqs, HKV, D), 8),
         "cu": i32([0] * (seqs + 1)), "slots": i32([-1] * tokens), "pos": i32([0] * tokens),
         "slots1": i32([-1] * seqs), "pos1": i32([0] * seqs), "lens1": i32([0] * seqs)}

    def layer(cache, b):
        rope = {"cos": cos, "sin": sin}
        q = c.kv_cache_write(cache, b["k"], b["v"], b["slots"], q=b["q"], q_dtype=dtype, positions=b["pos"], **rope)
        k, v = c.kv_cache_read(cache, table, b["cu"], tokens, dtype=dtype)
        y = c.attention_prefill(q, k, v, b["cu"])
        q1 = c.kv_cache_write(cache, b["k1"], b["v1"], b["slots1"], q=b["q1"], positions=b["pos1"], **rope)
        return q, k, v, y, q1, c.attention_decode(q1, cache, table, b["lens1"])

    cache = c.KvCache.empty(pages, HKV, PAGE, D, cache_dtype)
    layer(cache, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(cache, b)
    for turn, lens in enumerate(([500, 3, 200], [0, 639, 1], [333, 333, 334])):
        new = {n: randn(b[n].shape, 50 * turn + i) for i, n in enumerate(["q", "k", "v", "q1", "k1", "v1"])}
        seq = torch.repeat_interleave(torch.arange(seqs), torch.tensor(lens))
        pos = torch.cat([torch.arange(n) for n in lens])
        held = table.cpu()
        pad = tokens - len(pos)
        new["cu"] = torch.tensor([0] + lens).cumsum(0)
        new["pos"] = torch.nn.functional.pad(pos, (0, pad))
        new["slots"] = torch.nn.functional.pad(held[seq, pos // PAGE] * PAGE + pos % PAGE, (0, pad), value=-1)
        last = torch.tensor(lens)
        new["pos1"], new["lens1"] = last, last + 1
        new["slots1"] = held[torch.arange(seqs), last // PAGE] * PAGE + last % PAGE
        for name, x in new.items():
            b[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        eager = c.KvCache.empty(pages, HKV, PAGE, D, cache_dtype)
        want = layer(eager, b)
        for g, w in zip(got, want):
            assert torch.equal(g[:sum(lens)] if g.shape[0] == tokens else g, w[:sum(lens)] if w.shape[0] == tokens else w)
        assert not got[3][sum(lens):].any()  # rows of no sequence
