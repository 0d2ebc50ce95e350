"""The attention block of a decoder layer with IQ2_XXS projections: a prompt, then single tokens.

    python examples/attention_block.py                 (Llama-3-8B shapes: 4096 hidden, 32 / 8 heads of 128)

Prompt:  q, k, v projections (one grouped call) -> rotation and cache write -> attention over the prompt -> o projection.
Token:   the same with the attention over the cache. A prompt may also come in chunks: the earlier tokens are read back
from the cache and the chunk attends to them and itself.
"""
from __future__ import annotations

import sys
import time
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import candelora_metal_kernels_b200 as c  # noqa: E402
from candelora_metal_kernels_b200 import synth  # noqa: E402


@dataclass
class Shape:
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    theta: float = 500000.0


class AttentionBlock:
    """One layer's projections, its paged cache and a block table for `sequences` sequences of up to `most` tokens."""

    def __init__(self, shape: Shape, sequences: int, most: int, cache_dtype=torch.int8, page_size: int = 64, seed: int = 0):
        self.shape, self.page_size = shape, page_size
        rows = {"q": shape.heads * shape.head_dim, "k": shape.kv_heads * shape.head_dim, "v": shape.kv_heads * shape.head_dim}
        self.weights = {name: (*(t.cuda() for t in synth.iq2xxs_weights(n, shape.hidden, seed=seed + i)), n, shape.hidden)
                        for i, (name, n) in enumerate(rows.items())}
        self.weights["o"] = (*(t.cuda() for t in synth.iq2xxs_weights(shape.hidden, rows["q"], seed=seed + 9)), shape.hidden, rows["q"])
        pages = -(-most // page_size)
        self.cache = c.KvCache.empty(sequences * pages, shape.kv_heads, page_size, shape.head_dim, cache_dtype)
        self.table = torch.arange(sequences * pages, dtype=torch.int32, device="cuda").flip(0).view(sequences, pages).contiguous()
        half = shape.head_dim // 2
        angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * \
            shape.theta ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        self.cos, self.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()

    def _project(self, x, q_dtype, sequence, position):
        """Rotated q [tokens, heads, head_dim] in q_dtype; k and v of x [tokens, hidden] go to the cache. `sequence` and
        `position` [tokens] say where each token belongs."""
        s = self.shape
        q, k, v = c.iq2_matmul_grouped([(x, *self.weights[name]) for name in "qkv"])
        slots = self.table[sequence, position // self.page_size] * self.page_size + position % self.page_size
        k, v = (t.view(-1, s.kv_heads, s.head_dim) for t in (k, v))
        q = c.kv_cache_write(self.cache, k, v, slots.to(torch.int32), q=q.view(-1, s.heads, s.head_dim), q_dtype=q_dtype,
                             positions=position.to(torch.int32), cos=self.cos, sin=self.sin)
        return q, k, v

    def _output(self, attended):
        return c.iq2_xxs_matmul(attended.flatten(1), *self.weights["o"])

    def prompt(self, x, lengths, done=0):
        """x [tokens, hidden] (bf16) of packed prompts, or of their next chunks after `done` tokens each; f32 out."""
        dev = x.device
        seqs = len(lengths)
        cu = torch.tensor([0] + list(lengths), device=dev).cumsum(0).to(torch.int32)
        sequence = torch.repeat_interleave(torch.arange(seqs, device=dev), torch.tensor(lengths, device=dev))
        position = torch.arange(x.shape[0], device=dev) - cu[sequence].long() + done
        q, _, _ = self._project(x, torch.bfloat16, sequence, position)
        # the keys and values as the cache holds them, so that prompts, chunks and single tokens see the same ones
        cu_k = torch.tensor([0] + [n + done for n in lengths], device=dev).cumsum(0).to(torch.int32)
        k, v = c.kv_cache_read(self.cache, self.table[:seqs], cu_k, x.shape[0] + done * seqs, dtype=torch.bfloat16)
        return self._output(c.attention_prefill(q, k, v, cu, cu_k))

    def token(self, x, lengths):
        """x [sequences, hidden] (f32) of one new token each; `lengths` int32 [sequences] counts it. f32 out."""
        sequence = torch.arange(x.shape[0], device=x.device)
        q, _, _ = self._project(x, torch.float32, sequence, lengths.long() - 1)
        return self._output(c.attention_decode(q, self.cache, self.table[:x.shape[0]], lengths))


def run(shape: Shape = Shape(), lengths=(700, 1200, 333), steps: int = 8, cache_dtype=torch.int8):
    """A batch of prompts and `steps` tokens each; returns the largest relative difference (2-norm) between a token's
    output and the output of the prompt that ends with it, and the times."""
    block = AttentionBlock(shape, len(lengths), max(lengths) + steps, cache_dtype)
    gen = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn((n + steps, shape.hidden), generator=gen, device="cuda") for n in lengths]
    # normalised, with a gain that gives the synthetic weights' q, k and v values of about 1, as a trained layer's are
    block_gain = 4.0 / shape.hidden ** 0.5
    xs = [x / x.square().mean(-1, keepdim=True).sqrt() * block_gain for x in xs]

    torch.cuda.synchronize()
    start = time.perf_counter()
    block.prompt(torch.cat([x[:n] for x, n in zip(xs, lengths)]).bfloat16(), lengths)
    torch.cuda.synchronize()
    prompt_ms = (time.perf_counter() - start) * 1e3

    lens, outs = torch.tensor(lengths, dtype=torch.int32, device="cuda"), []
    start = time.perf_counter()
    for i in range(steps):
        lens += 1
        outs.append(block.token(torch.stack([x[n + i] for x, n in zip(xs, lengths)]), lens))
    torch.cuda.synchronize()
    token_ms = (time.perf_counter() - start) * 1e3 / steps

    worst = 0.0
    for b, n in enumerate(lengths):  # each sequence again, whole and in two chunks
        whole = AttentionBlock(shape, 1, n + steps, cache_dtype)
        want = whole.prompt(xs[b].bfloat16(), [n + steps])
        chunked = AttentionBlock(shape, 1, n + steps, cache_dtype)
        half = (n + steps) // 2
        again = torch.cat([chunked.prompt(xs[b][:half].bfloat16(), [half]), chunked.prompt(xs[b][half:].bfloat16(), [n + steps - half], half)])
        for got, expected in ((torch.stack([o[b] for o in outs]), want[n:]), (again, want)):
            worst = max(worst, float((got - expected).norm() / expected.norm()))
    return worst, prompt_ms, token_ms


if __name__ == "__main__":
    run(steps=1)  # (warm-up)
    for dtype in (torch.int8, torch.bfloat16):
        worst, prompt_ms, token_ms = run(cache_dtype=dtype)
        print(f"{dtype}: prompts {prompt_ms:.2f} ms, a token {token_ms:.3f} ms, tokens and chunks against whole prompts {worst:.1e}")
