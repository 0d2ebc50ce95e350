"""The attention block of a decoder layer with IQ2_XXS projections: a prompt, then single tokens.

    python examples/attention_block.py                 (Llama-3-8B shapes: 4096 hidden, 32 / 8 heads of 128)

Prompt:  pages for its tokens -> q, k, v projections (one grouped call) -> norms of the heads (where the layer has them), rotation
and cache write -> attention over the prompt -> o projection.
Token:   the same with the attention over the cache. A prompt may also come in chunks: the earlier tokens are read back
from the cache and the chunk attends to them and itself. The cache is 16-bit, int8, or 4-bit (torch.uint8).
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
    head_norms: bool = False


class AttentionBlock:
    """One layer's projections, its paged cache and the pages of `sequences` sequences of up to `most` tokens."""

    def __init__(self, shape: Shape, sequences: int, most: int, cache_dtype=torch.int8, page_size: int = 64, seed: int = 0):
        self.shape, self.page_size = shape, page_size
        rows = {"q": shape.heads * shape.head_dim, "k": shape.kv_heads * shape.head_dim, "v": shape.kv_heads * shape.head_dim}
        self.weights = {name: (*(t.cuda() for t in synth.iq2xxs_weights(n, shape.hidden, seed=seed + i)), n, shape.hidden)
                        for i, (name, n) in enumerate(rows.items())}
        self.weights["o"] = (*(t.cuda() for t in synth.iq2xxs_weights(shape.hidden, rows["q"], seed=seed + 9)), shape.hidden, rows["q"])
        pages = -(-most // page_size)
        self.cache = c.KvCache.empty(sequences * pages, shape.kv_heads, page_size, shape.head_dim, cache_dtype)
        self.pages = c.KvPages.empty(sequences * pages, page_size, sequences, pages)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        weights = [1 + 0.2 * torch.randn(shape.head_dim, generator=gen, device="cuda") for _ in range(2)] if shape.head_norms else [None] * 2
        self.q_norm, self.k_norm = weights
        half = shape.head_dim // 2
        angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * \
            shape.theta ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        self.cos, self.sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()

    def _project(self, x, q_dtype, step):
        """Rotated q [tokens, heads, head_dim] in q_dtype; k and v of x [tokens, hidden] go to the cache, where `step` says."""
        s = self.shape
        q, k, v = c.iq2_matmul_grouped([(x, *self.weights[name]) for name in "qkv"])
        k, v = (t.view(-1, s.kv_heads, s.head_dim) for t in (k, v))
        return c.kv_cache_write(self.cache, k, v, step.slots, q=q.view(-1, s.heads, s.head_dim), q_dtype=q_dtype,
                                positions=step.positions, cos=self.cos, sin=self.sin, q_norm=self.q_norm, k_norm=self.k_norm)

    def _output(self, attended):
        return c.iq2_xxs_matmul(attended.flatten(1), *self.weights["o"])

    def prompt(self, x, lengths):
        """x [tokens, hidden] (bf16) of packed prompts, or of their next chunks; f32 out."""
        step = c.kv_pages_step(self.pages, torch.tensor(lengths, dtype=torch.int32, device=x.device), x.shape[0])
        q = self._project(x, torch.bfloat16, step)
        # the keys and values as the cache holds them, so that prompts, chunks and single tokens see the same ones
        k, v = c.kv_cache_read(self.cache, self.pages.block_table, step.cu_seqlens_k, int(step.cu_seqlens_k[-1]), dtype=torch.bfloat16)
        return self._output(c.attention_prefill(q, k, v, step.cu_seqlens_q, step.cu_seqlens_k))

    def token(self, x):
        """x [sequences, hidden] (f32) of one new token each; f32 out."""
        step = c.kv_pages_step(self.pages, torch.ones(x.shape[0], dtype=torch.int32, device=x.device), x.shape[0])
        q = self._project(x, torch.float32, step)
        return self._output(c.attention_decode(q, self.cache, self.pages.block_table, self.pages.seq_lens))


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

    outs = []
    start = time.perf_counter()
    for i in range(steps):
        outs.append(block.token(torch.stack([x[n + i] for x, n in zip(xs, lengths)])))
    torch.cuda.synchronize()
    token_ms = (time.perf_counter() - start) * 1e3 / steps

    worst = 0.0
    for b, n in enumerate(lengths):  # each sequence again, whole and in two chunks
        whole = AttentionBlock(shape, 1, n + steps, cache_dtype)
        want = whole.prompt(xs[b].bfloat16(), [n + steps])
        chunked = AttentionBlock(shape, 1, n + steps, cache_dtype)
        half = (n + steps) // 2
        again = torch.cat([chunked.prompt(xs[b][:half].bfloat16(), [half]), chunked.prompt(xs[b][half:].bfloat16(), [n + steps - half])])
        for got, expected in ((torch.stack([o[b] for o in outs]), want[n:]), (again, want)):
            worst = max(worst, float((got - expected).norm() / expected.norm()))
    return worst, prompt_ms, token_ms


if __name__ == "__main__":
    run(steps=1)  # (warm-up)
    for dtype, norms in ((torch.int8, False), (torch.bfloat16, False), (torch.uint8, True)):
        worst, prompt_ms, token_ms = run(Shape(head_norms=norms), cache_dtype=dtype)
        print(f"{dtype}{', norms' if norms else ''}: prompts {prompt_ms:.2f} ms, a token {token_ms:.3f} ms, tokens and chunks against whole prompts {worst:.1e}")
