"""The example: projections, cache and attentions run together. Tokens one by one, and prompts in chunks, give what whole
prompts give. The prompt's projections round x to bf16 and its attention rounds q and p to bf16 (2^-8 each); the tokens' do
not, so that outputs differ by a few such units."""
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_dtype", [torch.int8, torch.bfloat16, torch.float16])
def test_tokens_and_chunks_agree_with_whole_prompts(cache_dtype):
    from attention_block import Shape, run
    worst, _, _ = run(Shape(hidden=512, heads=8, kv_heads=2, head_dim=128), lengths=(70, 1, 260), steps=3, cache_dtype=cache_dtype)
    assert worst <= 5 * 2.0 ** -8
