"""Rows in which one token takes nearly all of the weight (an attention sink) and has a value of nothing, so that the output is
made of probabilities far below the row's largest one.

Tolerances, element by element, A = sum_j p_j |v_j|, u half a unit of the type in the last place:
  attention_prefill  p rounded to the inputs' type, u A; the output rounded, u |o| <= u A, and no finer than half of f16's
                     smallest spacing, 2^-25; scores and sums in f32 within the third u A.
"""
import math

import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def sink_tokens(first, tokens, q_heads, kv_heads, d, gap, dtype, seed=1):
    """q [tokens, ...], k, v [first + tokens, ...]: every score of key 0 lies about `gap` nats above the others, which lie
    within about one nat of each other; the value of key 0 is zero, the others' are around 100."""
    q, k, v = randn((tokens, q_heads, d), seed), randn((first + tokens, kv_heads, d), seed + 1), randn((first + tokens, kv_heads, d), seed + 2) * 100
    q[..., 0] = 8
    k *= 0.3
    k[..., 0] = 0
    k[0] = 0
    k[0, :, 0] = gap * math.sqrt(d) / 8
    v[0] = 0
    return q.to(dtype), k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("gap", [8, 12, 15, 17.5])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,before", [([20], 0), ([130, 3], 0), ([600], 0), ([40], 3000)])
def test_prefill_sink(lens, before, dtype, gap):
    parts = [sink_tokens(before, n, 8, 2, 64, gap, dtype, 10 * i) for i, n in enumerate(lens)]
    q, k, v = (torch.cat(x) for x in zip(*parts))
    cu_q = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    cu_k = torch.tensor([0] + [n + before for n in lens]).cumsum(0).to(torch.int32)
    got = c.attention_prefill(q, k, v, cu_q.cuda(), cu_k.cuda()).double().cpu()
    want, size = ref.prefill(q, k, v, cu_q.tolist(), cu_k.tolist())
    worst = ((got - want).abs() - 3 * ref.UNIT[dtype] * size - (2.0 ** -25 if dtype == F16 else 0.0)).max()
    assert worst <= 0, worst
