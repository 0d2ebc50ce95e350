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


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,before", [([700], 0), ([64], 9000), ([333, 901], 0), ([17, 450], 3000)])
def test_prefill_infinities_in_items_cut_between_blocks(lens, before, dtype):
    """Values of both infinities and NaN that some rows of a tile see and others do not, in items that several blocks have parts
    of: each row has what the formula gives, every time."""
    keys = [n + before for n in lens]
    q, k, v = (randn((n, h, 16), 3 + i, dtype) for i, (n, h) in enumerate([(sum(lens), 32), (sum(keys), 8), (sum(keys), 8)]))
    end = torch.tensor(keys).cumsum(0)
    for i, back in enumerate([1, 2, 9, 30, 60, 130, 200]):  # places from each sequence's end, where the causal mask cuts
        for e, n in zip(end.tolist(), keys):
            if back < n:
                v[e - back, i % 8, i::5] = (float("inf"), -float("inf"), float("nan"))[i % 3]
                v[e - back, (i + 1) % 8, i::7] = (-float("inf"), float("inf"), float("inf"))[i % 3]
    cu_q = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    cu_k = torch.tensor([0] + keys).cumsum(0).to(torch.int32)
    want, _ = ref.prefill(q, k, v, cu_q.tolist(), cu_k.tolist())
    first = None
    for _ in range(10):
        got = c.attention_prefill(q, k, v, cu_q.cuda(), cu_k.cuda())
        first = got if first is None else first
        assert torch.equal(got.view(torch.int16), first.view(torch.int16))
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())
    finite = want.isfinite()
    clean, size = ref.prefill(q, k, v.nan_to_num(0, 0, 0), cu_q.tolist(), cu_k.tolist())
    assert ((got - clean).abs() <= 3 * ref.UNIT[dtype] * size + (2.0 ** -25 if dtype == F16 else 0.0))[finite].all()
