"""attention_decode where its 16-bit pieces have the least room: one token that takes nearly all of the weight and has a value
of nothing, and a channel of q that is thousands of times the others.

Tolerance, element by element, A = sum_j p_j |v_j|: the output rounded to q's type, u |o|, no finer than half of f16's smallest
spacing; the pieces and the sums within 2^-16 A over f16 and int8 caches.
"""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
from test_attention_range_gpu import sink_tokens

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def check(q, cache, table, lens, got):
    want, size = ref.decode(q, cache, table, lens)
    got = got.double().cpu()
    least = 2.0 ** -25 if q.dtype == F16 else 0.0
    worst = ((got - want).abs() - ref.UNIT[q.dtype] * want.abs() - 2.0 ** -16 * size - least).max()
    assert worst <= 0, worst


def paged(k, v, dtype, page=16):
    """A cache that holds one sequence's k, v [tokens, kv_heads, d] in order, and its table."""
    pages = -(-k.shape[0] // page)
    full = [torch.zeros((pages * page, *x.shape[1:]), device="cuda") for x in (k, v)]
    for f, x in zip(full, (k, v)):
        f[:x.shape[0]] = x.float()
    k, v = (f.view(pages, page, *f.shape[1:]).transpose(1, 2).contiguous() for f in full)
    table = torch.arange(pages, dtype=torch.int32)[None]
    if dtype != I8:
        return c.KvCache(k.to(dtype), v.to(dtype)), table
    (k, ks), (v, vs) = ref.quantised(k.cpu()), ref.quantised(v.cpu())
    return c.KvCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda()), table


@pytest.mark.parametrize("gap", [8, 12, 15, 17.5])
@pytest.mark.parametrize("cache_dtype", [F16, I8])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("tokens", [9, 64, 333, 5000])
def test_decode_sink(tokens, dtype, cache_dtype, gap):
    _, k, v = sink_tokens(0, tokens, 4, 2, 64, gap, F16)
    q = sink_tokens(0, 1, 4, 2, 64, gap, dtype, 7)[0]
    cache, table = paged(k, v, cache_dtype)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([tokens], dtype=torch.int32).cuda())
    check(q, cache, table, [tokens], got)


@pytest.mark.parametrize("cache_dtype", [F16, I8])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_decode_small_channels_beside_a_large_one(dtype, cache_dtype):
    """One channel of q is 2^12 and no key has anything there: the scores are made of the other channels."""
    gen = torch.Generator().manual_seed(3)
    q, k, v = torch.randn((1, 4, 64), generator=gen), torch.randn((700, 2, 64), generator=gen), torch.randn((700, 2, 64), generator=gen)
    q[..., 5], k[..., 5] = 4096, 0
    cache, table = paged(k.cuda(), v.cuda(), cache_dtype)
    q = q.to(dtype).cuda()
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([700], dtype=torch.int32).cuda())
    check(q, cache, table, [700], got)
