"""attention_decode where its 16-bit pieces have the least room: one token that takes nearly all of the weight and has a value
of nothing, a channel of q that is thousands of times the others, and value rows of an int8 cache down to the smallest that it
holds.

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


def small_value_rows(kind, tokens):
    """k and v [tokens, 2, 64]; value rows whose largest lies between 2^-100 (what an int8 cache still holds) and 2^-93, all of
    them or beside rows of zeros, of 2^-80 or (tokens 2, 52, ...) of ordinary size. The scores grow by seven nats along the
    sequence."""
    gen = torch.Generator().manual_seed(tokens)
    k, v = torch.randn((tokens, 2, 64), generator=gen), torch.randn((tokens, 2, 64), generator=gen)
    k[..., 0] = torch.linspace(0, 7, tokens)[:, None]
    v *= 2.0 ** torch.randint(-100, -93, (tokens, 2, 1), generator=gen)
    if kind == "zeros":
        v[::3] = 0
    elif kind == "larger":
        v[1::3] *= 2.0 ** 20
    elif kind == "ordinary":
        v[2::50] *= 2.0 ** 97
    return k.cuda(), v.cuda()


@pytest.mark.parametrize("kind", ["all", "zeros", "larger"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [1, 100, 20000])
def test_decode_small_value_rows(tokens, dtype, kind):
    k, v = small_value_rows(kind, tokens)
    q = torch.randn((1, 4, 64), generator=torch.Generator().manual_seed(1))
    q[..., 0] = 8  # with a scale of 1 / 8: the score's growth
    q = q.to(dtype).cuda()
    cache, table = paged(k, v, I8, 64)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([tokens], dtype=torch.int32).cuda())
    check(q, cache, table, [tokens], got)


def test_decode_value_rows_of_zeros():
    """Every value is zero: so is the result, however long the sequence and whatever the scores."""
    k, _ = small_value_rows("all", 20000)
    cache, table = paged(k, torch.zeros_like(k), I8, 64)
    q = torch.full((1, 4, 64), 8.0).cuda()
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([20000], dtype=torch.int32).cuda())
    assert not got.any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [100, 20000])
def test_decode_small_value_rows_beside_ordinary_ones(tokens, dtype):
    """A product of p and a value scale is off by 2^-43 of the head's largest one at most, whatever its own size: with codes of
    up to 127, tokens * 127 * 2^-43 of that on top. (Elements in which the ordinary rows have codes of zero are made of the
    small rows alone, 2^-97 of the others.)"""
    k, v = small_value_rows("ordinary", tokens)
    q = torch.randn((1, 4, 64), generator=torch.Generator().manual_seed(1))
    q[..., 0] = 8
    q = q.to(dtype).cuda()
    cache, table = paged(k, v, I8, 64)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([tokens], dtype=torch.int32).cuda()).double().cpu()
    want, size = ref.decode(q, cache, table, [tokens])
    kk, _ = ref.cached(cache, table[0], range(tokens))
    scales = cache.v_scale.double().cpu().transpose(1, 2).flatten(0, 1)[:tokens]
    for h in range(4):
        largest = (torch.softmax(kk[:, h // 2] @ q[0, h].double().cpu() / 8, 0) * scales[:, h // 2]).max()
        bound = ref.UNIT[dtype] * want[0, h].abs() + 2.0 ** -16 * size[0, h] + tokens * 127 * 2.0 ** -43 * largest + (2.0 ** -25 if dtype == F16 else 0.0)
        assert ((got[0, h] - want[0, h]).abs() <= bound).all()
