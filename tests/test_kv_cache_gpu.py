"""The cache's writer and reader on the GPU. The writer rounds each product and sum of the rotation by itself, so that its
results are those of the elementary f32 operations bit for bit: rotated values, codes and scales are compared exactly
with torch on the CPU. Against 64 bits a rotated value is off by at most 3 units of 2^-24 (|a| + |b|), and an int8 row by
half a step and that."""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def tables(rows, d):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2, dtype=torch.float64) * 2 / d)
    return angle.cos().float(), angle.sin().float()


def at_slots(x, slots):
    """[tokens, heads, ...] of a cache tensor [pages, heads, page, ...] at the slots."""
    page = x.shape[2]
    return x.cpu().transpose(1, 2).flatten(0, 1)[slots.long()] if page else x


@pytest.mark.parametrize("rope", ["none", "half", "pairs"])
@pytest.mark.parametrize("dtype,q_dtype,cache_dtype", [(F32, F32, I8), (F32, BF16, BF16), (BF16, BF16, I8), (F16, F32, F16),
                                                      (BF16, F16, F16), (F16, F16, I8)])
@pytest.mark.parametrize("tokens,hq,hkv,d,page", [(1, 4, 2, 128, 16), (37, 5, 1, 64, 7), (300, 8, 8, 96, 48), (19, 3, 3, 16, 64),
                                                  (50, 2, 1, 80, 1)])
def test_write(tokens, hq, hkv, d, page, dtype, q_dtype, cache_dtype, rope):
    pages = -(-tokens // page) + 2
    cache = c.KvCache.empty(pages, hkv, page, d, cache_dtype)
    q, k, v = randn((tokens, hq, d), 1, dtype), randn((tokens, hkv, d), 2, dtype), randn((tokens, hkv, d), 3, dtype)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(4))[:tokens].to(torch.int32)
    skipped = torch.zeros(tokens, dtype=torch.bool)
    skipped[tokens // 2::5] = tokens > 1
    given = torch.where(skipped, torch.where(slots % 2 == 0, -1, pages * page), slots).to(torch.int32)
    pos = torch.randint(0, 500, (tokens,), generator=torch.Generator().manual_seed(5)).to(torch.int32)
    cos, sin = tables(500, d)
    kw = {} if rope == "none" else {"positions": pos.cuda(), "cos": cos.cuda(), "sin": sin.cuda(), "interleaved": rope == "pairs"}
    got_q = c.kv_cache_write(cache, k.cuda(), v.cuda(), given.cuda(), q=q.cuda(), q_dtype=q_dtype, **kw).cpu()

    turn = (lambda x: x.float()) if rope == "none" else (lambda x: ref.rotated(x.float(), pos, cos, sin, rope == "pairs"))
    assert got_q.dtype == q_dtype and torch.equal(got_q, turn(q).to(q_dtype))
    for x, held, scale in ((turn(k), cache.k, cache.k_scale), (v.float(), cache.v, cache.v_scale)):
        got = at_slots(held, slots)
        assert not got[skipped].any()
        if cache_dtype != I8:
            assert torch.equal(got[~skipped], x.to(cache_dtype)[~skipped])
            continue
        codes, steps = ref.quantised(x)
        assert torch.equal(got[~skipped], codes[~skipped])
        assert torch.equal(at_slots(scale, slots)[~skipped], steps[~skipped])
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots.long()] = False
    assert not cache.k.cpu().transpose(1, 2).flatten(0, 1)[untouched].any()
    if rope != "none" and cache_dtype == I8 and dtype == F32:  # against the definition in 64 bits
        want = ref.rotated(k.double(), pos, cos, sin, rope == "pairs")
        got = at_slots(cache.k, slots).double() * at_slots(cache.k_scale, slots).double()[..., None]
        assert ((got - want).abs() <= (0.5 / 127 + 1e-5) * want.abs().amax(-1, keepdim=True))[~skipped].all()


@pytest.mark.parametrize("pad", [0, 4, 1])
def test_write_strided_and_unaligned_rows(pad):
    """k, v and q as slices of one projection, whose rows start on 16-byte boundaries or not."""
    hq, hkv, d, tokens = 4, 2, 64, 33
    rows = randn((tokens, (hq + 2 * hkv) * d + pad), 1).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    cache = c.KvCache.empty(3, hkv, 16, d, F16)
    slots = torch.arange(tokens, dtype=torch.int32).cuda()
    cos, sin = (x.cuda() for x in tables(40, d))
    out = c.kv_cache_write(cache, k, v, slots, q=q, positions=slots, cos=cos, sin=sin)
    pos = slots.cpu()
    assert torch.equal(out.cpu(), ref.rotated(q.cpu(), pos, cos.cpu(), sin.cpu(), False))
    assert torch.equal(at_slots(cache.v, pos), v.cpu().half())


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("pad", [0, 8, 4, 1])
def test_write_16_bit_rows_off_the_boundaries(pad, dtype, pairs):
    """16-bit slices of one projection that start on multiples of 16, 8 or 2 bytes: the same values, and codes, from all."""
    hq, hkv, d, tokens = 4, 2, 96, 21
    rows = randn((tokens, (hq + 2 * hkv) * d + pad), 2).to(dtype).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    slots = torch.arange(tokens, dtype=torch.int32).cuda()
    cos, sin = (x.cuda() for x in tables(40, d))
    cache = c.KvCache.empty(3, hkv, 8, d, I8)
    out = c.kv_cache_write(cache, k, v, slots, q=q, positions=slots, cos=cos, sin=sin, interleaved=pairs, q_dtype=F32)
    pos = slots.cpu()
    assert torch.equal(out.cpu(), ref.rotated(q.cpu().float(), pos, cos.cpu(), sin.cpu(), pairs))
    for got, x in ((cache.k, ref.rotated(k.cpu().float(), pos, cos.cpu(), sin.cpu(), pairs)), (cache.v, v.cpu().float())):
        assert torch.equal(at_slots(got, pos), ref.quantised(x)[0])


def test_write_rows_that_do_not_quantise():
    """Zeros, subnormal rows, infinities and NaN."""
    x = randn((6, 1, 64), 1)
    x[0], x[1], x[2, 0, 3], x[3, 0, 60] = 0, 1e-35, float("inf"), float("nan")
    x[4] *= 1e30
    cache = c.KvCache.empty(1, 1, 16, 64, I8)
    slots = torch.arange(6, dtype=torch.int32).cuda()
    c.kv_cache_write(cache, x.cuda(), x.cuda(), slots)
    table, cu = torch.zeros((1, 1), dtype=torch.int32).cuda(), torch.tensor([0, 6], dtype=torch.int32).cuda()
    k, v = (t.cpu()[:, 0] for t in c.kv_cache_read(cache, table, cu, 6, dtype=F32))
    assert not k[:2].any() and k[2:4].isnan().all() and torch.isfinite(k[4:]).all()
    want = ref.quantised(x)
    assert torch.equal(cache.k[0, 0, :6].cpu(), want[0][:, 0])
    assert torch.equal(k.nan_to_num(7), v.nan_to_num(7))


@pytest.mark.parametrize("cache_dtype,dtype", [(I8, BF16), (I8, F32), (BF16, BF16), (F16, F16), (F16, F32), (BF16, F16)])
@pytest.mark.parametrize("lens,start,hkv,d,page", [([1], 0, 2, 128, 16), ([0, 33, 0, 5, 100], 3, 3, 64, 7), ([700, 20], 0, 8, 96, 64),
                                                   ([64] * 9, 17, 1, 16, 48)])
def test_read(lens, start, hkv, d, page, cache_dtype, dtype):
    need = [-(-(n + start) // page) for n in lens]
    pages, total = sum(need) + 2, sum(lens)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b in range(len(lens)):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
    x = [randn((pages, hkv, page, d), s) for s in (2, 3)]
    if cache_dtype == I8:
        (k, ks), (v, vs) = (ref.quantised(t) for t in x)
        cache = c.KvCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
        held = [k.float() * ks[..., None], v.float() * vs[..., None]]
    else:
        cache = c.KvCache(*(t.to(cache_dtype).cuda() for t in x))
        held = [t.to(cache_dtype).float() for t in x]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    starts = torch.full((len(lens),), start, dtype=torch.int32).cuda()
    got = c.kv_cache_read(cache, table.cuda(), cu.cuda(), total + 3, starts=starts if start else None, dtype=dtype)
    for g, h in zip(got, held):
        want = [h[table[b, (start + i) // page], :, (start + i) % page] for b, n in enumerate(lens) for i in range(n)]
        assert g.dtype == dtype and torch.equal(g[:total].cpu(), torch.stack(want).to(dtype))
        assert not g[total:].any()  # rows of no sequence


def test_read_pages_outside_the_cache_are_zeros():
    cache = c.KvCache.empty(2, 1, 4, 16, F16)
    cache.k.fill_(1), cache.v.fill_(2)
    table = torch.tensor([[1, -1, 2, 0]], dtype=torch.int32).cuda()
    k, v = c.kv_cache_read(cache, table, torch.tensor([0, 20], dtype=torch.int32).cuda(), 20)
    want = torch.tensor([1.0] * 4 + [0.0] * 8 + [1.0] * 4 + [0.0] * 4)
    assert torch.equal(k[:, 0, 0].float().cpu(), want) and torch.equal(v[:, 0, 5].float().cpu(), 2 * want)


def test_default_dtypes_and_streams():
    cache = c.KvCache.empty(4, 2, 16, 64, I8)
    k = randn((10, 2, 64), 1, F16).cuda()
    slots = torch.arange(20, 30, dtype=torch.int32).cuda()
    table, cu = torch.arange(4, dtype=torch.int32)[None].cuda(), torch.tensor([0, 10], dtype=torch.int32).cuda()
    starts = torch.tensor([20], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = c.kv_cache_write(cache, k, k, slots, q=k)
        got, _ = c.kv_cache_read(cache, table, cu, 10, starts=starts)
    side.synchronize()
    assert q.dtype == F16 and torch.equal(q, k) and got.dtype == BF16
    assert ((got - k).abs().float() <= 0.01 * k.float().abs().amax(-1, keepdim=True)).all()
