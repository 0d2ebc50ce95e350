"""Attention of single tokens over 4-bit caches whose value rows are of any size: every token counts by its weight, whatever
the sizes of the values beside it; and queries and keys whose sizes' product passes f32.

Tolerance, element by element, as test_kv_int4_gpu.py derives it, with what f16 steps may do taken from the tokens' own weights and
rows: u |o| + 2^-15 max(1, scale sum |q k| / 13) A (2^-11 A more under 16-bit q) + n 2^-31 max_j p_j max |v_j|, A = sum_j p_j |v_j|. The
weights here are 2^-120 of the largest and more: f32's exponential ends at 2^-126.
"""
import math

import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
import kv_step_reference as step_ref
from test_kv_cache_gpu import randn

pytestmark = pytest.mark.gpu
BF16, F16, F32, I4 = torch.bfloat16, torch.float16, torch.float32, torch.uint8
LOG2E = 1.4426950408889634


def assert_near(q, k, v, got, scale, dtype, fine=False, lost=0.0):
    """q, got [heads, d] of one sequence and key head over k, v [n, d] as they are held, in 64 bits. `fine`: 22 bits of p. `lost`: the
    tokens' products that are too small, and half of the smallest number of the output's type."""
    q, got = q.double().cpu(), got.double().cpu()
    p = torch.softmax(q @ k.T * scale, -1)
    want, size = p @ v, p @ v.abs()
    part = 2.0 ** -15 * ((q.abs() @ k.abs().T * scale).amax(-1, keepdim=True) / 13).clamp(min=1)
    if dtype != F32 and not fine:
        part = part + ref.UNIT[F16]
    floor = len(k) * 2.0 ** -31 * (p * v.abs().amax(-1)).amax(-1, keepdim=True) + lost
    assert torch.isfinite(got).all()
    over = (got - want).abs() - ref.UNIT[dtype] * want.abs() - part * size - floor
    assert (over <= 0).all(), (over / size.clamp(min=1e-300)).max()


def sizes(kind, n, seed):
    """(log2 of each row's largest value, -inf: a row of zeros; log2 of each token's weight next to the largest)."""
    gen = torch.Generator().manual_seed(seed)
    weight = -torch.rand(n, generator=gen) * 14
    top = torch.full((n,), 127.9)
    if kind == "e36":
        top = torch.full((n,), 119.6)
    elif kind == "spread":  # any size beside any other
        top = torch.randint(-95, 128, (n,), generator=gen).float()
        weight = weight * 3
    elif kind == "zeros win":  # most of the weight is at rows of zeros
        top[::2] = -math.inf
        weight[1::2] -= 20
    elif kind == "zeros and e9":
        top = torch.full((n,), 30.0)
        top[::2] = -math.inf
    elif kind == "small win":
        top[::2] = -80
        weight[1::2] -= 100
    elif kind == "one large":
        top = torch.zeros(n)
        top[n // 2] = 127.9
    elif kind == "small":
        top = torch.full((n,), -99.0)
        top[::3] = -60
    return top, weight


def tokens(kind, n, d, seed, order):
    """K, V [n, d] and q [4, d] with about those weights (q along one direction, three quarters to all of it) and sizes."""
    top, weight = sizes(kind, n, seed)
    by = weight.argsort() if order == "rising" else weight.argsort(descending=True) if order == "falling" else torch.arange(n)
    top, weight = top[by], weight[by]
    along = randn((d,), seed + 1).sign()
    q = along[None] * torch.tensor([1.0, 0.95, 0.85, 0.75])[:, None]
    k = along[None] * (weight / LOG2E / d ** 0.5)[:, None] + 0.02 * randn((n, d), seed + 2)
    v = randn((n, d), seed + 3)
    v = v / v.abs().amax(-1, keepdim=True) * torch.exp2(top.double())[:, None]
    return k, v.clamp(-3.4e38, 3.4e38).float(), q


KINDS = ["e38", "e36", "spread", "zeros win", "zeros and e9", "small win", "one large", "small"]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("order", ["as they come", "rising", "falling"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,width", [(2, 2), (20, 2), (32, 1), (130, 9), (130, 600), (3000, 200)])
def test_value_rows_of_any_size(n, width, kind, order, dtype):
    """In a tile, across a warp's tiles, across the warps of a block, and across blocks (wide tables)."""
    d, page, hkv = 64, 16, 2
    pages = -(-n // page)
    cache = c.KvCache.empty(pages, hkv, page, d, I4)
    made = [tokens(kind, n, d, 10 * h + n, order) for h in range(hkv)]
    k, v = (torch.stack([m[i] for m in made], 1) for i in (0, 1))
    q = torch.cat([m[2] for m in made])[None].to(dtype)
    c.kv_cache_write(cache, k.cuda(), v.cuda(), torch.arange(n, dtype=torch.int32).cuda())
    table = torch.full((1, max(width, pages)), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages)
    got = c.attention_decode(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    held = [x.transpose(1, 2).reshape(-1, hkv, d)[:n] for x in step_ref.held4(cache)]
    for h in range(hkv):
        assert_near(q[0, 4 * h:4 * h + 4], held[0][:, h], held[1][:, h], got[0, 4 * h:4 * h + 4], d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sequences_of_different_sizes_in_a_batch(dtype):
    """A warp takes many items one after another: each has a reference and a level of its own."""
    d, page, n, batch = 128, 16, 45, 160
    cache = c.KvCache.empty(batch * 3, 1, page, d, I4)
    made = [tokens(KINDS[b % len(KINDS)], n, d, b, "as they come") for b in range(batch)]
    table = torch.randperm(batch * 3, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(batch, 3)
    pos = torch.arange(n)
    slots = (table[:, pos // page] * page + pos % page).flatten().to(torch.int32)
    k, v = (torch.cat([m[i] for m in made])[:, None] for i in (0, 1))
    q = torch.stack([m[2] for m in made]).to(dtype)
    c.kv_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    wide = torch.nn.functional.pad(table, (0, 500), value=-1).cuda()
    got = c.attention_decode(q.cuda(), cache, wide, torch.full((batch,), n, dtype=torch.int32).cuda())
    held = step_ref.held4(cache)
    for b in range(batch):
        rows = [x[table[b].long()].transpose(1, 2).reshape(-1, d)[:n] for x in held]
        assert_near(q[b], *rows, got[b], d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_top,k_top", [(1e30, 1e20), (3e38, 3e38), (1e19, 1e19), (1.0, 3e38), (3e38, 1.0)])
def test_large_keys_that_large_queries_do_not_see(q_top, k_top, dtype):
    """Products of the sizes of q and k that pass f32, where q . k is 0: the score is 0, beside scores of a few units."""
    d, n = 128, 70
    q, k, v = (randn(shape, i) for i, shape in enumerate(((1, 8, d), (n, 1, d), (n, 1, d))))
    q[..., 32:], k[..., :32] = 0, 0
    q, k = q / q.abs().max() * q_top, k / k.abs().max() * k_top
    if 1e3 < q_top < 1e31:  # these see q, by a few units
        k[::3, :, :32] = randn((len(k[::3]), 1, 32), 5) / q_top
        k[::3, :, 32:] = 0
    q = q.to(dtype)
    cache = c.KvCache.empty(5, 1, 16, d, I4)
    c.kv_cache_write(cache, k.cuda(), v.cuda(), torch.arange(n, dtype=torch.int32).cuda())
    table = torch.arange(5, dtype=torch.int32)[None]
    got = c.attention_decode(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    held = [x.transpose(1, 2).reshape(-1, d)[:n] for x in step_ref.held4(cache)]
    assert_near(q[0], *held, got[0], d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,width", [(3, 1), (32, 2), (77, 5), (1000, 200)])
@pytest.mark.parametrize("kind", ["either sign", "any size", "subnormal", "one of 2^120", "zero"])
def test_row_scales_that_the_write_does_not_make(kind, n, width, dtype):
    """Read and decode agree on every cache that the format allows: row scales below zero, of any size, no powers of two, zero under
    codes that are not. Products below 2^-125 may be lost (a level ends at 2^112)."""
    if dtype == F16 and kind == "one of 2^120":
        pytest.skip("f16 outputs end at 65504")
    d, page, pages = 64, 16, -(-n // 16)
    gen = torch.Generator().manual_seed(n)
    codes = [torch.randint(0, 256, (pages, 1, page, d // 2), generator=gen).to(torch.uint8) for _ in range(2)]
    groups = [torch.randint(40, 80, (pages, 1, page, 4), generator=gen).to(torch.uint8) for _ in range(2)]
    either = torch.randint(0, 2, (2, pages, 1, page), generator=gen) * 2.0 - 1
    scales = either * (0.5 + torch.rand(either.shape, generator=gen)) * 0.02
    size = torch.zeros(either.shape[1:], dtype=torch.float64)
    if kind == "any size":
        size = torch.randint(-140, 10 if dtype == F16 else 100, size.shape, generator=gen).double()
    elif kind == "subnormal":
        size -= 130
    elif kind == "one of 2^120":
        groups[1].view(-1, 4)[n // 2] = torch.tensor([0, 1, 2, 3])  # so that the elements stay finite
        size.view(-1)[n // 2] = 123
    elif kind == "zero":
        scales[:, ::2] = 0
    scales = [scales[0].contiguous(), (scales[1].double() * torch.exp2(size)).float()]
    (k, v), (kg, vg), (ks, vs) = ([x.cuda() for x in t] for t in (codes, groups, scales))
    cache = c.KvCache(k, v, ks, vs, kg.view(torch.float8_e4m3fn), vg.view(torch.float8_e4m3fn))
    table = torch.full((1, max(width, pages)), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages)
    held = [x.transpose(1, 2).reshape(-1, d)[:n] for x in step_ref.held4(cache)]
    assert torch.isfinite(held[1].float()).all()
    got = c.kv_cache_read(cache, table.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), n, dtype=F32)
    assert all(torch.equal(g[:, 0].cpu(), h.float()) for g, h in zip(got, held))
    q = 0.1 * randn((1, 8, d), 3, dtype)
    got = c.attention_decode(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    assert_near(q[0], *held, got[0], d ** -0.5, dtype, lost=n * 2.0 ** -125 + (2.0 ** -25 if dtype == F16 else 0.0))
