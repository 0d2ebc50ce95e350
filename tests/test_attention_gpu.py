"""The two attentions on the GPU against their definitions in 64 bits, at the lengths, head layouts, strides and masks
where they can go wrong.

Tolerances, element by element, with A = sum_j p_j |v_j| (so that |o| <= A):
  attention_prefill  rounds each p_j and the output to the inputs' type, unit u = 2^-8 (bf16) or 2^-11 (f16): each costs
                     at most u A. Scores come from exact products summed in f32, at most about 2^-24 * 128 * sum |q k|,
                     which the third u A covers.
  attention_decode   rounds the output, u A, and holds q and p in two pieces of the cache's 16-bit type. In bf16 pieces
                     (16 bits) p is off by 2^-16 and a score by up to 2^-17 scale sum |q k|, which is about 2^-14 at
                     head_dim 128 and moves o by twice that: 2^-12 A in all. In f16 pieces (22 bits and more; f16 and
                     int8 caches) everything is below 2^-16 A.
"""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
from candelora_metal_kernels_b200 import _lib

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def randn(shape, seed, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def check_prefill(q, k, v, cu_q, cu_k, got, **kw):
    want, size = ref.prefill(q, k, v, cu_q.tolist(), cu_k.tolist(), **kw)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - 3 * ref.UNIT[q.dtype] * size).max()
    assert worst <= 0, worst
    assert not got[size.sum(-1) == 0].any()  # rows that see no key


PREFILL = [
    # (query lengths, key lengths or None, q heads, kv heads, head_dim, causal)
    ([1], None, 4, 2, 128, True),
    ([2, 1, 3], None, 4, 4, 64, True),
    ([127], None, 4, 1, 128, True),
    ([128, 129], None, 2, 2, 128, True),
    ([255, 1, 256, 257], None, 2, 1, 64, True),
    ([300, 0, 41], None, 8, 2, 128, True),
    ([65, 130], None, 8, 1, 128, False),
    ([33, 64, 200], None, 6, 2, 80, True),
    ([190, 70], None, 7, 1, 128, True),
    ([20, 90], None, 24, 2, 48, True),
    ([50], None, 100, 1, 32, True),
    ([77, 130], None, 4, 2, 16, True),
    ([64, 1, 100], [300, 513, 100], 4, 1, 128, True),       # later chunks of longer prompts
    ([64, 1, 33], [200, 129, 0], 8, 2, 96, False),
    ([200, 130, 5], [60, 1, 0], 4, 2, 128, True),           # more queries than keys: rows that see nothing
    ([40, 0, 0, 7], [40, 50, 0, 7], 4, 2, 64, True),        # sequences without queries
    ([700], None, 4, 1, 128, True),
    ([130], [1100], 16, 2, 128, True),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lq,lk,hq,hkv,d,causal", PREFILL)
def test_prefill(lq, lk, hq, hkv, d, causal, dtype):
    lk = lq if lk is None else lk
    q, k, v = (randn((sum(n), h, d), 10 + i, dtype) for i, (n, h) in enumerate([(lq, hq), (lk, hkv), (lk, hkv)]))
    cu_q, cu_k = cu(lq), cu(lk)
    got = c.attention_prefill(q, k, v, cu_q.cuda(), cu_k.cuda(), causal=causal)
    assert got.shape == q.shape and got.dtype == dtype
    check_prefill(q, k, v, cu_q, cu_k, got, causal=causal)


@pytest.mark.parametrize("lq,lk", [([702], None), ([601], [1202]), ([333, 901], None), ([64], [9000]), ([17, 700, 450], [3017, 700, 2450])])
def test_prefill_items_cut_between_blocks(lq, lk):
    """Enough work that blocks end and begin inside items, also inside an item's last key tile."""
    lk = lq if lk is None else lk
    q, k, v = (randn((sum(n), h, 16), 20 + i, BF16) for i, (n, h) in enumerate([(lq, 32), (lk, 8), (lk, 8)]))
    cu_q, cu_k = cu(lq), cu(lk)
    got = c.attention_prefill(q, k, v, cu_q.cuda(), cu_k.cuda())
    check_prefill(q, k, v, cu_q, cu_k, got)
    for _ in range(3):
        assert torch.equal(c.attention_prefill(q, k, v, cu_q.cuda(), cu_k.cuda()), got)


def test_prefill_slices_of_one_projection():
    """q, k and v as strided slices of [tokens, (hq + 2 hkv) d], and slices whose rows are not 16-byte aligned."""
    hq, hkv, d, lens = 8, 2, 64, [150, 31]
    for pad in (0, 8, 3):
        rows = randn((sum(lens), (hq + 2 * hkv) * d + pad), 1, BF16)
        q, k, v = (x.unflatten(1, (-1, d)) for x in rows[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
        got = c.attention_prefill(q, k, v, cu(lens).cuda())
        check_prefill(q, k, v, cu(lens), cu(lens), got)


def test_prefill_heads_first_layout_and_shared_heads():
    q, k, v = randn((4, 70, 64), 1, F16), randn((2, 70, 64), 2, F16), randn((2, 70, 64), 3, F16)
    lens = cu([70])
    got = c.attention_prefill(*(x.transpose(0, 1) for x in (q, k, v)), lens.cuda())
    check_prefill(*(x.transpose(0, 1) for x in (q, k, v)), lens, lens, got)
    k1 = randn((70, 1, 64), 4, F16).expand(70, 2, 64)  # one head's keys broadcast to two
    got = c.attention_prefill(q.transpose(0, 1), k1, v.transpose(0, 1), lens.cuda())
    check_prefill(q.transpose(0, 1), k1, v.transpose(0, 1), lens, lens, got)


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_prefill_masked_values_do_not_matter(poison):
    """Keys and values that a query does not see -- later tokens of its own sequence, tokens of other sequences -- may
    hold anything: each row equals the row of a call without them, and rows that do see them are not compared."""
    poison = torch.finfo(BF16).min if poison == "lowest" else poison
    lens, at = [300, 190, 40], [299, 290, 129, 300 + 100]  # positions, in the packed tensors, that are poisoned
    q, k, v = randn((530, 4, 128), 1, BF16), randn((530, 2, 128), 2, BF16), randn((530, 2, 128), 3, BF16)
    clean = c.attention_prefill(q, k, v, cu(lens).cuda())
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at] = poison, poison
    got = c.attention_prefill(q, k2, v2, cu(lens).cuda())
    for first, last in ((0, 129), (300, 400), (490, 530)):
        assert torch.equal(got[first:last], clean[first:last])
    if poison != torch.finfo(BF16).min:
        assert not torch.isfinite(got[299].float()).all(-1).any() and not torch.isfinite(got[450].float()).all(-1).any()


def test_prefill_scale_stream_out_and_repeat():
    q, k, v = randn((200, 4, 64), 1, F16), randn((200, 2, 64), 2, F16), randn((200, 2, 64), 3, F16)
    lens = cu([200])
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    lens_dev = lens.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = c.attention_prefill(q, k, v, lens_dev, scale=0.3, out=out)
    side.synchronize()
    assert got is out
    check_prefill(q, k, v, lens, lens, got, scale=0.3)
    assert torch.equal(got, c.attention_prefill(q, k, v, lens_dev, scale=0.3))


def test_prefill_large_scores():
    """Scores of hundreds (peaked rows, and running maxima that move a lot) stay exact softmaxes."""
    q, k, v = randn((260, 2, 128), 1, BF16) * 8, randn((260, 1, 128), 2, BF16) * 8, randn((260, 1, 128), 3, BF16)
    k[:, 0] *= torch.linspace(0.1, 3, 260, device="cuda").to(BF16)[:, None]  # the maximum grows along the row
    lens = cu([260])
    want, _ = ref.prefill(q, k, v, lens.tolist(), lens.tolist())
    got = c.attention_prefill(q, k, v, lens.cuda()).double().cpu()
    # a score of 2000 is held to 2^-24 * 2000 by its last rounding alone and to some 2^-12 over the sum: 1 % of p
    assert (got - want).norm() / want.norm() < 0.02


def test_prefill_wait_that_runs_out_is_reported_and_the_context_stays_usable():
    """With the test hook one warpgroup withholds the probabilities of a key tile: the waits behind them run out after 20 ms,
    device_check reports it once, and the same call is right again afterwards. No GPU fault is involved."""
    lib = _lib.load()
    q, k, v = randn((700, 4, 128), 1, BF16), randn((700, 2, 128), 2, BF16), randn((700, 2, 128), 3, BF16)
    lens = cu([700]).cuda()
    want = c.attention_prefill(q, k, v, lens)
    c.device_check()
    for tile in (1, 3):
        assert lib.iq2_testing_set_gemm_stall(20_000_000, tile) == _lib.IQ2_OK
        try:
            c.attention_prefill(q, k, v, lens)
            with pytest.raises(c.Iq2Error, match="prefill attention gave up on a pipeline wait") as e:
                c.device_check()
            assert e.value.code == _lib.IQ2_ERR_TIMEOUT
        finally:
            lib.iq2_testing_set_gemm_stall(0, 0)
        c.device_check()
        assert torch.equal(c.attention_prefill(q, k, v, lens), want)


# ---- one token over the cache ----

def make_cache(lens, hkv, page, d, dtype, seed, spare=3, poison=None):
    """A cache with random tokens for sequences of `lens`, over shuffled pages; whatever no sequence holds is `poison`."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need, default=0)) + 1), -1, dtype=torch.int32)
    used = torch.zeros((pages, page), dtype=torch.bool)
    i = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[i:i + need[b]]
        for p in range(n):
            used[table[b, p // page], p % page] = True
        i += need[b]
    k, v = randn((pages, hkv, page, d), seed + 1), randn((pages, hkv, page, d), seed + 2)
    if dtype == I8:
        (k, ks), (v, vs) = ref.quantised(k), ref.quantised(v)
        if poison is not None:
            ks.masked_fill_(~used.cuda()[:, None], poison)
            vs.masked_fill_(~used.cuda()[:, None], poison)
        return c.KvCache(k, v, ks.contiguous(), vs.contiguous()), table
    if poison is not None:
        k.masked_fill_(~used.cuda()[:, None, :, None], poison)
        v.masked_fill_(~used.cuda()[:, None, :, None], poison)
    return c.KvCache(k.to(dtype), v.to(dtype)), table


def check_decode(q, cache, table, lens, got, scale=None):
    want, size = ref.decode(q, cache, table, lens, scale)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    pieces = 2.0 ** -12 if cache.dtype == BF16 else 2.0 ** -16
    worst = ((got - want).abs() - ref.UNIT[q.dtype] * want.abs() - pieces * size).max()
    assert worst <= 0, worst
    assert not got[size.sum(-1) == 0].any()


DECODE = [
    # (lengths, q heads, kv heads, head_dim, page size)
    ([1], 4, 2, 128, 16),
    ([2, 0, 17], 4, 4, 64, 16),
    ([15, 16, 31, 32, 33, 63, 64, 65], 8, 2, 128, 32),
    ([127, 128, 129, 255, 257], 4, 1, 128, 64),
    ([300, 1, 0, 999], 16, 2, 128, 48),
    ([100, 41], 12, 4, 96, 7),          # pages that end inside every tile
    ([64, 200], 7, 1, 80, 128),
    ([50, 129], 24, 2, 48, 1),
    ([130, 64], 40, 1, 32, 100),
    ([77], 2, 2, 16, 256),
    ([5000], 8, 1, 128, 64),
    ([3, 2500, 700], 16, 4, 64, 16),
]


@pytest.mark.parametrize("cache_dtype", [BF16, F16, I8])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens,hq,hkv,d,page", DECODE)
def test_decode(lens, hq, hkv, d, page, dtype, cache_dtype):
    cache, table = make_cache(lens, hkv, page, d, cache_dtype, 5, poison=float("nan"))
    q = randn((len(lens), hq, d), 9, dtype)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    assert got.shape == q.shape and got.dtype == dtype
    check_decode(q, cache, table, lens, got)


@pytest.mark.parametrize("dtype,cache_dtype", [(F32, I8), (BF16, BF16)])
def test_decode_many_sequences(dtype, cache_dtype):
    """More (sequence, head) items than thread blocks, most of them short, one long."""
    lens = [(i * 37) % 90 for i in range(300)] + [3000]
    cache, table = make_cache(lens, 2, 16, 64, cache_dtype, 6)
    q = randn((len(lens), 4, 64), 9, dtype)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    check_decode(q, cache, table, lens, got)


def test_decode_q_strides_scale_stream_workspace_and_repeat():
    lens = [200, 333]
    cache, table = make_cache(lens, 2, 32, 128, BF16, 3)
    table, lens_dev = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    q = randn((2, 3 * 8 * 128 + 1), 1, BF16)[:, 1:].unflatten(1, (24, 128))[:, ::3]
    ws = torch.empty(max(1, c.attention_decode_workspace_bytes(q, cache, table)), dtype=torch.uint8, device="cuda")
    ws.fill_(255)
    out = torch.empty((2, 8, 128), dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = c.attention_decode(q, cache, table, lens_dev, scale=0.2, out=out, workspace=ws)
    side.synchronize()
    assert got is out
    check_decode(q, cache, table, lens, got, scale=0.2)
    assert torch.equal(got, c.attention_decode(q, cache, table, lens_dev, scale=0.2))


def test_decode_length_past_the_table_and_pages_outside_the_cache():
    """A length beyond the table's pages stops at them; tokens of pages outside the cache take no part."""
    lens = [100, 96]
    cache, table = make_cache(lens, 2, 16, 64, F16, 3)
    table = table[:, :6]  # 96 tokens
    q = randn((2, 4, 64), 1, F16)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([100, 1 << 30], dtype=torch.int32).cuda())
    check_decode(q, cache, table, [96, 96], got)
    holed = table.clone()
    holed[0, 2], holed[1, 5] = -7, cache.num_pages
    got = c.attention_decode(q, cache, holed.cuda(), torch.tensor([96, 96], dtype=torch.int32).cuda())
    keep = [p for p in range(96) if p // 16 != 2]
    k, v = ref.cached(cache, table[0], keep)
    want, size = ref.attend(q[0, 3:].double().cpu(), k[:, 1], v[:, 1], [80], 64 ** -0.5)
    assert ((got[0, 3].double().cpu() - want[0]).abs() <= 2 * ref.UNIT[F16] * size[0]).all()
    check_decode(q[1:], cache, table[1:], [80], got[1:])


def test_decode_offsets_past_32_bits():
    """A cache of more than 2^32 elements, whose used pages lie at its end."""
    hkv, page, d = 8, 256, 128
    pages = 2 ** 32 // (hkv * page * d) + 9
    shape = (pages, hkv, page, d)
    cache = c.KvCache(torch.zeros(shape, dtype=I8, device="cuda"), torch.zeros(shape, dtype=I8, device="cuda"),
                      torch.zeros(shape[:3], device="cuda"), torch.zeros(shape[:3], device="cuda"))
    small, table = make_cache([700], hkv, page, d, I8, 4)
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(cache, name)[-small.num_pages:] = getattr(small, name)
    q = randn((1, 16, d), 9)
    far = torch.where(table >= 0, table + pages - small.num_pages, table)
    lens = torch.tensor([700], dtype=torch.int32).cuda()
    assert torch.equal(c.attention_decode(q, cache, far.cuda(), lens), c.attention_decode(q, small, table.cuda(), lens))
    k, v = (randn((3, hkv, d), s) for s in (1, 2))
    slots = torch.tensor([(pages - 1) * page + 5, pages * page - 1, pages * page], dtype=torch.int32).cuda()
    c.kv_cache_write(cache, k, v, slots)  # the third slot lies past the end
    codes, scale = ref.quantised(k)
    assert torch.equal(cache.k[-1, :, 5], codes[0]) and torch.equal(cache.k_scale[-1, :, 255], scale[1])
    cu_ = torch.tensor([0, 700], dtype=torch.int32).cuda()
    a, b = c.kv_cache_read(cache, far.cuda(), cu_, 700), c.kv_cache_read(cache, far.cuda(), cu_, 700)
    assert torch.equal(a[0], b[0])


def test_refusals():
    q, kv = randn((4, 4, 64), 1, BF16), randn((4, 2, 64), 2, BF16)
    lens, cache = cu([4]).cuda(), c.KvCache.empty(4, 2, 16, 64)
    table, one = torch.zeros((4, 2), dtype=torch.int32).cuda(), torch.ones(4, dtype=torch.int32).cuda()

    def refused(match, fn, *args, **kw):
        with pytest.raises(c.Iq2Error, match=match):
            fn(*args, **kw)

    refused("all in f16 or all in bf16", c.attention_prefill, q.float(), kv.float(), kv.float(), lens)
    refused("all in f16 or all in bf16", c.attention_prefill, q, kv.half(), kv, lens)
    refused("expects k of shape", c.attention_prefill, q, kv[..., :32], kv, lens)
    refused("k has 4 tokens, v 3", c.attention_prefill, q, kv, kv[:3], lens)
    refused("device mismatch", c.attention_prefill, q, kv.cpu(), kv, lens)
    refused("requires a CUDA device", c.attention_prefill, q.cpu(), kv, kv, lens)
    refused("int32 tensor of rank 1", c.attention_prefill, q, kv, kv, lens.long())
    refused("entries", c.attention_prefill, q, kv, kv, lens, cu([4, 4]).cuda())
    refused("not a multiple", c.attention_prefill, randn((4, 3, 64), 1, BF16), kv, kv, lens)
    refused("head_dim=24", c.attention_prefill, q[..., :24], kv[..., :24], kv[..., :24], lens)
    refused("head_dim=256", c.attention_prefill, *(randn((4, 2, 256), 1, BF16) for _ in range(3)), lens)
    refused("scale is not positive", c.attention_prefill, q, kv, kv, lens, scale=-1.0)
    refused("out must be", c.attention_prefill, q, kv, kv, lens, out=torch.empty_like(q).half())
    refused("expects q of shape", c.attention_decode, q[..., :32], cache, table, one)
    refused("batch of 4", c.attention_decode, q, cache, table[:3], one)
    refused("unsupported q dtype", c.attention_decode, q.double(), cache, table, one)
    refused("not a multiple", c.attention_decode, randn((4, 3, 64), 1), cache, table, one)
    refused("unsupported cache dtype", c.KvCache, kv[None].float(), kv[None].float())
    refused("takes contiguous f32 scales", c.KvCache, cache.k.to(I8), cache.v.to(I8))
    refused("contiguous layouts", c.KvCache, cache.k.transpose(1, 2), cache.v.transpose(1, 2))
    refused("head_dim=24", c.attention_decode, randn((1, 2, 24), 1), c.KvCache.empty(2, 2, 16, 24), table[:1], one[:1])
    refused("slots", c.kv_cache_write, cache, kv, kv, one.long())
    refused("k has 4 tokens", c.kv_cache_write, cache, kv, kv, one[:3])
    refused("go together", c.kv_cache_write, cache, kv, kv, one, cos=torch.ones(4, 32).cuda())
    refused("cos and sin", c.kv_cache_write, cache, kv, kv, one, positions=one, cos=torch.ones(4, 16).cuda(), sin=torch.ones(4, 16).cuda())
    refused("q, k and v in one of", c.kv_cache_write, cache, kv, kv.float(), one)
    refused("go with q", c.kv_cache_write, cache, kv, kv, one, q_dtype=BF16)
    refused("unsupported out dtype", c.kv_cache_read, cache, table, cu([1] * 4).cuda(), 4, dtype=I8)
    refused("cu_seqlens", c.kv_cache_read, cache, table, lens, 4)


def test_empty_calls():
    cache = c.KvCache.empty(2, 2, 16, 64)
    z = torch.zeros(1, dtype=torch.int32).cuda()
    q, kv = torch.empty((0, 4, 64), dtype=BF16).cuda(), torch.empty((0, 2, 64), dtype=BF16).cuda()
    assert c.attention_prefill(q, kv, kv, z).shape == (0, 4, 64)
    assert c.attention_decode(q, cache, torch.zeros((0, 1), dtype=torch.int32).cuda(), z[:0]).shape == (0, 4, 64)
    assert c.kv_cache_write(cache, kv, kv, z[:0], q=q).shape == (0, 4, 64)
    assert c.kv_cache_read(cache, torch.zeros((0, 1), dtype=torch.int32).cuda(), z, 0)[0].shape == (0, 2, 64)
    got = c.attention_prefill(randn((3, 4, 64), 1, BF16), kv, kv, cu([3]).cuda(), cu([0]).cuda())
    assert got.shape == (3, 4, 64) and not got.any()  # no keys at all
