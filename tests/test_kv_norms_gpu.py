"""The norms of queries and keys in the cache's write. The writer sums in 64 bits and rounds the reciprocal root and each product
to f32, so that its results are those of these operations on the CPU bit for bit (a root within 2^-28 of a rounding border
would not be). Against 64 bits a normed value is off by the three roundings, 3 2^-24 of itself and their products, and a
rotated one by 3 2^-24 (|a| + |b|) more."""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
import kv_step_reference as step_ref
from test_kv_cache_gpu import at_slots, randn, tables

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8, I4 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.uint8


def weights(heads, d, seed, own):
    return 1 + 0.3 * randn((heads, d) if own else (d,), seed)


def check_cache(cache, slots, k, v):
    """k and v in f32 against what the cache holds at the slots."""
    for x, name in ((k, "k"), (v, "v")):
        got = at_slots(getattr(cache, name), slots)
        if cache.dtype == I4:
            want = step_ref.quantised4(x)
            assert torch.equal(got, want[0]) and torch.equal(at_slots(getattr(cache, name + "_scale"), slots), want[2])
            groups = at_slots(getattr(cache, name + "_group").view(torch.uint8), slots)
            assert torch.equal(groups[..., :x.shape[-1] // 32], want[1][..., :x.shape[-1] // 32])
        elif cache.dtype == I8:
            codes, steps = ref.quantised(x)
            assert torch.equal(got, codes) and torch.equal(at_slots(getattr(cache, name + "_scale"), slots), steps)
        else:
            assert torch.equal(got, x.to(cache.dtype))


@pytest.mark.parametrize("rope", ["none", "half", "pairs"])
@pytest.mark.parametrize("dtype,q_dtype,cache_dtype", [(F32, F32, I4), (F32, BF16, BF16), (BF16, BF16, I8), (F16, F32, F16), (BF16, F16, I4),
                                                      (F16, F16, BF16)])
@pytest.mark.parametrize("tokens,hq,hkv,d,page,own", [(1, 4, 2, 128, 16, False), (37, 5, 1, 64, 7, True), (150, 8, 8, 96, 48, False),
                                                      (19, 3, 3, 32, 64, True)])
def test_write(tokens, hq, hkv, d, page, own, dtype, q_dtype, cache_dtype, rope):
    pages = -(-tokens // page) + 1
    cache = c.KvCache.empty(pages, hkv, page, d, cache_dtype)
    q, k, v = (randn((tokens, h, d), i, dtype) * s for i, (h, s) in enumerate(((hq, 3), (hkv, 0.2), (hkv, 1))))
    wq, wk = weights(hq, d, 5, own), weights(hkv, d, 6, own)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(4))[:tokens].to(torch.int32)
    pos = torch.randint(0, 500, (tokens,), generator=torch.Generator().manual_seed(5)).to(torch.int32)
    cos, sin = tables(500, d)
    kw = {} if rope == "none" else {"positions": pos.cuda(), "cos": cos.cuda(), "sin": sin.cuda(), "interleaved": rope == "pairs"}
    got_q = c.kv_cache_write(cache, k.cuda(), v.cuda(), slots.cuda(), q=q.cuda(), q_dtype=q_dtype, q_norm=wq.cuda(),
                             k_norm=wk.cuda(), norm_eps=1e-5, **kw).cpu()
    turn = (lambda x: x) if rope == "none" else (lambda x: ref.rotated(x, pos, cos, sin, rope == "pairs"))
    nq, nk = step_ref.normed(q, wq, 1e-5), step_ref.normed(k, wk, 1e-5)
    assert got_q.dtype == q_dtype and torch.equal(got_q, turn(nq).to(q_dtype))
    check_cache(cache, slots, turn(nk), v.float())
    exact = q.double() / (q.double().square().mean(-1, keepdim=True) + 1e-5).sqrt() * wq.double()
    assert ((nq.double() - exact).abs() <= 3.01 * 2.0 ** -24 * exact.abs()).all()
    if rope == "half" and q_dtype == F32:
        size = exact.abs() + exact.abs().roll(d // 2, -1)
        assert ((got_q.double() - ref.rotated(exact, pos, cos, sin, False)).abs() <= 6.1 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("cache_dtype", [I4, BF16])
@pytest.mark.parametrize("which", ["q", "k"])
def test_one_norm_only(which, cache_dtype):
    """Only the queries, or only the keys, have a norm; the others pass as they are. Also without queries at all."""
    tokens, hq, hkv, d = 21, 4, 2, 64
    q, k, v = (randn((tokens, h, d), i) for i, h in enumerate((hq, hkv, hkv)))
    w, slots = weights(1, d, 5, False), torch.arange(tokens, dtype=torch.int32)
    cache = c.KvCache.empty(2, hkv, 16, d, cache_dtype)
    out = c.kv_cache_write(cache, k.cuda(), v.cuda(), slots.cuda(), q=q.cuda(), **{which + "_norm": w.cuda()})
    assert torch.equal(out.cpu(), step_ref.normed(q, w, 1e-6) if which == "q" else q)
    check_cache(cache, slots, step_ref.normed(k, w, 1e-6) if which == "k" else k, v)
    if which == "k":
        again = c.KvCache.empty(2, hkv, 16, d, cache_dtype)
        assert c.kv_cache_write(again, k.cuda(), v.cuda(), slots.cuda(), k_norm=w.cuda()) is None
        check_cache(again, slots, step_ref.normed(k, w, 1e-6), v)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("pad", [0, 8, 4, 1])
def test_strided_rows_and_weights_off_the_boundaries(pad, dtype):
    hq, hkv, d, tokens = 4, 2, 96, 33
    rows = randn((tokens, (hq + 2 * hkv) * d + pad), 1, dtype).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    many = weights(1, 4 * d + 9, 5, False).cuda()
    wq, wk = many[1:1 + d], many[pad:pad + 2 * d].view(2, d)
    cache = c.KvCache.empty(3, hkv, 16, d, F16)
    slots = torch.arange(tokens, dtype=torch.int32).cuda()
    out = c.kv_cache_write(cache, k, v, slots, q=q, q_dtype=F32, q_norm=wq, k_norm=wk)
    assert torch.equal(out.cpu(), step_ref.normed(q.cpu(), wq.cpu(), 1e-6))
    check_cache(cache, slots.cpu(), step_ref.normed(k.cpu(), wk.cpu(), 1e-6), v.cpu().float())
    # weights that are not contiguous are copied
    wide = torch.stack([wq, wq], 1)
    assert torch.equal(c.kv_cache_write(cache, k, v, slots, q=q, q_dtype=F32, q_norm=wide[:, 0], k_norm=wk), out)


def test_rows_of_every_size():
    """Zeros, rows whose squares leave f32's range on either side, infinities and NaN."""
    d = 64
    x = randn((8, 1, d), 1)
    x[0], x[5, 0, 3], x[6, 0, 60] = 0, float("inf"), float("nan")
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3] = x[3].sign() * 3e38
    x[4] *= 1e-42
    w, slots = weights(1, d, 2, False), torch.arange(8, dtype=torch.int32)
    cache = c.KvCache.empty(1, 1, 8, d, BF16)
    for eps in (1e-6, 1e-38):
        out = c.kv_cache_write(cache, x.cuda(), x.cuda(), slots.cuda(), q=x.cuda(), q_norm=w.cuda(), k_norm=w.cuda(), norm_eps=eps).cpu()
        want = step_ref.normed(x, w, float(torch.tensor(eps)))
        assert torch.equal(out.nan_to_num(7), want.nan_to_num(7)) and torch.equal(out.isnan(), want.isnan())
        assert torch.isfinite(out[:5]).all() and not out[0].any() and out[6].isnan().all()
        assert ((out[2:4].square().mean(-1) - 1).abs() < 0.7).all()


def test_without_norms_it_is_the_plain_write():
    tokens, hkv, d = 40, 2, 128
    k, v, q = (randn((tokens, hkv, d), i, BF16).cuda() for i in range(3))
    slots = torch.arange(tokens, dtype=torch.int32).cuda()
    ones = torch.ones(d).cuda()
    a, b = (c.KvCache.empty(3, hkv, 16, d, I8) for _ in range(2))
    out = c.kv_cache_write(a, k, v, slots, q=q)
    normed = c.kv_cache_write(b, k, v, slots, q=q, q_norm=ones)
    assert torch.equal(out, q) and torch.equal(a.k, b.k) and torch.equal(a.v_scale, b.v_scale)
    assert torch.equal(normed.cpu(), step_ref.normed(q.cpu(), ones.cpu(), 1e-6).bfloat16())


def test_eps_is_an_f32():
    """Rows next to eps: they show in one of some ten whether eps is an f32 (0.1 is off by 1.5e-8) or has 64 bits."""
    x, w, eps = 0.01 * randn((500, 4, 32), 1), weights(4, 32, 2, True), float(torch.tensor(0.1))
    cache = c.KvCache.empty(1, 4, 8, 32, I4)
    out = c.kv_cache_write(cache, x.cuda(), x.cuda(), torch.full((500,), -1, dtype=torch.int32).cuda(), q=x.cuda(), q_norm=w.cuda(), norm_eps=0.1).cpu()
    assert torch.equal(out, step_ref.normed(x, w, eps)) and not torch.equal(out, step_ref.normed(x, w, 0.1))


def test_refusals():
    cache = c.KvCache.empty(2, 2, 16, 64)
    kv, q, one = torch.ones((4, 2, 64)).cuda(), torch.ones((4, 6, 64)).cuda(), torch.arange(4, dtype=torch.int32).cuda()
    w = torch.ones(64).cuda()

    def refused(match, **kw):
        with pytest.raises(c.Iq2Error, match=match):
            c.kv_cache_write(cache, kv, kv, one, **kw)

    refused("q_norm goes with q", q_norm=w)
    for eps in (0.0, -1.0, float("nan"), float("inf"), 1e300, 1e-60):
        refused("eps is not positive", k_norm=w, norm_eps=eps)
    refused("expects k_norm as f32", k_norm=w.half())
    refused("expects k_norm as f32", k_norm=torch.ones(32).cuda())
    refused("expects k_norm as f32", k_norm=torch.ones((3, 64)).cuda())
    refused("expects q_norm as f32", q=q, q_norm=torch.ones((2, 64)).cuda())
    refused("device mismatch", k_norm=w.cpu())
