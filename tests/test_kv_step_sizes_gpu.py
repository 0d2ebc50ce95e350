"""Sizes of a serving step that the other tests leave out: norms of head dimensions that are no multiple of 32, and decode attention over a
4-bit cache for more sequences than a warp's lanes many times over."""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
import kv_step_reference as step_ref
from test_kv_cache_gpu import at_slots, randn, tables
from test_kv_int4_gpu import check_decode, make_cache
from test_kv_norms_gpu import check_cache, weights

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.mark.parametrize("rope", ["none", "half", "pairs"])
@pytest.mark.parametrize("dtype,cache_dtype,pad", [(F32, BF16, 0), (BF16, I8, 0), (F16, F16, 3), (F32, I8, 1), (BF16, BF16, 8)])
@pytest.mark.parametrize("d", [16, 48, 80, 112])
@pytest.mark.parametrize("own", [False, True])
def test_norms_of_any_head_dim(own, d, dtype, cache_dtype, pad, rope):
    tokens, hq, hkv, page = 29, 6, 3, 8
    rows = randn((tokens, (hq + 2 * hkv) * d + pad), 1, dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    dev = rows.cuda()
    dq, dk, dv = (x.unflatten(1, (-1, d)) for x in dev[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    wq, wk = weights(hq, d, 5, own), weights(hkv, d, 6, own)
    cache = c.KvCache.empty(5, hkv, page, d, cache_dtype)
    slots = torch.randperm(5 * page, generator=torch.Generator().manual_seed(4))[:tokens].to(torch.int32)
    pos = torch.randint(0, 90, (tokens,), generator=torch.Generator().manual_seed(5)).to(torch.int32)
    cos, sin = tables(90, d)
    kw = {} if rope == "none" else {"positions": pos.cuda(), "cos": cos.cuda(), "sin": sin.cuda(), "interleaved": rope == "pairs"}
    got = c.kv_cache_write(cache, dk, dv, slots.cuda(), q=dq, q_dtype=F32, q_norm=wq.cuda(), k_norm=wk.cuda(), norm_eps=1e-5, **kw).cpu()
    turn = (lambda x: x) if rope == "none" else (lambda x: ref.rotated(x, pos, cos, sin, rope == "pairs"))
    assert torch.equal(got, turn(step_ref.normed(q, wq, 1e-5)))
    check_cache(cache, slots, turn(step_ref.normed(k, wk, 1e-5)), v.float())
    untouched = torch.ones(5 * page, dtype=torch.bool)
    untouched[slots.long()] = False
    assert not at_slots(cache.k, torch.arange(5 * page))[untouched].any() and not at_slots(cache.v, torch.arange(5 * page))[untouched].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,most,width", [(33, 400, 30), (513, 150, 200), (2000, 40, 3), (1000, 1, 1)])
def test_decode_of_many_sequences(n, most, width, dtype):
    lens = [(37 * i) % (most + 1) if i % 11 else 0 for i in range(n)]
    cache, table = make_cache(lens, 1, 16, 32, 7)
    table = torch.nn.functional.pad(table, (0, max(0, width - table.shape[1])), value=-1)
    q = randn((n, 4, 32), 8, dtype).cuda()
    check_decode(q, cache, table, lens, c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()))
