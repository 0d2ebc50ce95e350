"""What f32 queries get from attention_decode over each cache type, and reads past 2^32 elements.

Over each sequence's result, relative in the 2-norm, for normal q, k and v of 64 or 128 elements a head. f16 and int8 caches: q
and p in two pieces of 11 bits, 2^-22 each; bf16 caches: three pieces of 8 bits, 2^-24. Scores are sums of up to 384 products of
about one in f32, times a scale of 1/8 or less: off by some 2^-24 sqrt(384) / 8 = 1.5e-7 of a nat for each rounding of their sums, and p
by as much; the exponentials by 2^-22. p V is summed in steps of 16 tokens a warp, up to 16 of them for 2000 tokens (2^-24 a step,
towards zero: 5e-7 on average), 70 for 9000. Together below 1e-6 up to 2000 tokens, and below 4e-6 at 9000. With two bf16 pieces
p and q end at 2^-17 and the result at 3e-6; with the 128s of int8 codes inside the sums it ends at 2e-6 to 4e-6.
"""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
from test_attention_gpu import make_cache, randn

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.mark.parametrize("cache_dtype", [BF16, F16, I8])
@pytest.mark.parametrize("lens,hq,hkv,d,page", [([40, 1, 333], 8, 2, 128, 16), ([9000], 8, 1, 128, 64), ([700, 1900], 6, 2, 64, 48)])
def test_decode_of_f32_queries(lens, hq, hkv, d, page, cache_dtype):
    cache, table = make_cache(lens, hkv, page, d, cache_dtype, 11)
    q = randn((len(lens), hq, d), 12)
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()).double().cpu()
    want, _ = ref.decode(q, cache, table, lens)
    error = (got - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))
    assert error.max() <= (1e-6 if max(lens) <= 2000 else 4e-6), error


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_read_past_32_bits(dtype):
    """A cache of more than 2^32 elements whose used pages lie at its end reads as the small cache that holds the same pages."""
    hkv, page, d = 8, 256, 128
    pages = 2 ** 32 // (hkv * page * d) + 9
    shape = (pages, hkv, page, d)
    small, table = make_cache([700, 300], hkv, page, d, I8, 4)
    cache = c.KvCache.empty(*shape, I8)
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(cache, name)[-small.num_pages:] = getattr(small, name)
    far = torch.where(table >= 0, table + pages - small.num_pages, table).cuda()
    cu = torch.tensor([0, 700, 1000], dtype=torch.int32).cuda()
    got, want = (c.kv_cache_read(x, t, cu, 1000, dtype=dtype) for x, t in ((cache, far), (small, table.cuda())))
    for g, w in zip(got, want):
        assert w.any() and torch.equal(g, w)
