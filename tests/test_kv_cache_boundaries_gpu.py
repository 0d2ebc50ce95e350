"""The cache's write where rows, tables or both lie off the 16-byte boundaries gives what it gives on them, bit for bit, whichever
kernel takes the call."""
import pytest
import torch

import candelora_metal_kernels_b200 as c
from test_kv_cache_gpu import randn, tables

pytestmark = pytest.mark.gpu
BF16, F16, F32, I8, I4 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.uint8


def shifted(x, by):
    """x on the device, `by` elements behind a 16-byte boundary."""
    held = torch.empty(x.numel() + by, dtype=x.dtype, device="cuda")
    held[by:].copy_(x.flatten())
    return held[by:].view(x.shape)


@pytest.mark.parametrize("rope", ["none", "half", "pairs"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cache_dtype", [BF16, F16, I8, I4])
@pytest.mark.parametrize("tokens,hq,hkv,d", [(1, 4, 2, 128), (45, 6, 3, 64), (200, 8, 8, 96), (33, 2, 1, 32)])
def test_write_on_and_off_the_boundaries(tokens, hq, hkv, d, cache_dtype, dtype, rope):
    q, k, v = (randn((tokens, h, d), i, dtype) for i, h in enumerate((hq, hkv, hkv)))
    slots = torch.randperm(tokens + 9, generator=torch.Generator().manual_seed(4))[:tokens].to(torch.int32).cuda()
    pos = torch.randint(0, 60, (tokens,), generator=torch.Generator().manual_seed(5)).to(torch.int32).cuda()
    cos, sin = tables(60, d)
    want = None
    for rows_by, tables_by in ((0, 0), (0, 1), (1, 0), (1, 3)):
        cache = c.KvCache.empty(-(-(tokens + 9) // 8), hkv, 8, d, cache_dtype)
        kw = {} if rope == "none" else {"positions": pos, "cos": shifted(cos, tables_by), "sin": shifted(sin, tables_by),
                                        "interleaved": rope == "pairs"}
        out = c.kv_cache_write(cache, shifted(k, rows_by), shifted(v, rows_by), slots, q=shifted(q, rows_by), q_dtype=F32, **kw)
        got = [out, *(t.view(torch.uint8) for t in cache._tensors)]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
