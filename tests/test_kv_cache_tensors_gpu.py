"""A KvCache and its tensors: calls use the memory that the tensors have, or refuse."""
import pytest
import torch

import candelora_metal_kernels_b200 as c

pytestmark = pytest.mark.gpu
BF16, I8 = torch.bfloat16, torch.int8


def calls(cache):
    """Each operator that takes a cache, over its first page."""
    x = torch.ones((1, 2, 64), dtype=BF16, device="cuda")
    zero, one = (torch.full((1,), n, dtype=torch.int32, device="cuda") for n in (0, 1))
    table, cu = zero[None], torch.arange(2, dtype=torch.int32, device="cuda")
    return [lambda: c.kv_cache_write(cache, x, x, zero), lambda: c.kv_cache_read(cache, table, cu, 1),
            lambda: c.attention_decode(x, cache, table, one)]


@pytest.mark.parametrize("dtype", [BF16, I8])
def test_tensors_cannot_be_replaced(dtype):
    cache, other = (c.KvCache.empty(n, 2, 16, 64, dtype) for n in (2, 4))
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(other, name))
    assert cache.k.shape[0] == 2
    for call in calls(cache):
        call()


@pytest.mark.parametrize("dtype,name", [(BF16, "k"), (BF16, "v"), (I8, "k"), (I8, "v"), (I8, "k_scale"), (I8, "v_scale")])
def test_tensors_that_moved_are_refused(dtype, name):
    cache = c.KvCache.empty(2, 2, 16, 64, dtype)
    kept = getattr(cache, name).clone()
    getattr(cache, name).data = kept  # other memory under the same tensor
    for call in calls(cache):
        with pytest.raises(c.Iq2Error, match="have moved"):
            call()
    again = c.KvCache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    for call in calls(again):
        call()
