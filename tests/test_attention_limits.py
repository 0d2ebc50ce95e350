"""Sizes at which the attention operators' 32-bit numbers end: refused before anything is launched."""
import pytest
import torch

import candelora_metal_kernels_b200 as c
from candelora_metal_kernels_b200 import _lib
from candelora_metal_kernels_b200.build import build

I8 = torch.int8


@pytest.mark.gpu
def test_decode_units_of_an_item_line_past_32_bits():
    """A sequence of 2^31 - 1 tokens has 2^25 units of 64 tokens (and three more) in each of its 128 key heads' items."""
    cache = c.KvCache.empty(1, 128, 1 << 16, 16, torch.float16)
    table = torch.zeros((1, 1 << 15), dtype=torch.int32).cuda()  # the one page again and again
    lens = torch.tensor([5], dtype=torch.int32).cuda()
    q = torch.ones((1, 128, 16)).cuda()
    with pytest.raises(c.Iq2Error, match="too long a sequence"):
        c.attention_decode(q, cache, table, lens)
    half = c.KvCache(cache.k[:, :64].contiguous(), cache.v[:, :64].contiguous())
    assert not c.attention_decode(q[:, :64], half, table, lens).any()
    assert not c.attention_decode(torch.ones((1, 512, 16)).cuda(), half, table, lens).any()  # eight heads share an item


def _prefill(queries, keys):
    """iq2_attention_prefill of one query and key head, with pointers that are no memory of a device."""
    build()
    lib = _lib.load()
    args = _lib.ATTENTION_PROMPTS.pack(1 << 12, 64, 64, 1 << 12, 64, 64, 1 << 12, 64, 64, _lib.DTYPE_BF16, 1, queries, keys, 1, 1, 64,
                                       1 << 12, 1 << 12, 1, 0.0, 1 << 12)
    return lib.iq2_attention_prefill(args, None, 0, None), lib.iq2_last_error()


@pytest.mark.parametrize("queries,keys", [(4, 2 ** 31 - 1), (4, 2 ** 31 - 300), (2 ** 30, 2 ** 30)])
def test_prefill_lengths_past_31_bits(queries, keys):
    """A key's number, a tile of keys past it and the cost of an item on top are int32."""
    assert _prefill(queries, keys)[0] == _lib.IQ2_ERR_OVERFLOW
    assert _prefill(4, 2 ** 31 - 5000)[0] == _lib.IQ2_ERR_DEVICE  # (fits; the pointers are looked at next)
