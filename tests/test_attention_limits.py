"""Sizes at which the attention operators' 32-bit numbers end: refused before anything is launched."""
import pytest
import torch

import candelora_metal_kernels_b200 as c

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
