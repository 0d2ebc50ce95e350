"""attention_prefill's rows that belong to no sequence: what lies before cu_seqlens_q[0] and from its last entry on, as in a
batch that is padded to a fixed size."""
import pytest
import torch

import candelora_metal_kernels_b200 as c

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cu,tokens,d", [([0, 5, 40], 43, 64), ([3, 3, 130], 700, 128), ([0, 0], 9, 16), ([7, 300], 300, 96), ([2, 2, 2], 2, 48)])
def test_rows_of_no_sequence_are_zeros(cu, tokens, d, dtype):
    q, k, v = (torch.randn((tokens, h, d), generator=torch.Generator().manual_seed(h)).to(dtype).cuda() for h in (6, 2, 3))
    k, v = k, v[:, :2].contiguous()
    out = torch.full_like(q, float("nan"))
    got = c.attention_prefill(q, k, v, torch.tensor(cu, dtype=torch.int32).cuda(), out=out)
    assert got is out
    assert not got[:cu[0]].any() and not got[cu[-1]:].any()
    inner = c.attention_prefill(q[cu[0]:cu[-1]], k[cu[0]:cu[-1]], v[cu[0]:cu[-1]], torch.tensor(cu, dtype=torch.int32).cuda() - cu[0])
    assert torch.equal(got[cu[0]:cu[-1]], inner)
