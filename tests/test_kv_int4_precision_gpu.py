"""How many bits of the weights the attention of single tokens over 4-bit caches keeps: 22 under f32 and f16 q, whose outputs would
show fewer, 11 under bf16 q. Values that cancel show it, since the output's own rounding is small then.

Tolerance, as test_kv_int4_gpu.py derives it: u |o| + 2^-15 max(1, scale sum |q k| / 13) A + n 2^-31 max_j p_j max |v_j|,
A = sum_j p_j |v_j|, and 2^-11 A more under bf16 q only."""
import pytest
import torch

import candelora_metal_kernels_b200 as c
import kv_step_reference as step_ref
from test_kv_cache_gpu import randn
from test_kv_int4_range_gpu import assert_near

pytestmark = pytest.mark.gpu
BF16, F16, F32, I4 = torch.bfloat16, torch.float16, torch.float32, torch.uint8


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,width,d", [(2, 1, 128), (6, 1, 64), (40, 3, 96), (500, 300, 128), (500, 300, 32)])
def test_weights_of_values_that_cancel(n, width, d, dtype):
    page, pages = 16, -(-n // 16)
    cache = c.KvCache.empty(pages, 1, page, d, I4)
    v = randn((n, 1, d), 1)
    v[1::2] = -v[0::2] * (1 + 0.02 * randn((n // 2, 1, 1), 2))
    k, q = randn((n, 1, d), 3) * 0.3, randn((1, 8, d), 4, dtype)
    c.kv_cache_write(cache, k.cuda(), v.cuda(), torch.arange(n, dtype=torch.int32).cuda())
    table = torch.full((1, max(width, pages)), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages)
    got = c.attention_decode(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    held = [x.transpose(1, 2).reshape(-1, d)[:n] for x in step_ref.held4(cache)]
    assert_near(q[0], *held, got[0], d ** -0.5, dtype, fine=dtype != BF16)
