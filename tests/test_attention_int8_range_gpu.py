"""Attention of single tokens over int8 caches whose value rows are of any size: every token counts by its weight, whatever the
sizes of the values beside it, and value scales have either sign.

Tolerance, element by element, A = sum_j p_j |v_j|: the output's rounding, u |o|; pieces and sums within 2^-16 A
(test_attention_gpu.py), in proportion where scale sum |q k| is more than 13; a product of p and a value scale is off by 2^-43 of the
head's largest one, 127 2^-43 with its code, a token; under bf16 q the 128s that codes are held with are in the sums: 2^-16 of
sum_j p_j max |v_j| once more, a code being up to 127 and 255 with them.
"""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
from test_kv_cache_gpu import randn
from test_kv_int4_range_gpu import KINDS, tokens

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def assert_near(q, k, v, got, dtype):
    q, got = q.double().cpu(), got.double().cpu()
    p = torch.softmax(q @ k.T * q.shape[-1] ** -0.5, -1)
    want, size, rows = p @ v, p @ v.abs(), (p * v.abs().amax(-1))
    part = 2.0 ** -16 * ((q.abs() @ k.abs().T * q.shape[-1] ** -0.5).amax(-1, keepdim=True) / 13).clamp(min=1)
    floor = len(k) * 2.0 ** -43 * rows.amax(-1, keepdim=True)
    if dtype == BF16:
        floor = floor + 3 * part * rows.sum(-1, keepdim=True)
    assert torch.isfinite(got).all()
    over = (got - want).abs() - ref.UNIT[dtype] * want.abs() - part * size - floor
    assert (over <= 0).all(), (over / size.clamp(min=1e-300)).max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("order", ["as they come", "rising", "falling"])
@pytest.mark.parametrize("kind", KINDS + ["either sign"])
@pytest.mark.parametrize("n", [2, 20, 130, 5000])
def test_value_rows_of_any_size(n, kind, order, dtype):
    d, page, hkv = 64, 16, 2
    pages = -(-n // page)
    made = [tokens(kind, n, d, 10 * h + n, order) for h in range(hkv)]
    if kind == "either sign":
        made = [(k, v * 1e-38, q) for k, v, q in made]
    held = []
    for i in (0, 1):
        x = torch.zeros((pages * page, hkv, d))
        x[:n] = torch.stack([m[i] for m in made], 1)
        codes, scale = ref.quantised(x.view(pages, page, hkv, d).transpose(1, 2).contiguous())
        if kind == "either sign":
            scale *= torch.randint(0, 2, scale.shape, generator=torch.Generator().manual_seed(i)) * 2.0 - 1
        held.append((codes, scale))
    (k, ks), (v, vs) = held
    cache = c.KvCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda())
    q = torch.cat([m[2] for m in made])[None].to(dtype)
    got = c.attention_decode(q.cuda(), cache, torch.arange(pages, dtype=torch.int32)[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    k, v = ((x.double() * s.double()[..., None]).transpose(1, 2).flatten(0, 1)[:n] for x, s in held)
    for h in range(hkv):
        assert_near(q[0, 4 * h:4 * h + 4], k[:, h], v[:, h], got[0, 4 * h:4 * h + 4], dtype)
