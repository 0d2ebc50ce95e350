"""The attention operators' definitions in 64 bits, on the CPU, one head and one sequence at a time: only what a row sees
enters its sums, so that masked values cannot matter."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a unit in the last place


def attend(q, k, v, shown, scale):
    """q [r, d] over the first shown[r] of k, v [l, d]: (output, sum of p |v|), zeros where shown[r] <= 0."""
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for r in range(q.shape[0]):
        n = int(shown[r])
        if n > 0:
            p = torch.softmax(k[:n] @ q[r] * scale, 0)
            out[r], size[r] = p @ v[:n], p @ v[:n].abs()
    return out, size


def prefill(q, k, v, cu_q, cu_k, causal=True, scale=None):
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        lq, lk = q1 - q0, k1 - k0
        shown = [min(lk, i + 1 + lk - lq) if causal else lk for i in range(lq)]
        for h in range(q.shape[1]):
            out[q0:q1, h], size[q0:q1, h] = attend(q[q0:q1, h], k[k0:k1, h // group], v[k0:k1, h // group], shown, scale)
    return out, size


def cached(cache, table_row, positions):
    """K and V [tokens, kv_heads, d] of one sequence's positions, in 64 bits."""
    got = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = x.detach().cpu().double()
        if s is not None:
            x = x * s.detach().cpu().double()[..., None]
        rows = [x[int(table_row[p // cache.page_size]), :, p % cache.page_size] for p in positions]
        got.append(torch.stack(rows) if rows else x.new_zeros((0, x.shape[1], x.shape[3])))
    return got


def decode(q, cache, table, lens, scale=None):
    q, table = q.detach().double().cpu(), table.cpu()
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // cache.kv_heads
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(lens):
        if n > 0:
            k, v = cached(cache, table[b], range(n))
            for h in range(q.shape[1]):
                o, s = attend(q[b, h:h + 1], k[:, h // group], v[:, h // group], [n], scale)
                out[b, h], size[b, h] = o[0], s[0]
    return out, size


def rotated(x, positions, cos, sin, interleaved):
    """The rotation in x's type, each product and sum rounded by itself."""
    c, s = cos[positions.long()][:, None, :].to(x.dtype), sin[positions.long()][:, None, :].to(x.dtype)
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y = (a * c - b * s, b * c + a * s)
    return torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)


def quantised(x):
    """int8 codes and scale of each row of x, in x's type."""
    a = x.abs().amax(-1)
    bad, zero = ~torch.isfinite(a), a < 2.0 ** -100
    inv = torch.where(zero | bad, torch.zeros_like(a), torch.full_like(a, 127.0) / a)
    codes = torch.where(bad[..., None], torch.zeros_like(x), torch.round(x * inv[..., None]))
    scale = torch.where(zero, torch.zeros_like(a), a / 127.0)
    return codes.to(torch.int8), torch.where(bad, torch.full_like(a, math.nan), scale)
