"""The definitions of the 4-bit cache, the head norms and the pages' step, on the CPU: row by row and token by token."""
import math

import torch

import attention_reference as ref

E4M3 = torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)  # the numbers of the type from 0 to 448, in the order of their bits


def nearest_e4m3(x):
    """The bits of the e4m3 number nearest to x >= 0 (64 bits), ties to the even bits."""
    above = torch.bucketize(x, E4M3).clamp(max=126)  # the first number >= x
    below = (above - 1).clamp(min=0)
    up, down = E4M3[above] - x, x - E4M3[below]
    pick_above = (up < down) | ((up == down) & (above % 2 == 0))
    return torch.where(pick_above, above, below)


def quantised4(x):
    """(bytes, e4m3 bits [..., 4], f32 row scales) of the rows of x [..., d], in 64 bits."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    rows = torch.where(finite[..., None], x, torch.zeros_like(x))
    most = rows.unflatten(-1, (-1, 32)).abs().amax(-1)
    top = most.amax(-1)
    some = top >= 2.0 ** -100
    # the power of two with 224 < top / 7s <= 448
    exponent = torch.tensor([math.ceil(math.log2(v / 3136)) if v > 0 else 0 for v in top.flatten().tolist()]).view(top.shape)
    scale = torch.where(some, torch.ldexp(torch.ones_like(top), exponent), torch.zeros_like(top))
    assert ((top[some] <= 3136 * scale[some]) & (top[some] > 1568 * scale[some])).all()
    bits = torch.where(some[..., None], nearest_e4m3(most / 7 / torch.where(some, scale, torch.ones_like(scale))[..., None]), 0)
    step = scale[..., None] * E4M3[bits]
    quotient = rows.unflatten(-1, (-1, 32)) / torch.where(step > 0, step, torch.full_like(step, math.inf))[..., None]
    code = (torch.round(quotient).clamp(-7, 7) + 8).flatten(-2).to(torch.uint8)
    groups = torch.zeros((*x.shape[:-1], 4), dtype=torch.uint8)
    groups[..., :bits.shape[-1]] = bits.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), groups, torch.where(finite, scale, torch.full_like(scale, math.nan)).float()


def values4(codes, groups, scale):
    """What they stand for, in 64 bits."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
    g = E4M3[(groups[..., :code.shape[-1] // 32].long() & 127).clamp(max=126)]
    return (code.unflatten(-1, (-1, 32)) * g[..., None]).flatten(-2) * scale.double()[..., None]


def held4(cache):
    """K and V of a 4-bit KvCache in 64 bits, [pages, heads, page, d]."""
    return [values4(c.cpu(), g.cpu().view(torch.uint8), s.cpu()) for c, g, s in
            ((cache.k, cache.k_group, cache.k_scale), (cache.v, cache.v_group, cache.v_scale))]


def decode4(q, cache, table, lens, scale=None):
    """As attention_reference.decode, over a 4-bit cache."""
    q, table = q.detach().double().cpu(), table.cpu()
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    group, held = q.shape[1] // cache.kv_heads, held4(cache)
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(lens):
        if n > 0:
            at = torch.arange(n)
            k, v = (x[table[b, at // cache.page_size].long(), :, at % cache.page_size] for x in held)
            for h in range(q.shape[1]):
                o, s = ref.attend(q[b, h:h + 1], k[:, h // group], v[:, h // group], [n], scale)
                out[b, h], size[b, h] = o[0], s[0]
    return out, size


def normed(x, weight, eps):
    """The norm with its roundings: the reciprocal root and both products in f32."""
    x = x.float()
    r = (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)).float()
    return x * r * weight


def pages_step(state, page, new, total, keep=None):
    """One step of {table, lens, free, count} (lists, changed in place); returns slots, positions, cu_q, cu_k, granted."""
    table, lens, free = state["table"], state["lens"], state["free"]
    n, width, pages = len(lens), len(table[0]), len(free)
    most = min(width * page, 2 ** 31 - 1)

    def up(x):
        return -(-x // page)

    held = [min(max(x, 0), most) for x in lens]
    kept = [x if keep is None else min(x, max(k, 0)) for x, k in zip(held, keep or held)]
    new = [max(x, 0) for x in new]
    for b in range(n):
        for col in range(up(kept[b]), up(held[b])):
            free[state["count"]] = table[b][col]
            state["count"] += 1
    slots, positions, cu_q, cu_k, granted = [-1] * total, [0] * total, [0], [0], []
    row, asked, top = 0, 0, state["count"]
    for b in range(n):
        need = up(kept[b] + new[b]) - up(kept[b])
        fits = row + new[b] <= total and kept[b] + new[b] <= most
        asked += need if fits else 0
        if fits and (need == 0 or asked <= top):
            for col in range(up(kept[b]), up(kept[b] + new[b])):
                state["count"] -= 1
                table[b][col] = free[state["count"]]
            for i in range(new[b]):
                at = kept[b] + i
                number = table[b][at // page]
                slots[row + i] = number * page + at % page if 0 <= number < pages else -1
                positions[row + i] = at
            granted.append(new[b])
        else:
            granted.append(0)
        lens[b] = kept[b] + granted[b]
        row += new[b]
        cu_q.append(min(row, total))
        cu_k.append(min(sum(lens[:b + 1]), 2 ** 31 - 1))
    return slots, positions, cu_q, cu_k, granted
