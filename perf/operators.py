"""The attention operators' cases: what is measured of them, and their plain forms.

Four operators that stand between a decoder layer's q/k/v projections and its output projection: the rotation of q and k
with the write of k and v into a paged cache (16-bit, or int8 with a scale for each token and head), the read of cached
tokens back into packed tensors, the attention of whole prompts, and the attention of one new token over the cache.
With `own` false, `run` computes them with elementary torch operations in 32 bits; with `own` true it calls the package.

A cache is [pages, kv_heads, page_size, head_dim], its int8 scales f32 [pages, kv_heads, page_size].
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1}
MIN_AMAX = 2.0 ** -100  # rows of the int8 cache whose largest value is below this are held as zeros


def listed():
    llama8b, llama70b = {"hq": 32, "hkv": 8, "d": 128}, {"hq": 64, "hkv": 8, "d": 128}
    return [
        # --- prompts ---
        # a scheduler's small batch: nine short prompts of unlike lengths, one slot of them empty
        {"name": "prefill_short", "op": "prefill", **llama8b, "n": 9, "length": 200, "prefix": 0, "ragged": True,
         "causal": True, "dtype": "bf16"},
        # an ordinary prompt: 2048 tokens, the benchmark's prefill size
        {"name": "prefill_2048", "op": "prefill", **llama8b, "n": 1, "length": 2048, "prefix": 0, "ragged": False,
         "causal": True, "dtype": "bf16"},
        # a chunk of 512 tokens of three long prompts, whose earlier tokens were read back from the cache
        {"name": "prefill_chunk", "op": "prefill", **llama70b, "n": 3, "length": 512, "prefix": 7001, "ragged": True,
         "causal": True, "dtype": "f16"},
        # a long document in one piece: the largest call
        {"name": "prefill_16384", "op": "prefill", **llama8b, "n": 1, "length": 16384, "prefix": 0, "ragged": False,
         "causal": True, "dtype": "bf16"},
        # --- single tokens ---
        # one user's chat, a few hundred tokens in: latency is all
        {"name": "decode_1x333", "op": "decode", **llama8b, "n": 1, "length": 333, "ragged": False, "page": 16,
         "dtype": "bf16", "cache": "bf16"},
        # an ordinary serving batch with f32 activations over the int8 cache
        {"name": "decode_16x2048_int8", "op": "decode", **llama8b, "n": 16, "length": 2048, "ragged": True,
         "page": 64, "dtype": "f32", "cache": "int8"},
        # one very long context, heads of the larger model
        {"name": "decode_1x100001", "op": "decode", **llama70b, "n": 1, "length": 100001, "ragged": False,
         "page": 64, "dtype": "bf16", "cache": "int8"},
        # a full serving batch: the largest call
        {"name": "decode_128x4096", "op": "decode", **llama8b, "n": 128, "length": 4096, "ragged": True, "page": 64,
         "dtype": "bf16", "cache": "bf16"},
        # --- the cache ---
        # the new tokens of a decode step (f32 projections), written and read back
        {"name": "cache_step_16", "op": "write", **llama8b, "n": 16, "length": 1, "start": 777, "ragged": False,
         "page": 16, "dtype": "f32", "q_dtype": "f32", "cache": "int8", "rope": "half"},
        # a prompt of 2048 tokens into a 16-bit cache, with its queries
        {"name": "cache_write_2048", "op": "write", **llama8b, "n": 1, "length": 2048, "start": 0, "ragged": False,
         "page": 64, "dtype": "f32", "q_dtype": "bf16", "cache": "bf16", "rope": "pairs"},
        # a batch of prompts into the int8 cache, and back
        {"name": "cache_write_int8", "op": "write", **llama8b, "n": 7, "length": 2048, "start": 0, "ragged": True,
         "page": 48, "dtype": "f32", "q_dtype": "bf16", "cache": "int8", "rope": "half"},
        # the cached part of long prompts, read back for their next chunk
        {"name": "cache_read_int8", "op": "read", **llama70b, "n": 4, "length": 32768, "start": 0, "ragged": True,
         "page": 64, "cache": "int8", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "decode", "write", "read"])
    hq, hkv = rng.choice([(32, 8), (64, 8), (8, 8), (16, 1), (12, 4), (14, 2)])
    c = {"op": op, "hq": hq, "hkv": hkv, "d": rng.choice([128, 128, 64, 96]), "ragged": rng.random() < 0.7}
    if op == "prefill":
        n, length = _log(rng, 1, 16), _log(rng, 1, 8192)
        prefix = _log(rng, 1, 8192) if rng.random() < 0.4 else 0
        while n * length * (length + prefix) * hq * c["d"] > 16384 * 16384 * 32 * 64:  # the plain form fills n x length x keys
            n, length, prefix = max(1, n // 2), length - length // 4, prefix // 2
        c |= {"n": n, "length": length, "prefix": prefix, "causal": rng.random() < 0.8,
              "dtype": rng.choice(["bf16", "f16"])}
    else:
        c |= {"page": rng.choice([16, 32, 48, 64, 128]), "cache": rng.choice(["bf16", "f16", "int8"])}
        n, most = _log(rng, 1, 128), 131072 if op == "decode" else 16384
        length = _log(rng, 1, max(1, min(most, 400_000_000 // (n * hkv * c["d"]))))
        if op == "write":
            length = _log(rng, 1, max(1, min(4096, 40_000_000 // (n * (hq + 2 * hkv) * c["d"]))))
        c |= {"n": n, "length": length}
        if op == "decode":
            c |= {"dtype": rng.choice(["f32", "bf16", "f16"])}
        elif op == "write":
            c |= {"start": _log(rng, 1, 2048) if rng.random() < 0.5 else 0, "dtype": rng.choice(["f32", "bf16", "f16"]),
                  "q_dtype": rng.choice(["f32", "bf16", "f16"]), "rope": rng.choice(["half", "pairs", "none"])}
        else:
            c |= {"start": _log(rng, 1, 2048) if rng.random() < 0.3 else 0, "dtype": rng.choice(["bf16", "f16"])}
    return c


def lengths(case):
    """Each sequence's tokens: the longest first, the others spread down to a quarter of it, one of five or more empty."""
    n, length = case["n"], case["length"]
    if not case["ragged"]:
        return [length] * n
    part = [max(1, round(length * (1 - 0.75 * ((i * 0.6180339887) % 1)))) for i in range(n)]
    return part[:-1] + [0] if n >= 5 else part


def _cumulative(lens, dev):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(device=dev, dtype=torch.int32)


def _pages(case, ends, gen, dev):
    """A block table over shuffled pages for sequences of `ends` tokens; columns past a sequence's end hold -1."""
    page = case["page"]
    need = [-(-e // page) for e in ends]
    width, total = max(1, max(need)), sum(need) + 3
    order = torch.randperm(total, generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
    first = torch.tensor([0] + need, dtype=torch.int64).cumsum(0)[:-1].to(dev)[:, None]
    col = torch.arange(width, device=dev)[None, :]
    held = col < torch.tensor(need, device=dev)[:, None]
    table = torch.where(held, order[(first + col).clamp(max=total - 1)], -1)
    return table.to(torch.int32).contiguous(), total


def _values(shape, gen, dev, dtype, outliers=False):
    """Normal values; q and k have channels (one in sixteen) that are three times as large."""
    x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)
    if outliers:
        x[..., 5::16] *= 3.0
    return x.to(dtype)


def _quantised(x):
    """int8 codes and the f32 scale of each last-dimension row."""
    a = x.abs().amax(-1, keepdim=True)
    zero = a < MIN_AMAX
    code = torch.where(zero, torch.zeros_like(x), torch.round(x * (torch.full_like(a, 127.0) / a.masked_fill(zero, 1.0))))
    return code.to(torch.int8), torch.where(zero, torch.zeros_like(a), a / 127.0)[..., 0]


def _cache(case, pages, gen, dev):
    shape = (pages, case["hkv"], case["page"], case["d"])
    if case["cache"] != "int8":
        return {"k": _values(shape, gen, dev, DTYPES[case["cache"]], True), "v": _values(shape, gen, dev, DTYPES[case["cache"]]),
                "k_scale": None, "v_scale": None}
    k, ks = _quantised(_values(shape, gen, dev, torch.float32, True))
    v, vs = _quantised(_values(shape, gen, dev, torch.float32))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    hq, hkv, d, lens = case["hq"], case["hkv"], case["d"], lengths(case)
    s = {"case": dict(case), "lens": lens}
    if case["op"] == "prefill":
        dt = DTYPES[case["dtype"]]
        keys = [n + case["prefix"] if n else 0 for n in lens]
        s |= {"q": _values((sum(lens), hq, d), gen, dev, dt, True), "k": _values((sum(keys), hkv, d), gen, dev, dt, True),
              "v": _values((sum(keys), hkv, d), gen, dev, dt), "cu_q": _cumulative(lens, dev), "cu_k": _cumulative(keys, dev),
              "longest_q": max(lens), "longest_k": max(keys)}
        return s
    start = case.get("start", 0)
    table, pages = _pages(case, [start + n if n else 0 for n in lens], gen, dev)
    s |= _cache(case, pages, gen, dev) | {"table": table, "longest": max(lens)}
    if case["op"] == "decode":
        s |= {"q": _values((case["n"], hq, d), gen, dev, DTYPES[case["dtype"]], True),
              "seq_lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    else:
        total = sum(lens)
        seq = torch.repeat_interleave(torch.arange(case["n"]), torch.tensor(lens)).to(dev)
        s |= {"cu": _cumulative(lens, dev), "starts": torch.full((case["n"],), start, dtype=torch.int32, device=dev), "total": total}
        pos = torch.arange(total, device=dev) - s["cu"][seq].long() + start
        slots = table[seq, pos // case["page"]].long() * case["page"] + pos % case["page"]
        s |= {"positions": pos.to(torch.int32), "slots": slots.to(torch.int32)}
    if case["op"] == "write":
        dt = DTYPES[case["dtype"]]
        s |= {"q": _values((total, hq, d), gen, dev, dt, True), "new_k": _values((total, hkv, d), gen, dev, dt, True),
              "new_v": _values((total, hkv, d), gen, dev, dt), "cos": None, "sin": None}
        if case["rope"] != "none":
            angle = torch.arange(start + max(lens), device=dev, dtype=torch.float64)[:, None] * (
                500000.0 ** (-torch.arange(d // 2, device=dev, dtype=torch.float64) * 2 / d))[None, :]
            s |= {"cos": angle.cos().float().contiguous(), "sin": angle.sin().float().contiguous()}
    if own:
        import candelora_metal_kernels_b200 as c
        s["cache"] = c.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if case["op"] == "decode":
            s["workspace"] = torch.empty(c.attention_decode_workspace_bytes(s["q"], s["cache"], table), dtype=torch.uint8, device=dev)
    return s


# ---- the package's calls ----

def _run_own(s):
    import candelora_metal_kernels_b200 as c
    case = s["case"]
    if case["op"] == "prefill":
        return c.attention_prefill(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=case["causal"])
    if case["op"] == "decode":
        return c.attention_decode(s["q"], s["cache"], s["table"], s["seq_lens"], workspace=s["workspace"])
    if case["op"] == "read":
        return c.kv_cache_read(s["cache"], s["table"], s["cu"], s["total"], starts=s["starts"], dtype=DTYPES[case["dtype"]])
    q = c.kv_cache_write(s["cache"], s["new_k"], s["new_v"], s["slots"], q=s["q"], q_dtype=DTYPES[case["q_dtype"]],
                         positions=s["positions"], cos=s["cos"], sin=s["sin"], interleaved=case["rope"] == "pairs")
    if case["cache"] != "int8":
        return q, s["k"], s["v"]
    k, v = c.kv_cache_read(s["cache"], s["table"], s["cu"], s["total"], starts=s["starts"], dtype=torch.bfloat16)
    return q, k, v


# ---- the plain forms ----

def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v in 32 bits: q [b, h, g*r, d] (g heads of r rows), k, v [b, h, l, d], `seen` [b, r, l]."""
    b, h, rows, d = q.shape
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
    s = s.view(b, h, rows // seen.shape[1], seen.shape[1], -1)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, h, rows, -1), v).view(*s.shape[:-1], d)
    return o / total.masked_fill_(total == 0, 1.0)  # a row that sees nothing is zero


def _plain_prefill(s):
    case = s["case"]
    hq, hkv, d, n, rows, cols = case["hq"], case["hkv"], case["d"], case["n"], s["longest_q"], s["longest_k"]
    q0, k0 = s["cu_q"][:-1].long(), s["cu_k"][:-1].long()
    lq, lk = s["cu_q"][1:].long() - q0, s["cu_k"][1:].long() - k0
    i = torch.arange(rows, device=q0.device)
    j = torch.arange(cols, device=q0.device)
    at_q = torch.where(i < lq[:, None], q0[:, None] + i, 0)
    at_k = torch.where(j < lk[:, None], k0[:, None] + j, 0)
    q = s["q"][at_q].float().view(n, rows, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k, v = (s[x][at_k].float().transpose(1, 2) for x in "kv")
    seen = (j < lk[:, None])[:, None, :].expand(n, rows, cols)
    if case["causal"]:
        seen = seen & (j <= (i + (lk - lq)[:, None])[:, :, None])
    o = _attend(q, k, v, seen).permute(0, 3, 1, 2, 4).reshape(n, rows, hq, d)
    return o[i < lq[:, None]].to(DTYPES[case["dtype"]])


def _gathered(s, seq, pos):
    """K and V in 32 bits, [..., kv_heads, head_dim], of the tokens at `pos` of the sequences `seq`."""
    page = s["case"]["page"]
    at, off = s["table"][seq, pos // page].long(), pos % page
    k, v = s["k"][at, :, off].float(), s["v"][at, :, off].float()
    if s["k_scale"] is None:
        return k, v
    return k * s["k_scale"][at, :, off][..., None], v * s["v_scale"][at, :, off][..., None]


def _plain_decode(s):
    case = s["case"]
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    j = torch.arange(s["longest"], device=s["q"].device)
    seen = j < s["seq_lens"].long()[:, None]
    pos = torch.where(seen, j, 0)
    k, v = _gathered(s, torch.arange(n, device=pos.device)[:, None].expand_as(pos), pos)
    q = s["q"].float().view(n, hkv, hq // hkv, d)
    return _attend(q, k.transpose(1, 2), v.transpose(1, 2), seen[:, None, :]).reshape(n, hq, d).to(s["q"].dtype)


def _rotated(x, s):
    x = x.float()
    if s["cos"] is None:
        return x
    c, n = (s[t][s["positions"].long()][:, None, :] for t in ("cos", "sin"))
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if s["case"]["rope"] == "pairs" else (x[..., :half], x[..., half:])
    y = (a * c - b * n, b * c + a * n)
    return torch.stack(y, -1).reshape(x.shape) if s["case"]["rope"] == "pairs" else torch.cat(y, -1)


def _plain_read(s, dtype):
    pos = s["positions"].long()
    seq = torch.searchsorted(s["cu"][1:].long(), torch.arange(s["total"], device=pos.device), right=True)
    return tuple(x.to(dtype) for x in _gathered(s, seq, pos))


def _plain_write(s):
    case = s["case"]
    at, off = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    q, k, v = _rotated(s["q"], s).to(DTYPES[case["q_dtype"]]), _rotated(s["new_k"], s), s["new_v"].float()
    if case["cache"] != "int8":
        s["k"][at, :, off] = k.to(s["k"].dtype)
        s["v"][at, :, off] = v.to(s["v"].dtype)
        return q, s["k"], s["v"]
    s["k"][at, :, off], s["k_scale"][at, :, off] = _quantised(k)
    s["v"][at, :, off], s["v_scale"][at, :, off] = _quantised(v)
    return (q, *_plain_read(s, torch.bfloat16))


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "prefill":
        return _plain_prefill(state)
    if op == "decode":
        return _plain_decode(state)
    if op == "write":
        return _plain_write(state)
    return _plain_read(state, DTYPES[state["case"]["dtype"]])


# ---- what a pass cannot do without ----

def work(case):
    hq, hkv, d, lens = case["hq"], case["hkv"], case["d"], lengths(case)
    total = sum(lens)
    if case["op"] == "prefill":
        keys, pairs = sum(n + case["prefix"] for n in lens if n), 0
        for n in lens:
            pairs += n * case["prefix"] + (n * (n + 1) // 2 if case["causal"] else n * n)
        e = SIZES[case["dtype"]]
        return {"bytes": (2 * total * hq + 2 * keys * hkv) * d * e, "flops": 4 * d * hq * pairs}
    held = hkv * (d * SIZES[case["cache"]] + (4 if case["cache"] == "int8" else 0)) * 2  # a token's K and V in the cache
    if case["op"] == "decode":
        return {"bytes": total * held + 2 * case["n"] * hq * d * SIZES[case["dtype"]], "flops": 4 * d * hq * total}
    if case["op"] == "read":
        return {"bytes": total * (held + 2 * hkv * d * SIZES[case["dtype"]]), "flops": 2 * total * hkv * d}
    bytes_ = total * ((hq + 2 * hkv) * d * SIZES[case["dtype"]] + hq * d * SIZES[case["q_dtype"]] + held + 8)
    bytes_ += (case["start"] + case["length"]) * d * 4 if case["rope"] != "none" else 0
    bytes_ += total * (held + 2 * hkv * d * 2) if case["cache"] == "int8" else 0  # the read back, in bf16
    return {"bytes": bytes_, "flops": 6 * total * (hq + hkv) * d}


# ---- the definitions in 64 bits, one sequence and one head at a time ----

def _exact_rows(q, k, v, shown):
    """Each row of q [r, d] over the first shown[r] of k, v [l, d], in pieces that fit."""
    def piece(part, limit):
        p = part @ k.T / math.sqrt(q.shape[1])
        hidden = torch.arange(k.shape[0], device=q.device)[None, :] >= limit[:, None]
        return torch.softmax(p.masked_fill(hidden, -1e300), -1).masked_fill(hidden, 0.0) @ v
    return torch.cat([piece(*x) for x in zip(q.split(4096), shown.split(4096))])


def _exact_cached(s, b, count, start=0):
    """K and V of `count` tokens of sequence b in 64 bits, [tokens, kv_heads, head_dim]."""
    page = s["case"]["page"]
    pages = s["table"][b, start // page:-(-(start + count) // page)].long()
    got = []
    for name in "kv":
        x = s[name][pages].double()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
        x = x.permute(0, 2, 1, 3).reshape(-1, *x.shape[1::2])
        got.append(x[start % page:start % page + count])
    return got


def _exact_turned(x, s):
    x = x.double()
    if s["cos"] is None:
        return x
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None, :]
    if s["case"]["rope"] == "pairs":
        z = torch.view_as_complex(x.view(*x.shape[:-1], -1, 2).contiguous()) * turn
        return torch.view_as_real(z).flatten(-2)
    first, second = x.chunk(2, -1)
    z = torch.complex(first.contiguous(), second.contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)


def _exact_int8(x):
    step = x.abs().amax(-1, keepdim=True) / 127
    return torch.round(x / step.clamp(min=1e-300)) * step


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d, lens, group = case["hq"], case["hkv"], case["d"], s["lens"], case["hq"] // case["hkv"]
    if case["op"] == "prefill":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        q0 = k0 = 0
        for n in lens:
            keys = n + case["prefix"] if n else 0
            rows = torch.arange(n, device=out.device)
            shown = rows + 1 + case["prefix"] if case["causal"] else torch.full_like(rows, keys)
            for h in range(hq):
                k, v = (s[x][k0:k0 + keys, h // group].double() for x in "kv")
                out[q0:q0 + n, h] = _exact_rows(s["q"][q0:q0 + n, h].double(), k, v, shown)
            q0, k0 = q0 + n, k0 + keys
        return out
    if case["op"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        for b, n in enumerate(lens):
            if n:
                k, v = _exact_cached(s, b, n)
                for h in range(hkv):
                    part = s["q"][b, h * group:(h + 1) * group].double()
                    out[b, h * group:(h + 1) * group] = _exact_rows(part, k[:, h], v[:, h], torch.full((group,), n, device=out.device))
        return out
    if case["op"] == "read":
        parts = [_exact_cached(s, b, n, case["start"]) for b, n in enumerate(lens) if n]
        return tuple(torch.cat(x) for x in zip(*parts))
    q, k, v = _exact_turned(s["q"], s), _exact_turned(s["new_k"], s), s["new_v"].double()
    if case["cache"] == "int8":
        return q, _exact_int8(k), _exact_int8(v)
    slots = s["slots"].long()
    caches = []
    for old, new in ((s["k"], k), (s["v"], v)):
        flat = old.double().transpose(1, 2).reshape(-1, hkv, d)
        flat[slots] = new
        caches.append(flat.view(old.shape[0], case["page"], hkv, d).transpose(1, 2).contiguous())
    return q, *caches
