"""The cases of a serving step's further operators, and their plain forms.

What a step does around the attention: the pages of the sequences (`kv_pages_step`: pages taken and given back, the slots,
positions and offsets of the new tokens), the norms of queries and keys for each head in the pass that rotates them and
writes the cache, and a cache held in 4 bits (written, read back, and attended to by one new token a sequence).
With `own` false, `run` computes them with elementary torch operations in 32 bits (sums of squares in 64, since 4-bit codes
lie next to borders); with `own` true it calls the package.

A 16-bit cache is [pages, kv_heads, page_size, head_dim]. A 4-bit one has bytes [..., head_dim / 2] (element 2i in the low
half of byte i, code + 8), e4m3 scales [..., 4] for the groups of 32 elements and f32 scales [...] for the rows: an element
is code x group's scale x row's scale.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
MIN_AMAX = 2.0 ** -100  # rows of the 4-bit cache whose largest value is below this are held as zeros
EPS = 1e-6


def listed():
    llama8b, llama70b = {"hq": 32, "hkv": 8, "d": 128}, {"hq": 64, "hkv": 8, "d": 128}
    return [
        # --- norms, rotation and cache write ---
        # the new tokens of a decode step, f32 projections, into the 4-bit cache and back
        {"name": "norm_step_16", "op": "write", **llama8b, "n": 16, "length": 1, "start": 777, "ragged": False, "page": 16,
         "dtype": "f32", "q_dtype": "f32", "cache": "int4", "rope": "half", "norm": "shared"},
        # a prompt of 2048 tokens, the benchmark's prefill size, into a 16-bit cache
        {"name": "norm_write_2048", "op": "write", **llama8b, "n": 1, "length": 2048, "start": 0, "ragged": False, "page": 64,
         "dtype": "f32", "q_dtype": "bf16", "cache": "bf16", "rope": "half", "norm": "shared"},
        # a batch of prompts into the 4-bit cache and back, a weight row for each head
        {"name": "norm_write_int4", "op": "write", **llama8b, "n": 7, "length": 2048, "start": 0, "ragged": True, "page": 48,
         "dtype": "bf16", "q_dtype": "bf16", "cache": "int4", "rope": "pairs", "norm": "heads"},
        # --- the 4-bit cache read back ---
        # the earlier tokens of three prompts for their next chunk, from the middle of a page
        {"name": "read_int4_700", "op": "read", **llama8b, "n": 3, "length": 700, "start": 129, "ragged": True, "page": 16,
         "cache": "int4", "dtype": "f16"},
        # the cached part of long prompts
        {"name": "read_int4_32768", "op": "read", **llama70b, "n": 4, "length": 32768, "start": 0, "ragged": True, "page": 64,
         "cache": "int4", "dtype": "bf16"},
        # --- single tokens over the 4-bit cache ---
        # one user's chat, a few hundred tokens in: latency is all
        {"name": "decode_int4_1x333", "op": "decode", **llama8b, "n": 1, "length": 333, "ragged": False, "page": 16,
         "dtype": "bf16", "cache": "int4"},
        # an ordinary serving batch with f32 activations
        {"name": "decode_int4_16x2048", "op": "decode", **llama8b, "n": 16, "length": 2048, "ragged": True, "page": 64,
         "dtype": "f32", "cache": "int4"},
        # one very long context, heads of the larger model
        {"name": "decode_int4_1x100001", "op": "decode", **llama70b, "n": 1, "length": 100001, "ragged": False, "page": 64,
         "dtype": "bf16", "cache": "int4"},
        # a full serving batch: the largest call
        {"name": "decode_int4_128x4096", "op": "decode", **llama8b, "n": 128, "length": 4096, "ragged": True, "page": 64,
         "dtype": "bf16", "cache": "int4"},
        # --- the pages of a step ---
        # a step that verifies four drafted tokens and one more of 64 sequences, after the last step's were cut back
        {"name": "pages_64x5", "op": "pages", "n": 64, "length": 5, "start": 2048, "ragged": False, "page": 16, "finished": 8,
         "free": "enough"},
        # an ordinary decode step of a large batch
        {"name": "pages_512x1", "op": "pages", "n": 512, "length": 1, "start": 1024, "ragged": False, "page": 64, "finished": 32,
         "free": "enough"},
        # prompts that come in for many finished sequences, more than the pool has pages for
        {"name": "pages_prompts", "op": "pages", "n": 96, "length": 2048, "start": 4096, "ragged": True, "page": 16,
         "finished": 2, "free": "short"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "decode", "decode", "pages"])
    c = {"op": op, "ragged": rng.random() < 0.7}
    if op == "pages":
        n = _log(rng, 1, 2048)
        c |= {"n": n, "length": _log(rng, 1, max(1, min(8192, 131072 // n))), "page": rng.choice([1, 16, 16, 32, 48, 64, 128]),
              "start": _log(rng, 1, max(1, min(65536, 1_000_000 // n))), "finished": rng.choice([0, 1, 2, 5, 32]),
              "free": rng.choice(["enough", "enough", "short"])}
        return c
    hq, hkv = rng.choice([(32, 8), (64, 8), (8, 8), (16, 1), (12, 4), (14, 2)])
    c |= {"hq": hq, "hkv": hkv, "d": rng.choice([128, 128, 64, 96, 32]), "page": rng.choice([16, 32, 48, 64, 128]), "cache": "int4"}
    n, most = _log(rng, 1, 128), 131072 if op == "decode" else 16384
    length = _log(rng, 1, max(1, min(most, 400_000_000 // (n * hkv * c["d"]))))
    if op == "write":
        length = _log(rng, 1, max(1, min(4096, 40_000_000 // (n * (hq + 2 * hkv) * c["d"]))))
    c |= {"n": n, "length": length}
    if op == "decode":
        c |= {"dtype": rng.choice(["f32", "bf16", "f16"])}
    elif op == "read":
        c |= {"start": _log(rng, 1, 2048) if rng.random() < 0.3 else 0, "dtype": rng.choice(["bf16", "f16", "f32"])}
    else:
        # (a 16-bit cache goes with norms: without them its write is an operator that was there before)
        cache = rng.choice(["int4", "int4", "bf16", "f16"])
        c |= {"start": _log(rng, 1, 2048) if rng.random() < 0.5 else 0, "dtype": rng.choice(["f32", "bf16", "f16"]),
              "q_dtype": rng.choice(["f32", "bf16", "f16"]), "rope": rng.choice(["half", "pairs", "none"]), "cache": cache,
              "norm": rng.choice(["shared", "shared", "heads"] + (["none"] if cache == "int4" else []))}
    return c


def lengths(case):
    """Each sequence's tokens: the longest first, the others spread down to a quarter of it, one of five or more empty."""
    n, length = case["n"], case["length"]
    if not case["ragged"]:
        return [length] * n
    part = [max(1, round(length * (1 - 0.75 * ((i * 0.6180339887) % 1)))) for i in range(n)]
    return part[:-1] + [0] if n >= 5 else part


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _cumulative(lens, dev):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(device=dev, dtype=torch.int32)


def _pages(page, ends, spare, gen, dev):
    """A block table over shuffled pages for sequences of `ends` tokens (columns past a sequence's end hold -1), the order
    of all pages and how many of them the sequences have."""
    need = [-(-e // page) for e in ends]
    width, held = max(1, max(need)), sum(need)
    order = torch.randperm(held + spare, generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
    first = torch.tensor([0] + need, dtype=torch.int64).cumsum(0)[:-1].to(dev)[:, None]
    col = torch.arange(width, device=dev)[None, :]
    mine = col < torch.tensor(need, device=dev)[:, None]
    table = torch.where(mine, order[(first + col).clamp(max=held + spare - 1)], -1)
    return table.to(torch.int32).contiguous(), order, held


def _values(shape, gen, dev, dtype, outliers=False):
    """Normal values; q and k have channels (one in sixteen) that are three times as large."""
    x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)
    if outliers:
        x[..., 5::16] *= 3.0
    return x.to(dtype)


def _weights(case, heads, gen, dev):
    """The norm weights of a trained layer: about 1, of [head_dim] or [heads, head_dim]."""
    shape = (heads, case["d"]) if case["norm"] == "heads" else (case["d"],)
    return 1.0 + 0.3 * torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)


def _quantised(x):
    """The bytes, group scales (the e4m3 numbers' bits) and row scales (powers of two) of rows x [..., d] in 32 bits. Quotients
    are taken in 64: codes and group scales lie next to borders."""
    groups = x.unflatten(-1, (-1, 32))
    most = groups.abs().amax(-1)
    top = most.amax(-1, keepdim=True)
    zero = top < MIN_AMAX
    # the power of two s with 224 < top / 7s <= 448, the largest e4m3
    part, exponent = torch.frexp(top.masked_fill(zero, 1.0))
    scale = ((exponent - 12 + (part > 0.765625) + 127) << 23).to(torch.int32).view(torch.float32).masked_fill(zero, 0.0)
    g = (most.double() / (7.0 * scale.double().masked_fill(zero, 1.0))).masked_fill(zero, 0.0).float().to(torch.float8_e4m3fn)
    step = scale.double() * g.double()
    code = torch.round(groups.double() / step.masked_fill(step == 0, math.inf)[..., None]).clamp(-7, 7) + 8
    code = code.flatten(-2).to(torch.uint8)
    held = torch.zeros((*x.shape[:-1], 4), dtype=torch.uint8, device=x.device)
    held[..., :g.shape[-1]] = g.view(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), held, scale[..., 0]


def _valued(codes, groups, scale):
    """What rows of the 4-bit cache stand for, in 32 bits."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    g = groups.view(torch.float8_e4m3fn).float()[..., :code.shape[-1] // 32]
    return (code.unflatten(-1, (-1, 32)) * g[..., None]).flatten(-2) * scale[..., None]


def _cache(case, pages, gen, dev):
    shape = (pages, case["hkv"], case["page"], case["d"])
    if case["cache"] != "int4":
        return {"k": _values(shape, gen, dev, DTYPES[case["cache"]], True), "v": _values(shape, gen, dev, DTYPES[case["cache"]]),
                "k_scale": None, "v_scale": None, "k_group": None, "v_group": None}
    k, kg, ks = _quantised(_values(shape, gen, dev, torch.float32, True))
    v, vg, vs = _quantised(_values(shape, gen, dev, torch.float32))
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "k_group": kg, "v_group": vg}


def _prepare_pages(case, gen, dev):
    n, start, lens, page = case["n"], case["start"], lengths(case), case["page"]
    # every sequence has last step's tokens, of which `keep` are kept; one in `finished` has ended and a new one takes its place
    before = [start - (i * 7) % min(start, 97) for i in range(n)]
    ended = [case["finished"] > 0 and i % case["finished"] == 0 for i in range(n)]
    keep = [0 if e else b for e, b in zip(ended, before)]
    # (where pages are to run short, the ones that have ended were half as long as those that follow)
    held = [(b if case["free"] == "enough" else new // 2) if e else b + new for e, b, new in zip(ended, before, lens)]
    want = [k + new for k, new in zip(keep, lens)]
    takes = sum(-(-w // page) + (-(-h // page)) for w, h in zip(want, held))
    table, order, used = _pages(page, held, 3 + (takes if case["free"] == "enough" else takes // 64), gen, dev)
    width = max(table.shape[1], max(-(-w // page) for w in want))
    table = torch.nn.functional.pad(table, (0, width - table.shape[1]), value=-1).contiguous()
    free = torch.full_like(order, -1)
    free[:order.shape[0] - used] = order[used:]
    total = sum(lens)
    return {"case": dict(case), "lens": lens, "total": total, "table": table, "held": _i32(held, dev), "free": free,
            "count": _i32([order.shape[0] - used], dev), "keep": _i32(keep, dev), "new": _i32(lens, dev)}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    if case["op"] == "pages":
        s = _prepare_pages(case, gen, dev)
        if own:
            import candelora_metal_kernels_b200 as c
            s["pages"] = c.KvPages(s["table"], s["held"], s["free"], s["count"], case["page"])
            s["step"] = c.KvStep.empty(s["pages"], s["total"])
        return s
    hq, hkv, d, lens, start = case["hq"], case["hkv"], case["d"], lengths(case), case.get("start", 0)
    s = {"case": dict(case), "lens": lens}
    table, order, _ = _pages(case["page"], [start + n if n else 0 for n in lens], 3, gen, dev)
    s |= _cache(case, order.shape[0], gen, dev) | {"table": table, "longest": max(lens)}
    if case["op"] == "decode":
        s |= {"q": _values((case["n"], hq, d), gen, dev, DTYPES[case["dtype"]], True), "seq_lens": _i32(lens, dev)}
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
              "new_v": _values((total, hkv, d), gen, dev, dt), "cos": None, "sin": None, "q_norm": None, "k_norm": None}
        if case["rope"] != "none":
            angle = torch.arange(start + max(lens), device=dev, dtype=torch.float64)[:, None] * (
                500000.0 ** (-torch.arange(d // 2, device=dev, dtype=torch.float64) * 2 / d))[None, :]
            s |= {"cos": angle.cos().float().contiguous(), "sin": angle.sin().float().contiguous()}
        if case["norm"] != "none":
            s |= {"q_norm": _weights(case, hq, gen, dev), "k_norm": _weights(case, hkv, gen, dev)}
    if own:
        import candelora_metal_kernels_b200 as c
        groups = [None if s[x] is None else s[x].view(torch.float8_e4m3fn) for x in ("k_group", "v_group")]
        s["cache"] = c.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"], *groups)
        if case["op"] == "decode":
            s["workspace"] = torch.empty(c.attention_decode_workspace_bytes(s["q"], s["cache"], table), dtype=torch.uint8, device=dev)
    return s


# ---- the package's calls ----

def _run_own(s):
    import candelora_metal_kernels_b200 as c
    case = s["case"]
    if case["op"] == "pages":
        t = c.kv_pages_step(s["pages"], s["new"], s["total"], keep=s["keep"], out=s["step"])
        return (t.slots, t.positions, t.cu_seqlens_q, t.cu_seqlens_k, t.granted, s["table"], s["held"], s["free"], s["count"])
    if case["op"] == "decode":
        return c.attention_decode(s["q"], s["cache"], s["table"], s["seq_lens"], workspace=s["workspace"])
    if case["op"] == "read":
        return c.kv_cache_read(s["cache"], s["table"], s["cu"], s["total"], starts=s["starts"], dtype=DTYPES[case["dtype"]])
    q = c.kv_cache_write(s["cache"], s["new_k"], s["new_v"], s["slots"], q=s["q"], q_dtype=DTYPES[case["q_dtype"]],
                         positions=s["positions"], cos=s["cos"], sin=s["sin"], interleaved=case["rope"] == "pairs",
                         q_norm=s["q_norm"], k_norm=s["k_norm"], norm_eps=EPS)
    if case["cache"] != "int4":
        return q, s["k"], s["v"]
    k, v = c.kv_cache_read(s["cache"], s["table"], s["cu"], s["total"], starts=s["starts"], dtype=torch.bfloat16)
    return q, k, v


# ---- the plain forms ----

def _plain_pages(s):
    page, total, table = s["case"]["page"], s["total"], s["table"]
    (n, width), room = table.shape, s["free"].shape[0]
    i64 = {"dtype": torch.int64, "device": table.device}

    def before(x):  # the sum of the sequences before, and of all
        return torch.cat([torch.zeros(1, **i64), x.cumsum(0)])

    def pages_of(x):
        return (x + page - 1) // page

    held, new = s["held"].long(), s["new"].long().clamp(min=0)
    kept = torch.minimum(held, s["keep"].long().clamp(min=0))
    row0 = before(new)
    # the pages that are given back, onto the free ones in the order of sequences and columns
    col = torch.arange(width, **i64)[None, :]
    back = (col >= pages_of(kept)[:, None]) & (col < pages_of(held)[:, None])
    count = s["count"].long()
    at = torch.where(back, count + back.flatten().cumsum(0).view(n, width) - 1, room)
    free = torch.cat([s["free"], s["free"].new_zeros(1)]).scatter_(0, at.flatten(), table.flatten())[:room]
    top = count + back.sum()
    # the pages that are asked for, as far as there are any
    fits = (row0[1:] <= total) & (kept + new <= width * page)
    need = torch.where(fits, pages_of(kept + new) - pages_of(kept), 0)
    need0 = before(need)
    granted = torch.where(fits & ((need0[1:] <= top) | (need == 0)), new, 0)
    grown = kept + granted
    fresh = (col >= pages_of(kept)[:, None]) & (col < pages_of(grown)[:, None])
    pick = (top - 1 - need0[:-1, None] - (col - pages_of(kept)[:, None])).clamp(0, room - 1)
    table = torch.where(fresh, free[pick], table)
    # where the new tokens go
    t = torch.arange(total, **i64)
    seq = torch.searchsorted(row0[1:].contiguous(), t, right=True).clamp(max=n - 1)
    live = (t < row0[-1]) & (granted[seq] > 0)
    pos = torch.where(live, kept[seq] + t - row0[seq], 0)
    slots = torch.where(live, table[seq, (pos // page).clamp(max=width - 1)].long() * page + pos % page, -1)
    s["table"].copy_(table), s["held"].copy_(grown), s["free"].copy_(free), s["count"].copy_(top - torch.where(granted > 0, need, 0).sum())
    out = (slots, pos, row0.clamp(max=total), before(grown), granted)
    return (*(x.to(torch.int32) for x in out), s["table"], s["held"], s["free"], s["count"])


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v in 32 bits: q [b, h, g, d], k, v [b, h, l, d], `seen` [b, l]."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(q.shape[-1]))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    return torch.matmul(s, v) / total.masked_fill_(total == 0, 1.0)  # a row that sees nothing is zero


def _gathered(s, seq, pos):
    """K and V in 32 bits, [..., kv_heads, head_dim], of the tokens at `pos` of the sequences `seq`."""
    page = s["case"]["page"]
    at, off = s["table"][seq, pos // page].long(), pos % page
    return tuple(_valued(s[x][at, :, off], s[x + "_group"][at, :, off], s[x + "_scale"][at, :, off]) for x in "kv")


def _plain_decode(s):
    case = s["case"]
    n, hq, hkv, d = case["n"], case["hq"], case["hkv"], case["d"]
    j = torch.arange(s["longest"], device=s["q"].device)
    seen = j < s["seq_lens"].long()[:, None]
    pos = torch.where(seen, j, 0)
    k, v = _gathered(s, torch.arange(n, device=pos.device)[:, None].expand_as(pos), pos)
    q = s["q"].float().view(n, hkv, hq // hkv, d)
    return _attend(q, k.transpose(1, 2), v.transpose(1, 2), seen).reshape(n, hq, d).to(s["q"].dtype)


def _normed(x, weight):
    x = x.float()
    if weight is None:
        return x
    r = torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS).reciprocal().float()
    return x * r * weight


def _rotated(x, s):
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
    q = _rotated(_normed(s["q"], s["q_norm"]), s).to(DTYPES[case["q_dtype"]])
    k, v = _rotated(_normed(s["new_k"], s["k_norm"]), s), s["new_v"].float()
    if case["cache"] != "int4":
        s["k"][at, :, off] = k.to(s["k"].dtype)
        s["v"][at, :, off] = v.to(s["v"].dtype)
        return q, s["k"], s["v"]
    s["k"][at, :, off], s["k_group"][at, :, off], s["k_scale"][at, :, off] = _quantised(k)
    s["v"][at, :, off], s["v_group"][at, :, off], s["v_scale"][at, :, off] = _quantised(v)
    return (q, *_plain_read(s, torch.bfloat16))


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "pages":
        return _plain_pages(state)
    if op == "decode":
        return _plain_decode(state)
    if op == "write":
        return _plain_write(state)
    return _plain_read(state, DTYPES[state["case"]["dtype"]])


# ---- what a pass cannot do without ----

def work(case):
    lens = lengths(case)
    total = sum(lens)
    if case["op"] == "pages":
        n, page = case["n"], case["page"]
        # lengths in (held, kept, new), out (held, granted, two offsets); a slot and a position a row; a number read and one
        # written for each page that is taken or given back
        return {"bytes": 28 * n + 8 * total + 16 * sum(-(-x // page) for x in lens), "flops": 8 * total}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    held = 2 * hkv * (d // 2 + d // 32 + 4 if case["cache"] == "int4" else d * 2)  # a token's K and V in the cache
    if case["op"] == "decode":
        return {"bytes": total * held + 2 * case["n"] * hq * d * SIZES[case["dtype"]], "flops": 4 * d * hq * total}
    if case["op"] == "read":
        return {"bytes": total * (held + 2 * hkv * d * SIZES[case["dtype"]]), "flops": 4 * total * hkv * d}
    bytes_ = total * ((hq + 2 * hkv) * d * SIZES[case["dtype"]] + hq * d * SIZES[case["q_dtype"]] + held + 8)
    bytes_ += (case["start"] + case["length"]) * d * 4 if case["rope"] != "none" else 0
    bytes_ += total * (held + 2 * hkv * d * 2) if case["cache"] == "int4" else 0  # the read back, in bf16
    return {"bytes": bytes_, "flops": 10 * total * (hq + hkv) * d}


# ---- the definitions in 64 bits ----

def _exact_cached(s, b, count, start=0):
    """K and V of `count` tokens of sequence b in 64 bits, [tokens, kv_heads, head_dim]."""
    page, d = s["case"]["page"], s["case"]["d"]
    pages = s["table"][b, start // page:-(-(start + count) // page)].long()
    levels = torch.arange(-8, 8, dtype=torch.float64, device=pages.device)
    # e4m3 without its sign: the exponent above three bits of the fraction, subnormals at exponent 0
    bits = torch.arange(128, device=pages.device)
    e4m3 = torch.where(bits < 8, bits * 2.0 ** -9, (8 + bits % 8) * 2.0 ** (bits // 8 - 10).double())
    got = []
    for name in "kv":
        x = s[name][pages].long()
        value = torch.empty((*x.shape[:-1], d), dtype=torch.float64, device=x.device)
        value[..., 0::2], value[..., 1::2] = levels[x % 16], levels[x // 16]
        value *= e4m3[s[name + "_group"][pages][..., :d // 32].long()].repeat_interleave(32, -1)
        value *= s[name + "_scale"][pages].double().unsqueeze(-1)
        value = value.permute(0, 2, 1, 3).reshape(-1, *value.shape[1::2])
        got.append(value[start % page:start % page + count])
    return got


def _exact_int4(x):
    """What 4 bits keep of rows x: steps of a row's power of two times a number of four significant bits (a multiple of 2^-9)."""
    power = torch.tensor([2.0 ** i for i in range(-200, 200)], dtype=torch.float64, device=x.device)
    groups = x.unflatten(-1, (-1, 32))
    most = groups.abs().amax(-1, keepdim=True)
    top = most.amax(-2, keepdim=True).clamp(min=1e-30) / 3136
    part, exponent = torch.frexp(top)
    row = power[exponent + 199 + (part > 0.5)]  # the power of two at or above
    ratio = most / 7 / row
    unit = power[(torch.frexp(ratio).exponent - 4).clamp(min=-9) + 200]
    step = torch.round(ratio / unit) * unit * row
    return (torch.round(groups / step.clamp(min=1e-300)).clamp(-7, 7) * step).flatten(-2)


def _exact_turned(x, weight, s):
    x = x.double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    if s["cos"] is None:
        return x
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None, :]
    if s["case"]["rope"] == "pairs":
        z = torch.view_as_complex(x.view(*x.shape[:-1], -1, 2).contiguous()) * turn
        return torch.view_as_real(z).flatten(-2)
    first, second = x.chunk(2, -1)
    z = torch.complex(first.contiguous(), second.contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers
    s = prepare(case, seed)
    hq, hkv, lens, group = case["hq"], case["hkv"], s["lens"], case["hq"] // case["hkv"]
    if case["op"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        for b, n in enumerate(lens):
            if n:
                k, v = _exact_cached(s, b, n)
                q = s["q"][b].double().view(hkv, group, -1)
                p = torch.softmax(torch.einsum("hgd,lhd->hgl", q, k) / math.sqrt(case["d"]), -1)
                out[b] = torch.einsum("hgl,lhd->hgd", p, v).reshape(hq, -1)
        return out
    if case["op"] == "read":
        parts = [_exact_cached(s, b, n, case["start"]) for b, n in enumerate(lens) if n]
        return tuple(torch.cat(x) for x in zip(*parts))
    q, k, v = _exact_turned(s["q"], s["q_norm"], s), _exact_turned(s["new_k"], s["k_norm"], s), s["new_v"].double()
    if case["cache"] == "int4":
        return q, _exact_int4(k), _exact_int4(v)
    slots, caches = s["slots"].long(), []
    for old, new in ((s["k"], k), (s["v"], v)):
        flat = old.double().transpose(1, 2).reshape(-1, hkv, case["d"])
        flat[slots] = new
        caches.append(flat.view(old.shape[0], case["page"], hkv, case["d"]).transpose(1, 2).contiguous())
    return q, *caches
