"""The 4-bit cache on the GPU: its writer, reader and the attention of single tokens over it.

The writer's codes and scales are those of the quotients themselves, which the reference takes in 64 bits, so that they are
compared exactly (f32 rows whose quotients lie within 2^-50 of a border would not be, and there are none here). The reader
rounds code x group's scale x row's scale once, or twice to 16 bits: exact where eight bits fit.

attention_decode, element by element, with A = sum_j p_j |v_j|: the output's rounding, u |o|; q in two f16 pieces (22 bits; one piece
is exact for 16-bit q) moves a score by 2^-23 scale sum |q k|, and the f32 sums of its products by up to ten roundings of that,
2^-16 in all at scale sum |q k| <= 13 (normal values, head_dim 128); the exponential is good to 2^-22 and its f32 argument below
2^5 to 2^-20; p keeps 22 bits under f32 q. A relative change of p by e moves o by 2 e A at most: 2^-15 A, and in proportion where
scale sum |q k| is more than 13. Under 16-bit q p is rounded to f16 once more, 2^-11 of itself at most: 2^-11 A (its sum is that
of p itself). Then, p s (s a row's scale) is made of f16 numbers, which have steps of 2^-24 at least: it is off by half of one, where
the largest p s is 2^7 or more, so by 2^-32 of the largest. An element is at most 3136 s, which is less than twice its row's
largest, so that each of n tokens may move o by 2^-31 of the largest p max |v|.
"""
import pytest
import torch

import attention_reference as ref
import candelora_metal_kernels_b200 as c
import kv_step_reference as step_ref
from test_attention_gpu import DECODE
from test_kv_cache_gpu import at_slots, randn, tables

pytestmark = pytest.mark.gpu
BF16, F16, F32, I4 = torch.bfloat16, torch.float16, torch.float32, torch.uint8
E4M3 = torch.float8_e4m3fn


def held(cache, slots):
    """(bytes, group scales' bits, row scales) of K and V at the slots."""
    return [(at_slots(x, slots), at_slots(g.view(torch.uint8), slots), at_slots(s, slots)) for x, g, s in
            ((cache.k, cache.k_group, cache.k_scale), (cache.v, cache.v_group, cache.v_scale))]


def same_rows(got, want, d):
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[1][..., :d // 32], want[1][..., :d // 32])
    assert torch.equal(got[2].nan_to_num(-1.0), want[2].nan_to_num(-1.0))


@pytest.mark.parametrize("rope", ["none", "half", "pairs"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,hq,hkv,d,page", [(1, 4, 2, 128, 16), (37, 5, 1, 64, 7), (300, 8, 8, 96, 48), (19, 3, 3, 32, 64),
                                                  (50, 2, 1, 128, 1), (9, 7, 7, 96, 3)])
def test_write(tokens, hq, hkv, d, page, dtype, rope):
    pages = -(-tokens // page) + 2
    cache = c.KvCache.empty(pages, hkv, page, d, I4)
    q, k, v = randn((tokens, hq, d), 1, dtype), randn((tokens, hkv, d), 2, dtype), randn((tokens, hkv, d), 3, dtype)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(4))[:tokens].to(torch.int32)
    skipped = torch.zeros(tokens, dtype=torch.bool)
    skipped[tokens // 2::5] = tokens > 1
    given = torch.where(skipped, torch.where(slots % 2 == 0, -1, pages * page), slots).to(torch.int32)
    pos = torch.randint(0, 500, (tokens,), generator=torch.Generator().manual_seed(5)).to(torch.int32)
    cos, sin = tables(500, d)
    kw = {} if rope == "none" else {"positions": pos.cuda(), "cos": cos.cuda(), "sin": sin.cuda(), "interleaved": rope == "pairs"}
    got_q = c.kv_cache_write(cache, k.cuda(), v.cuda(), given.cuda(), q=q.cuda(), q_dtype=F32, **kw).cpu()
    turn = (lambda x: x.float()) if rope == "none" else (lambda x: ref.rotated(x.float(), pos, cos, sin, rope == "pairs"))
    assert torch.equal(got_q, turn(q))
    for got, x in zip(held(cache, slots), (turn(k), v.float())):
        want = step_ref.quantised4(x)
        same_rows([t[~skipped] for t in got], [t[~skipped] for t in want], d)
        assert (got[0][skipped] == 0x88).all() and not got[2][skipped].any()
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[slots.long()] = False
    assert (at_slots(cache.k, torch.arange(pages * page))[untouched] == 0x88).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_write_codes_on_borders(dtype):
    """Rows made of multiples of half a step: the quotients are exact ties, which go to the even code; and group maxima whose
    scales lie between two e4m3 numbers."""
    d, rows = 128, 64
    gen = torch.Generator().manual_seed(3)
    halves = torch.randint(-13, 14, (rows, 1, d), generator=gen).float()
    scales = step_ref.E4M3[torch.randint(64, 126, (rows, 1, 4), generator=gen)].float()  # normal, below 448
    halves[..., 0::32] = 14.0  # each group's maximum is seven steps
    x = (halves / 2 * scales.repeat_interleave(32, -1) * 2.0 ** torch.randint(-9, 5, (rows, 1, 1), generator=gen)).to(dtype)
    between = (torch.randint(8, 16, (rows, 1, d), generator=gen) * 2 + 1).float() * 7 * 2.0 ** torch.randint(-6, 1, (rows, 1, d), generator=gen)
    for t in (x, between.to(dtype)):
        cache = c.KvCache.empty(1, 1, rows, d, I4)
        c.kv_cache_write(cache, t.cuda(), t.cuda(), torch.arange(rows, dtype=torch.int32).cuda())
        want = step_ref.quantised4(t.float())
        for got in held(cache, torch.arange(rows)):
            same_rows(got, want, d)


def test_write_rows_that_do_not_quantise():
    """Zeros, subnormal rows, infinities and NaN, the largest and smallest rows, groups far below their row's largest."""
    x = randn((12, 1, 64), 1)
    x[0], x[1], x[2, 0, 3], x[3, 0, 60] = 0, 1e-35, float("inf"), float("nan")
    x[4] *= 1e30
    x[5] = torch.where(x[5] > 0, 3.4028e38, -3.4028e38)
    x[6] = x[6].sign() * 2.0 ** -100
    x[7, :, 32:] *= 2.0 ** -12   # group scales among e4m3's subnormals
    x[8, :, 32:] *= 2.0 ** -17
    x[9, :, 32:] *= 2.0 ** -30   # and below the smallest of them
    x[10, :, :32] = 0
    x[11] = x[11].sign() * 2.0 ** -101  # zeros, as rows below 2^-100 are
    cache = c.KvCache.empty(1, 1, 16, 64, I4)
    slots = torch.arange(12, dtype=torch.int32).cuda()
    c.kv_cache_write(cache, x.cuda(), x.cuda(), slots)
    want = step_ref.quantised4(x)
    for got in held(cache, torch.arange(12)):
        same_rows(got, want, 64)
    table, cu = torch.zeros((1, 1), dtype=torch.int32).cuda(), torch.tensor([0, 12], dtype=torch.int32).cuda()
    k, v = (t.cpu()[:, 0] for t in c.kv_cache_read(cache, table, cu, 12, dtype=F32))
    assert not k[:2].any() and k[2:4].isnan().all() and torch.isfinite(k[4:]).all() and not k[11].any()
    assert torch.equal(k.nan_to_num(7), v.nan_to_num(7))
    good = [0, 4, 5, 6, 7, 8, 9, 10]
    assert torch.equal(k[good].double(), step_ref.values4(*want)[good, 0])


@pytest.mark.parametrize("pad", [0, 8, 4, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_write_strided_and_unaligned_rows(pad, dtype):
    hq, hkv, d, tokens = 4, 2, 96, 33
    rows = randn((tokens, (hq + 2 * hkv) * d + pad), 1, dtype).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    cache = c.KvCache.empty(3, hkv, 16, d, I4)
    slots = torch.arange(tokens, dtype=torch.int32).cuda()
    cos, sin = (x.cuda() for x in tables(40, d))
    c.kv_cache_write(cache, k, v, slots, q=q, positions=slots, cos=cos, sin=sin, interleaved=True)
    pos = slots.cpu()
    for got, x in zip(held(cache, pos), (ref.rotated(k.cpu().float(), pos, cos.cpu(), sin.cpu(), True), v.cpu().float())):
        same_rows(got, step_ref.quantised4(x), d)


def random_cache(pages, hkv, page, d, seed, arbitrary=False):
    """A 4-bit cache of random rows (K with channels three times as large), or of any bytes and scales."""
    if arbitrary:
        gen = torch.Generator().manual_seed(seed)
        parts = []
        for _ in range(2):
            parts.append((torch.randint(0, 256, (pages, hkv, page, d // 2), generator=gen).to(torch.uint8),
                          torch.randint(0, 127, (pages, hkv, page, 4), generator=gen).to(torch.uint8),
                          torch.rand((pages, hkv, page), generator=gen) * 0.01))
    else:
        k, v = randn((pages, hkv, page, d), seed), randn((pages, hkv, page, d), seed + 1)
        k[..., 5::16] *= 3
        parts = [step_ref.quantised4(x) for x in (k, v)]
    (k, kg, ks), (v, vg, vs) = parts
    return c.KvCache(k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), kg.cuda().view(E4M3), vg.cuda().view(E4M3))


@pytest.mark.parametrize("arbitrary", [False, True])
@pytest.mark.parametrize("dtype", [None, BF16, F16, F32])
@pytest.mark.parametrize("lens,start,hkv,d,page", [([1], 0, 2, 128, 16), ([0, 33, 0, 5, 100], 3, 3, 64, 7), ([700, 20], 0, 8, 96, 64),
                                                   ([64] * 9, 17, 1, 32, 48)])
def test_read(lens, start, hkv, d, page, dtype, arbitrary):
    need = [-(-(n + start) // page) for n in lens]
    pages, total = sum(need) + 2, sum(lens)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b in range(len(lens)):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
    cache = random_cache(pages, hkv, page, d, 5, arbitrary)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    starts = torch.full((len(lens),), start, dtype=torch.int32).cuda()
    got = c.kv_cache_read(cache, table.cuda(), cu.cuda(), total + 3, starts=starts if start else None, dtype=dtype)
    dtype = dtype or BF16
    for g, h in zip(got, step_ref.held4(cache)):
        want = torch.stack([h[table[b, (start + i) // page], :, (start + i) % page] for b, n in enumerate(lens) for i in range(n)])
        assert g.dtype == dtype and torch.equal(g[:total].cpu(), want.float().to(dtype))
        assert not g[total:].any()  # rows of no sequence
        if not arbitrary and dtype != F16:
            assert torch.equal(g[:total].double().cpu(), want)


def test_read_pages_outside_the_cache_are_zeros():
    cache = random_cache(2, 1, 4, 32, 1)
    table = torch.tensor([[1, -1, 2, 0]], dtype=torch.int32).cuda()
    k, _ = c.kv_cache_read(cache, table, torch.tensor([0, 20], dtype=torch.int32).cuda(), 20)
    have = torch.tensor([True] * 4 + [False] * 8 + [True] * 4 + [False] * 4)
    assert k.cpu().ne(0).flatten(1).any(1).equal(have) and not torch.signbit(k.cpu()[~have]).any()


# ---- one token over the cache ----

def make_cache(lens, hkv, page, d, seed, spare=3, poison=None, arbitrary=False):
    """A cache of random tokens for sequences of `lens` over shuffled pages; what no sequence holds has `poison` scales."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need, default=0)) + 1), -1, dtype=torch.int32)
    used = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
        at = torch.arange(n)
        used[table[b, at // page].long(), at % page] = True
    cache = random_cache(pages, hkv, page, d, seed + 1, arbitrary)
    if poison is not None:
        unused = ~used.cuda()[:, None].expand(pages, hkv, page)
        for s, g, x in ((cache.k_scale, cache.k_group, cache.k), (cache.v_scale, cache.v_group, cache.v)):
            s.masked_fill_(unused, poison)
            g.view(torch.uint8).masked_fill_(unused[..., None], 255)  # NaN
            x.masked_fill_(unused[..., None], 0)
            g.view(torch.uint8)[..., d // 32:] = 255                  # and in the scales past head_dim
    return cache, table


def check_decode(q, cache, table, lens, got, scale=None, most=None):
    """`most`: the largest value of the sequences' rows, where it is not among a few normal ones (8 at most)."""
    want, size = step_ref.decode4(q, cache, table, lens, scale)
    # |q| |k| >= sum |q k|, |k| of normal rows with larger channels at most 20 at head_dim 128
    scores = (q.double().norm(dim=-1).max().item() * 20 * (128 ** -0.5 if scale is None else scale))
    part = 2.0 ** -15 * max(1.0, scores / 13) + (0.0 if q.dtype == F32 else ref.UNIT[F16])
    floor = max(lens) * 2.0 ** -31 * (8.0 if most is None else most)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() - ref.UNIT[q.dtype] * want.abs() - part * size - floor).max()
    assert worst <= 0, worst
    assert not got[size.sum(-1) == 0].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens,hq,hkv,d,page", [x for x in DECODE if x[3] % 32 == 0] + [([45, 7, 130], 8, 2, 96, 16), ([33, 500], 3, 3, 32, 16)])
def test_decode(lens, hq, hkv, d, page, dtype):
    cache, table = make_cache(lens, hkv, page, d, 5, poison=float("nan"))
    q = randn((len(lens), hq, d), 9, dtype).cuda()
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    assert got.shape == q.shape and got.dtype == dtype
    check_decode(q, cache, table, lens, got)


@pytest.mark.parametrize("d", [128, 64])
def test_decode_any_bytes_and_scales(d):
    """All sixteen codes and all group scales, row scales that are not powers of two."""
    lens = [77, 260]
    cache, table = make_cache(lens, 2, 16, d, 3, arbitrary=True)
    q = 0.02 * randn((2, 8, d), 4).cuda()
    check_decode(q, cache, table, lens, c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()))


def test_decode_many_sequences():
    lens = [(37 * i) % 300 for i in range(200)]
    cache, table = make_cache(lens, 2, 16, 64, 7)
    q = randn((200, 4, 64), 8).cuda()
    check_decode(q, cache, table, lens, c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()))


def test_decode_rows_of_the_smallest_and_largest_scales():
    """Value rows of every size a row may have, in one sequence: the largest decide, and alone each is itself."""
    d, page = 64, 8
    tops = [2.0 ** -100, 1e-25, 1e-3, 1.0, 1e4, 1e30, 3e38, 0.0]
    x = randn((len(tops), 1, d), 1)
    x = x / x.abs().amax(-1, keepdim=True) * torch.tensor(tops)[:, None, None]
    k = randn((len(tops), 1, d), 2)
    for rows in [list(range(len(tops)))] + [[i] for i in range(len(tops))] + [[0, 7], [1, 0], [7]]:
        cache = c.KvCache.empty(1, 1, page, d, I4)
        c.kv_cache_write(cache, k[rows].cuda(), x[rows].cuda(), torch.arange(len(rows), dtype=torch.int32).cuda())
        table, lens = torch.zeros((1, 1), dtype=torch.int32), [len(rows)]
        q = randn((1, 2, d), 3).cuda()
        got = c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
        check_decode(q, cache, table, lens, got, most=max(tops[i] for i in rows))


def test_decode_a_row_that_is_no_number_and_one_token_of_all_the_weight():
    d, lens = 128, [50]
    cache, table = make_cache(lens, 1, 64, d, 3)
    q = randn((1, 4, d), 4).cuda()
    k = step_ref.held4(cache)[0][table[0, 0]][0, 20].float()
    check_decode(k.cuda().expand(1, 4, d) * 3, cache, table, lens,
                 c.attention_decode(k.cuda().expand(1, 4, d) * 3, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()))
    cache.v_scale[table[0, 0], 0, 30] = float("nan")
    assert c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()).isnan().all()
    assert torch.isfinite(c.attention_decode(q, cache, table.cuda(), torch.tensor([30], dtype=torch.int32).cuda())).all()


@pytest.mark.parametrize("q_top,k_top", [(1e-37, 3e38), (3e38, 1e-29), (1e38, 1.0), (1e-30, 1e30), (1e30, 1e-30), (1.0, 0.0), (0.0, 1.0)])
def test_decode_queries_and_keys_at_the_ends_of_f32(q_top, k_top):
    """Scores of a few units from factors of any size; where they pass them by far, the largest takes all."""
    d, n = 64, 40
    k, v = randn((n, 1, d), 1), randn((n, 1, d), 2)
    k, q = k / k.abs().max() * k_top, randn((1, 2, d), 3)
    q = q / q.abs().max() * q_top
    cache = c.KvCache.empty(2, 1, 32, d, I4)
    c.kv_cache_write(cache, k.cuda(), v.cuda(), torch.arange(n, dtype=torch.int32).cuda())
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    got = c.attention_decode(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda()).double().cpu()
    want, size = step_ref.decode4(q, cache, table, [n])
    # scores up to 30: relative errors of p of 30 times those of the docstring above
    near = ((got - want).abs() <= 2.0 ** -14 * 30 / 13 * size + n * 2.0 ** -31 * 8).all(-1)[0]
    # (scores are f32 numbers times log2(e): a head in which one of them passes 2^128 has no softmax in f32)
    held = step_ref.held4(cache)[0][table[0].long()].transpose(1, 2).reshape(-1, d)[:n]
    past = (q[0].double() @ held.T * d ** -0.5 * 1.4427).abs().amax(-1) >= 2.0 ** 128
    assert (near | (past & got[0].isnan().all(-1))).all() and (q_top == 1e38 or not past.any())


def test_decode_strides_scale_stream_workspace_and_repeat():
    lens, d = [300, 0, 1000], 128
    cache, table = make_cache(lens, 2, 48, d, 11)
    rows = randn((3, 3, 10 * d + 3), 12, F16).cuda()
    q = rows[:, 1, 3:3 + 8 * d].unflatten(1, (8, d))
    dev_table, dev_lens = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    ws = torch.empty(c.attention_decode_workspace_bytes(q, cache, dev_table), dtype=torch.uint8, device="cuda").fill_(255)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = c.attention_decode(q, cache, dev_table, dev_lens, scale=0.03, workspace=ws)
        again = c.attention_decode(q, cache, dev_table, dev_lens, scale=0.03, workspace=ws)
    side.synchronize()
    check_decode(q, cache, table, lens, got, 0.03)
    assert torch.equal(got, again)


def test_decode_length_past_the_table_and_pages_outside_the_cache():
    """The length is cut to the table; tokens of pages outside the cache take no part."""
    d, page = 64, 16
    cache, _ = make_cache([64], 2, page, d, 3, spare=0)
    table = torch.tensor([[2, 7, -1, 0]], dtype=torch.int32)
    q = randn((1, 4, d), 5).cuda()
    got = c.attention_decode(q, cache, table.cuda(), torch.tensor([1000], dtype=torch.int32).cuda())
    want = c.attention_decode(q, cache, table[:, [0, 3]].contiguous().cuda(), torch.tensor([32], dtype=torch.int32).cuda())
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()


def test_offsets_past_32_bits():
    """Codes past 2^32 bytes into the cache, and 2^32 elements well before."""
    pages, hkv, page, d = 9500, 8, 1024, 128
    k = torch.full((pages, hkv, page, d // 2), 0x88, dtype=torch.uint8, device="cuda")
    assert k.numel() > 2 ** 32 + 2 ** 29
    groups = torch.zeros((pages, hkv, page, 4), dtype=torch.uint8, device="cuda").view(E4M3)
    scale = torch.zeros((pages, hkv, page), device="cuda")
    cache = c.KvCache(k, k, scale, scale, groups, groups)
    x = randn((700, hkv, d), 1)
    far = pages - 1
    slots = (torch.arange(700) + far * page).to(torch.int32)
    c.kv_cache_write(cache, x.cuda(), x.cuda(), slots.cuda())
    want = step_ref.values4(*step_ref.quantised4(x))
    table, cu = torch.tensor([[far]], dtype=torch.int32).cuda(), torch.tensor([0, 700], dtype=torch.int32).cuda()
    got, _ = c.kv_cache_read(cache, table, cu, 700, dtype=F32)
    assert torch.equal(got.double().cpu(), want)
    q = randn((1, hkv, d), 2).cuda()
    out = c.attention_decode(q, cache, table, torch.tensor([700], dtype=torch.int32).cuda()).double().cpu()
    for h in range(hkv):
        o, size = ref.attend(q[0, h:h + 1].double().cpu(), want[:, h], want[:, h], [700], d ** -0.5)
        assert ((out[0, h] - o[0]).abs() <= 2.0 ** -15 * size[0] + 2.0 ** -24 * o[0].abs()).all()


def test_captured_write_and_decode():
    """A layer's write and decode in one graph, replayed with other inputs and lengths, give what eager calls give."""
    n, hq, hkv, d, page = 5, 8, 2, 128, 16
    caches = [c.KvCache.empty(40, hkv, page, d, I4) for _ in range(2)]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(n, 8).cuda()
    lens, slots = torch.zeros(n, dtype=torch.int32).cuda(), torch.full((n,), -1, dtype=torch.int32).cuda()
    q, k, v = (randn((n, h, d), i).cuda() for i, h in enumerate((hq, hkv, hkv)))
    ws = torch.empty(c.attention_decode_workspace_bytes(q, caches[0], table), dtype=torch.uint8, device="cuda")

    def layer(cache):
        return c.attention_decode(c.kv_cache_write(cache, k, v, slots, q=q), cache, table, lens, workspace=ws)

    layer(caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(caches[0])
    for turn in range(12):
        for i, x in enumerate((q, k, v)):
            x.copy_(randn(x.shape, 100 * turn + i))
        at = torch.tensor([turn, turn, 0 if turn % 3 else turn, turn * 2, 100 + turn], dtype=torch.int32).cuda()
        slots.copy_(table.gather(1, (at // page).long()[:, None])[:, 0] * page + at % page)
        lens.copy_(torch.where(torch.arange(n).cuda() == 2, 0, at + 1))
        graph.replay()
        assert torch.equal(out, layer(caches[1])) and not out[2].any()


def test_refusals():
    cache = c.KvCache.empty(2, 2, 16, 64, I4)
    k, s, g = cache.k, cache.k_scale, cache.k_group

    def refused(match, fn, *args, **kw):
        with pytest.raises(c.Iq2Error, match=match):
            fn(*args, **kw)

    refused("a 4-bit cache takes contiguous f32 scales", c.KvCache, k, k)
    refused("group scales", c.KvCache, k, k, s, s)
    refused("group scales", c.KvCache, k, k, s, s, g, g.view(torch.uint8))
    refused("group scales", c.KvCache, k, k, s, s, g, g[..., :2].contiguous())
    refused("only a 4-bit cache", c.KvCache, k.to(torch.int8), k.to(torch.int8), s, s, g, g)
    refused("takes scales", c.KvCache, k.half(), k.half(), s, s)
    refused("head_dim=48", c.KvCache, k[..., :24].contiguous(), k[..., :24].contiguous(), s, s, g, g)
    refused("head_dim=160", c.kv_cache_read, c.KvCache.empty(2, 2, 16, 160, I4), torch.zeros((1, 1), dtype=torch.int32).cuda(),
            torch.tensor([0, 1], dtype=torch.int32).cuda(), 1)
    refused("device mismatch", c.KvCache, k, k, s, s, g, g.cpu())
    # views off the 16-byte boundaries
    shifted = torch.zeros(s.numel() + 4, device="cuda")[1:1 + s.numel()].view(s.shape)
    moved = torch.zeros(g.numel() + 16, dtype=torch.uint8, device="cuda")[4:4 + g.numel()].view(g.shape).view(E4M3)
    one, x = torch.zeros(1, dtype=torch.int32).cuda(), torch.ones((1, 2, 64), device="cuda")
    refused("v_scale is not 16-byte aligned", c.kv_cache_write, c.KvCache(k, k, s, shifted, g, g), x, x, one)
    refused("k_group is not 16-byte aligned", c.attention_decode, x, c.KvCache(k, k, s, s, moved, g), one[None], one)
    refused("expects q of shape", c.attention_decode, torch.zeros((1, 2, 32)).cuda(), cache, torch.zeros((1, 1), dtype=torch.int32).cuda(),
            torch.ones(1, dtype=torch.int32).cuda())
    for name in ("k_group", "v_group"):
        with pytest.raises(AttributeError):
            setattr(cache, name, g)
    kept = cache.v_group.clone()
    cache.v_group.data = kept
    x = torch.ones((1, 2, 64), device="cuda")
    refused("have moved", c.kv_cache_write, cache, x, x, torch.zeros(1, dtype=torch.int32).cuda())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [1, 12, 24, 48, 200])
@pytest.mark.parametrize("lens,hq,hkv,d", [([1], 4, 2, 128), ([12, 0, 32, 33], 8, 1, 64), ([350, 1, 384, 385, 0, 70], 20, 2, 128), ([500, 31, 0], 9, 3, 96)])
def test_decode_with_tables_of_any_width(lens, hq, hkv, d, width, dtype):
    """Short tables let a block take an item, wide ones have the line of work: both give the same for lengths up to the table's."""
    page, lens = 32, [min(n, 32 * width) for n in lens]
    cache, table = make_cache(lens, hkv, page, d, 5, poison=float("nan"))
    table = torch.nn.functional.pad(table, (0, max(0, width - table.shape[1])), value=-1)[:, :max(width, 1)].contiguous()
    q = randn((len(lens), hq, d), 9, dtype).cuda()
    check_decode(q, cache, table, lens, c.attention_decode(q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()))
