"""How the decode attentions deal their work, by the kernels' own code: tests/decode_work_host.cu runs Cursor of attention_decode.cuh on
the host. Every token of every item is taken once and in order, a warp leaves two pieces at most, the blocks' parts lie where the
records look for them, no place is used twice, and what is joined is what there is; and the constants that the models of the same on
the CPU restate are the kernels'."""
import random
import subprocess

import pytest

import test_attention_work_model as others_model
import test_kv_int4_work_model as int4_model
from candelora_metal_kernels_b200.build import ARCH, CSRC, nvcc
from conftest import ROOT


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    out = tmp_path_factory.mktemp("work") / "decode_work"
    subprocess.run([nvcc(), "-std=c++17", "-O1", *ARCH, "--expt-relaxed-constexpr", "-I", str(CSRC), "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "decode_work_host.cu"), "-o", str(out)], check=True)
    return out


def dealt(program, calls):
    """The constants, and for each call (kind, blocks, items, lens) its blocks: [(parts, joins)]."""
    text = "\n".join(" ".join(map(str, (kind, blocks, items, len(lens), *lens))) for kind, blocks, items, lens in calls)
    lines = subprocess.run([str(program)], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
    out, now = [], []
    for line in lines[1:]:
        word, *numbers = line.split()
        numbers = tuple(map(int, numbers))
        if word == "block":
            now.append(([], []))
        elif word == "end":
            out.append(now)
            now = []
        else:
            now[-1][word == "join"].append(numbers)
    assert len(out) == len(calls)
    return tuple(map(int, lines[0].split())), out


def check(blocks, items, lens):
    outputs, places = {}, {}

    def whole(key, spans):
        assert key not in outputs
        outputs[key] = spans

    for block, (parts, _) in enumerate(blocks):
        pieces = []
        for warp, b, item, t0, t1, is_whole, first in parts:
            assert t0 < t1 <= lens[b] and is_whole == ((t0, t1) == (0, lens[b]))
            if is_whole:
                whole((b, item), [(t0, t1)])
            else:
                pieces.append(((b, item), t0, t1, warp, first))
        for warp in {p[3] for p in pieces}:
            assert sum(p[3] == warp for p in pieces) <= 2
        while pieces:
            key = pieces[0][0]
            same = [p for p in pieces if p[0] == key]
            assert pieces[:len(same)] == same and all(a[2] == b[1] for a, b in zip(same, same[1:]))
            pieces = pieces[len(same):]
            span = (same[0][1], same[-1][2])
            if span == (0, lens[key[0]]):
                whole(key, [span])
            else:
                place = (block, 0 if same[0][4] else 1)
                assert place not in places
                places[place] = (key, span)
    for _, joins in blocks:
        for b, item, c0, c1, slot in joins:
            got = [places.pop((c, slot if c == c0 else 0)) for c in range(c0, c1 + 1)]
            assert all(key == (b, item) for key, _ in got)
            whole((b, item), [span for _, span in got])
    assert not places
    assert sorted(outputs) == [(b, i) for b, n in enumerate(lens) if n for i in range(items)]
    for (b, _), spans in outputs.items():
        assert spans[0][0] == 0 and spans[-1][1] == lens[b] and all(x[1] == y[0] for x, y in zip(spans, spans[1:]))


def test_constants_of_the_models(program):
    (unit, cost, warps, others_cost), _ = dealt(program, [])
    assert (unit, cost, warps) == (int4_model.UNIT, int4_model.COST, int4_model.WARPS)
    assert others_cost == others_model.decode_parts.__defaults__[-1]


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("blocks", [1, 2, 7, 148])
def test_every_token_once(program, blocks, kind):
    rng, calls = random.Random(blocks), []
    for _ in range(80):
        n = rng.choice([1, 1, 2, 5, 30, 300])
        most = rng.choice([1, 31, 33, 200, 3000, 400000 if n < 3 else 500])
        calls.append((kind, blocks, rng.choice([1, 2, 8, 16]), [rng.choice([0, 1, 32, most, rng.randint(1, most)]) for _ in range(n)]))
    for (_, _, items, lens), got in zip(calls, dealt(program, calls)[1]):
        check(got, items, lens)


@pytest.mark.parametrize("kind", [0, 1])
def test_lines_of_about_a_unit_a_warp(program, kind):
    calls = [(kind, blocks, items, lens) for units in range(1, 60) for blocks in (1, 2, 3, 4)
             for items, lens in ((1, [32 * units]), (2, [32] * units), (3, [0, units, 0]))]
    for (_, _, items, lens), got in zip(calls, dealt(program, calls)[1]):
        check(got, items, lens)


def test_the_longest_lines(program):
    """Units past 32 bits in a line, sequences at the end of int32, of as many items as a call may have (2^32 - 1 units a sequence)."""
    calls = [(1, 148, 63, [2 ** 31 - 1, 5]), (0, 148, 255, [5, 2 ** 31 - 1]), (1, 148, 63, [2 ** 31 - 1] * 40)]
    for (_, _, items, lens), got in zip(calls, dealt(program, calls)[1]):
        check(got, items, lens)
