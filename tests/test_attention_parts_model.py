"""Who adds up the parts of an item that several thread blocks had, modelled on the CPU in random interleavings of their steps
(attention_parts.cuh): with all flags down before a launch, whatever an earlier one left, every item is added up, and from
this launch's parts alone. Flags that each block takes down for itself when it starts do not give that."""
import random

import pytest


def run(r, blocks, flags, cleared_before):
    """The parts that each joining block adds up: "new", or "old" where this launch had not written them yet."""
    flags = [False] * blocks if cleared_before else list(flags)
    parts, step, live, joined = ["old"] * blocks, [0] * blocks, list(range(blocks)), []
    while live:
        b = r.choice(live)
        others = [c for c in range(blocks) if c != b]
        if step[b] == 0:  # start
            if not cleared_before:
                flags[b] = False
        elif step[b] in (1, 4):  # are the others' there?
            if all(flags[c] for c in others):
                joined.append(["new" if c == b else parts[c] for c in range(blocks)])
                live.remove(b)
            elif step[b] == 4:
                live.remove(b)
        elif step[b] == 2:
            parts[b] = "new"
        elif step[b] == 3:
            flags[b] = True
        step[b] += 1
    return joined


@pytest.mark.parametrize("blocks", [2, 3, 4])
def test_parts_are_added_up_once_they_are_all_there(blocks):
    stale = 0
    for seed in range(2000):
        left = [random.Random(seed).random() < 0.5 for _ in range(blocks)]
        joined = run(random.Random(seed), blocks, left, True)
        assert joined and all(x == ["new"] * blocks for x in joined)
        stale += any("old" in x for x in run(random.Random(seed), blocks, left, False))
    assert stale > 0
