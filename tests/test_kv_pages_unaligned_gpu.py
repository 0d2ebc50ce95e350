"""A step's slots and positions where the C ABI allows them, on any 4-byte boundary: with as many rows as the second kernel of a large step
takes (and one block of a small one), off the 16-byte boundaries each and both, and nothing written beside them."""
import ctypes
import random

import pytest
import torch

import candelora_metal_kernels_b200 as c
import kv_step_reference as ref
from candelora_metal_kernels_b200 import _lib
from test_kv_pages_gpu import empty, i32

pytestmark = pytest.mark.gpu
MARK = -77


@pytest.mark.parametrize("slots_off,positions_off", [(0, 0), (1, 0), (0, 1), (1, 1), (2, 3)])
@pytest.mark.parametrize("rows", [5, 4097, 9001, 9004])
def test_slots_and_positions_on_any_boundary(rows, slots_off, positions_off):
    rng, n, page = random.Random(rows), 70, 16
    pages, state = empty(900, page, n, 40)
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    for turn in range(2):
        new = [rng.randint(0, 2 * rows // n) for _ in range(n)]
        new[3] += 40
        while sum(new) > rows:
            new[rng.randrange(n)] = 0
        keep = [rng.choice([2 ** 31 - 1, 0, 100]) for _ in range(n)]
        room = -(-rows // 4) * 4 + 8
        held = torch.full((2 * room + 3 * n + 2,), MARK, dtype=torch.int32).cuda()
        at = held.data_ptr()
        slots, positions, rest = 4 + slots_off, room + 4 + positions_off, 2 * room
        addresses = [at + 4 * i for i in (slots, positions, rest, rest + n + 1, rest + 2 * n + 2)]
        dev_new, dev_keep = i32(new), i32(keep)
        args = _lib.KV_STEP.pack(dev_keep.data_ptr(), dev_new.data_ptr(), rows, *addresses)
        _lib.check(lib.iq2_kv_pages_step(ctypes.addressof(pages._struct), args, stream))
        want = ref.pages_step(state, page, new, rows, keep)
        got = held.tolist()
        assert got[slots:slots + rows] == want[0] and got[positions:positions + rows] == want[1]
        assert got[rest:rest + n + 1] == want[2] and got[rest + n + 1:rest + 2 * n + 2] == want[3] and got[rest + 2 * n + 2:] == want[4]
        assert all(x == MARK for x in got[:slots] + got[slots + rows:positions] + got[positions + rows:rest])
        assert pages.seq_lens.tolist() == state["lens"] and pages.block_table.tolist() == state["table"]
