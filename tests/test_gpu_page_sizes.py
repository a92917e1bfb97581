"""b200_page_step at the ends of its 32-bit sizes."""
import numpy as np
import pytest

import fake_runtime
import kv4_util as u
from buddy_mlir_b200 import _lib


def test_the_grid_of_very_many_rows(tmp_path):
    fake_runtime.run(tmp_path, "test_gpu_page_sizes", "grids")


def grids(fake):
    import ctypes as C
    lib, seen = _lib.load(), []
    fake.on_launch(lambda name, grid, args: seen.append(grid))
    buf = np.zeros(4096, np.uint8)
    at = (buf.ctypes.data + 15) // 16 * 16
    names = ("held", "add", "held_out", "block_table", "free_pages", "n_free", "n_free_out", "row_start", "slots", "row_seq", "row_pos", "status")
    for max_rows, ctas in ((0, 1), (2048, 1), (2049, 3), (148 * 1024, 148), (2 ** 31 - 1024, 148), (2 ** 31 - 1, 148)):
        a = _lib.PageStep(n_seqs=2, page=16, table_stride=4, n_pages=8, max_rows=max_rows, **{n: at + 64 * i for i, n in enumerate(names)})
        _lib.check(lib.b200_page_step(C.byref(a), None))
        assert seen.pop() == (ctas, 1, 1) and not seen


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
def test_as_many_rows_as_an_int_counts(in_place):
    """Loops over rows end where the next step of a thread would pass 2^31."""
    import torch
    max_rows = 2 ** 31 - 1
    step = u.Step([3, 20], [[0, -1], [1, 2]], [3, 4, 5], 6, 16, 0, in_place)
    slots = torch.full((max_rows + 1,), -9, dtype=torch.int64, device="cuda")
    step.args.max_rows, step.args.slots, step.args.row_seq, step.args.row_pos = max_rows, slots.data_ptr(), None, None
    step([15, 1])
    assert int(step.status) == 0 and step.held_out.tolist() == [18, 21] and step.row_start.tolist() == [0, 15, 16]
    assert slots[:16].tolist() == [3 + i for i in range(13)] + [5 * 16, 5 * 16 + 1, 2 * 16 + 4]
    assert int(slots[-1]) == -9
    for i in range(16, max_rows, 1 << 28):
        assert bool((slots[i:min(i + (1 << 28), max_rows)] == -1).all())
    del slots
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("page,held", [(2 ** 31 - 1, 5), (2 ** 31 - 1, 2 ** 31 - 2), (2 ** 30 + 1, 2 ** 30), (2 ** 30, 2 ** 30)])
def test_very_large_pages(page, held):
    """A sequence in one page of up to 2^31 - 1 positions, none of them free: its next row lies in that page, or nothing is done."""
    step = u.Step([held], [[1]], [], 2, page, 2)
    step([1])
    if held < page:
        assert int(step.status) == 0 and step.slots.tolist() == [page + held, -1, -9] and step.held_out.tolist() == [held + 1] and step.table.tolist() == [[1]]
    else:
        assert int(step.status) == _lib.PAGES_TABLE and step.slots.tolist() == [-1, -1, -9]
    step = u.Step([held, 7], [[1], [0]], [], 2, page, 2)                  # its end gives the page back
    step([-1, 0])
    assert int(step.status) == 0 and int(step.n_free_out) == 1 and step.free.tolist()[0] == 1 and step.held_out.tolist() == [0, 7]
