"""b200_kv4_attention with many rows of a sequence, and so much to do that it has a form of its own: where that can go wrong and the few-rows form cannot."""
import numpy as np
import pytest

import kv4_util as u
from buddy_mlir_b200 import _lib
from test_gpu_kv4 import Batch, dev, poison

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])


class Rows(Batch):
    """A batch beside a long prompt (the last sequence, not looked at), with which there is enough to do."""

    def __init__(self, lens, counts, q_heads, *args, **kw):
        m = int((64e6 / q_heads) ** 0.5) + 1
        self.mine, self.pad = sum(counts), kw.get("pad", 0)
        super().__init__(list(lens) + [m], list(counts) + [m], q_heads, *args, **kw)

    def run(self, stream=None):
        return super().run(stream)[:self.mine]

    def check(self, every=1):
        out = self.run()
        got = out.float().cpu().numpy().reshape(self.mine, self.q_heads, -1)
        if self.extra:
            rest = self.outs.float().cpu().numpy()
            assert (rest[:, :self.extra] == 7.0).all() and (rest[:, -self.extra:] == 7.0).all()
        for s, c in enumerate(self.counts[:-1]):
            for i in sorted(set(range(0, c, every)) | {c - 1} if c else ()):
                want, most = self.want(s, i)
                at = self.row_start[s] + i
                assert np.abs(got[at] - want).max() <= most, (s, i, np.abs(got[at] - want).max(), most)
        assert (self.arrays()[1][self.n_rows - self.pad:] == 0).all()
        return out


def sound(b):
    from gpu_util import stream
    assert _lib.load().b200_kv4_attention_status(b.ws.data_ptr(), stream()) == 0


def slot(b, s, j):
    return int(b.table[s, j // b.host.page]) * b.host.page + j % b.host.page


@KINDS
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_changes_nothing(kind, what):
    """Infinities and NaN behind the ends (no bit changes), and at a position that only later rows see (earlier ones stay within their bound)."""
    lens, counts, page = [301, 90], [90, 40], 16
    b = Rows(lens, counts, 6, 2, 64, page, kind, 30)
    before = b.run().clone()
    poison(b, [slot(b, s, j) for s, n in enumerate(lens) for j in range(n, -(-n // page) * page)], what)
    assert (b.run() == before).all()
    poison(b, [slot(b, 0, 250)], what)
    after = b.run().float().cpu().numpy().reshape(b.mine, 6, 64)
    first = 250 - (301 - 90)                                              # the first row that sees it
    assert not np.isfinite(after[first:90]).any()
    for i in range(0, first, 3):
        want, most = b.want(0, i)
        assert np.abs(after[i] - want).max() <= most
    assert (dev(after[90:].reshape(40, -1)) == before[90:].float()).all()
    sound(b)


@KINDS
@pytest.mark.parametrize("which", [0, 1])
def test_one_group_of_one_head_that_is_not_finite(kind, which):
    """K: every output of the rows and heads that see it; V: those of its 64 dims."""
    b = Rows([200], [150], 4, 2, 128, 32, kind, 31)
    before = b.run().clone().reshape(150, 4, 128)
    tile, _, _, pair = b.host._parts(slot(b, 0, 120), which)
    pairs = tile[1, pair].copy().view(np.float16)
    pairs[2:] = np.nan                                                    # (scale, lo) of the second group
    tile[1, pair] = pairs.view(np.uint8)
    b.pool.copy_(dev(b.host.pool))
    after = b.run().reshape(150, 4, 128)
    assert (after[:, :2] == before[:, :2]).all()                          # the other kv head's
    bad = after[70:, 2:, 64 * which:]
    assert bad.isnan().all() and after[:70].isfinite().all()
    if which == 1:
        assert after[:, :, :64].isfinite().all()


def rewrite(b, s, j, x):
    """Position j of sequence s holds x [kv heads, D] instead, in K and V."""
    row = dev(np.ascontiguousarray(x, np.float32).reshape(1, -1))
    u.write(b.cache, row, row, "f32", dev(np.array([slot(b, s, j)], np.int64)))
    b.host.pool = b.pool.cpu().numpy()


@KINDS
@pytest.mark.parametrize("size", [1e-6, 1.0, 3e3, np.inf])
def test_how_large_a_key_is_changes_no_row_that_does_not_see_it(kind, size):
    """A position of other magnitude than the fifteen beside it, up to f16's whole range (where a group's scale rounds beyond it)."""
    b = Rows([301], [90], 6, 2, 64, 16, kind, 47)
    before = b.run().clone().reshape(90, 6, 64)
    x = np.where(b.rng.standard_normal((2, 64)) < 0, -1.0, 1.0)
    rewrite(b, 0, 250, np.where(x < 0, -size, size) if size == np.inf else x * size * (1 + b.rng.random((2, 64))))
    assert (b.run().reshape(90, 6, 64)[:39] == before[:39]).all()         # (row 39 is the first to see it)
    b.scale = 2.0 ** -20 if size > 1 else b.scale
    if kind == "f16" and size == np.inf:
        return                                                            # (65536 is no f16)
    b.check(every=3)


@KINDS
def test_pages_outside_the_pool_are_not_seen(kind):
    b = Rows([170, 100, 40], [70, 64, 40], 4, 2, 128, 16, kind, 32)
    b.table[0, 1], b.table[0, 3], b.table[0, 10] = -1, b.host.n_pages, -2 ** 31
    b.table[1, :4] = 2 ** 31 - 1
    b.table[2, :] = -5                                                    # no position is left: zero
    out = b.check()
    assert (out[134:174] == 0).all()
    sound(b)


@KINDS
def test_lengths_beyond_the_table_and_rows_without_positions(kind):
    b = Rows([96, 70], [80, 70], 4, 2, 64, 16, kind, 33)
    b.lens[:2] = [2 ** 31 - 1, 20]                                            # all rows of 0 see the whole table; fifty of 1 see nothing
    b.check()
    b = Rows([96, 70], [80, 70], 4, 2, 64, 16, kind, 33)
    b.lens[:2] = [-2 ** 31, 0]
    assert (b.run() == 0).all()
    sound(b)


@KINDS
@pytest.mark.parametrize("lens,counts,pad,spare", [([140], [100], 9, 2), ([1], [70], 3, 0), ([64], [64], 0, 0), ([129, 0, 257], [129, 0, 80], 30, 1)])
def test_rows_behind_the_last(kind, lens, counts, pad, spare):
    Rows(lens, counts, 6, 2, 64, 16, kind, 34, pad=pad, spare=spare).check()


def test_rows_before_the_first_and_starts_out_of_order():
    """Rows that no sequence has are zero; row_start outside 0 .. rows, or decreasing, reads and writes nothing out of range."""
    import torch
    b = Batch([150], [100], 4, 2, 64, 16, "bf16", 35, pad=2700)           # (one sequence: the rows that there could be count)
    b.arrays()
    b.ds.copy_(torch.tensor([25, 125], dtype=torch.int32))
    out = b.run().clone()
    assert (out[:25] == 0).all() and (out[125:] == 0).all()
    got = out[25:125].float().cpu().numpy().reshape(100, 4, 64)
    b.row_start = np.array([25, 125])
    for i in range(0, 100, 9):
        want, most = b.want(0, i)
        assert np.abs(got[i] - want).max() <= most
    for start in ([-50, 5000], [120, 20], [2 ** 31 - 1, -2 ** 31]):
        b.ds.copy_(torch.tensor(start, dtype=torch.int32))
        b.run()
    sound(b)


@KINDS
@pytest.mark.parametrize("extra", [1, 3, 8])
def test_rows_that_are_not_aligned(kind, extra):
    Rows([140, 7, 80], [100, 3, 33], 6, 2, 64, 16, kind, 36, extra=extra).check(every=3)


@KINDS
@pytest.mark.parametrize("scale", [0.0, -0.07, 1.5])
def test_scales(kind, scale):
    b = Rows([200, 90], [130, 1], 8, 2, 128, 16, kind, 37)
    b.scale = scale
    b.check(every=5)


def test_large_and_small_queries():
    for kind in ("f32", "f16", "bf16"):
        for q_scale in (20.0, 1e-4, 0.0):
            Rows([300], [140], 8, 2, 128, 16, kind, 38, q_scale=q_scale).check(every=5)


@KINDS
def test_a_query_that_is_not_finite_spoils_its_own_heads_only(kind):
    b = Rows([200], [100], 6, 2, 64, 16, kind, 39)
    before = b.run().clone().reshape(100, 6, 64)
    b.dq[41, 64 * 4 + 3] = float("nan")
    b.dq[99, 64 * 1 + 3] = float("inf")
    after = b.run().reshape(100, 6, 64)
    keep = np.ones((100, 6), bool)
    keep[41, 4] = keep[99, 1] = False
    assert (before[keep] == after[keep]).all() and not after[41, 4].isfinite().any() and not after[99, 1].isfinite().any()


@KINDS
@pytest.mark.parametrize("q_heads,kv_heads,D", [(128, 1, 64), (127, 1, 128), (129, 1, 64), (20, 4, 128), (5, 5, 64)])
def test_heads_that_share(kind, q_heads, kv_heads, D):
    Rows([190, 3], [90, 1], q_heads, kv_heads, D, 16, kind, 40).check(every=17)


@KINDS
def test_a_prompt_beside_decode_steps(kind):
    """Both forms in one call, each with its own rows."""
    lens = [300] + [1 + 37 * i for i in range(20)] + [200]
    Rows(lens, [280] + [1] * 20 + [64], 8, 2, 64, 16, kind, 41).check(every=11)


@pytest.mark.parametrize("kind,n,long", [("bf16", 1499, 700), ("bf16", 1500, 700), ("f32", 799, 300), ("f32", 800, 300), ("bf16", 4095, 600)])
def test_a_prompt_among_very_many_sequences(kind, n, long):
    """Around the number of sequences from which on the few-rows form has all of them, and the most that a call takes."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 4, n)]
    counts = [int(x) for x in rng.integers(0, 2, n)]
    lens[n // 2], counts[n // 2] = long, long
    Rows(lens, counts, 128, 1, 64, 16, kind, 42).check(every=101)


def test_keys_of_one_prompt_over_the_whole_chip():
    for kind in ("f32", "f16", "bf16"):
        b = Rows([9000, 40], [66, 1], 8, 8, 64, 64, kind, 43)
        first = b.check(every=13).clone()
        for _ in range(10):
            assert (b.run() == first).all()                               # parts meet in the same order
        sound(b)


def test_calls_at_once_on_two_streams():
    import torch
    a, b = (Rows([900, 40, 2000], [200, 2, 100], 8, 2, 128, 16, "bf16", s) for s in (44, 45))
    want = a.run().clone(), b.run().clone()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(30):
        for x, s in ((a, one), (b, two)):
            x.run(s.cuda_stream)
    torch.cuda.synchronize()
    assert (a.arrays()[1][:a.mine] == want[0]).all() and (b.arrays()[1][:b.mine] == want[1]).all()
    sound(a)
    sound(b)


@KINDS
def test_captured_and_replayed_with_other_lengths(kind):
    """What is launched depends on host sizes alone: a graph serves steps of every shape."""
    import torch
    b = Rows([260, 90, 33], [140, 60, 1], 8, 2, 64, 16, kind, 46)
    m = b.counts[-1]
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    everything = b.n_rows
    for lens, counts in (([260, 90, 33], [140, 60, 1]), ([260, 90, 33], [1, 1, 1]), ([0, 0, 0], [0, 0, 0]), ([100, 90, 33], [100, 7, 30]), ([260, 90, 17], [0, 90, 0]),
                         ([260, 90, 33], [140, 60, 1])):
        b.lens, b.counts, lens, counts = lens + [m], counts + [m], lens + [m], counts + [m]
        b.row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        b.ds.copy_(dev(b.row_start))
        b.dl.copy_(dev(np.array(lens, np.int32)))
        b.outs.fill_(7.0)
        graph.replay()
        got = b.arrays()[1].float().cpu().numpy().reshape(everything, 8, 64)
        for s, c in enumerate(counts[:-1]):
            for i in range(0, c, 5):
                want, most = b.want(s, i)
                assert np.abs(got[b.row_start[s] + i] - want).max() <= most, (counts, s, i)
        assert (got[b.row_start[-1]:] == 0).all()
    sound(b)
