"""The 4-bit KV cache on a GPU: b200_kv4_write and _read against the format in numpy (bit for bit), b200_page_step against an allocator of lists,
b200_kv4_attention against f64, and the three in a row."""
import numpy as np
import pytest

import kv4_util as u
from buddy_mlir_b200 import _lib

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # half a step, relative to the value


def dev(a, kind=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if kind is None else t.to(u.torch_type(kind))


def as_held(a, kind):
    """What a value is after it has been given in this type."""
    import torch
    return torch.from_numpy(np.asarray(a, np.float32)).to(u.torch_type(kind)).float().numpy()


def rows_of(rng, n, H, D):
    width = np.exp(rng.standard_normal(D))
    return (rng.standard_normal((n, H, D)) * width + rng.standard_normal(D)).astype(np.float32)


# ---- writing and reading -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,H,D,page,odd", [(1, 1, 64, 16, 0), (1, 2, 128, 16, 0), (5, 3, 64, 48, 0), (37, 2, 128, 32, 0), (64, 8, 128, 64, 0), (41, 2, 128, 16, 1),
                                               (33, 1, 64, 16, 3)])
def test_write_and_read_bit_for_bit(kind, rows, H, D, page, odd):
    """Rows between others of a projection's output, at any slots; odd: strides and starts that only the elements are aligned to."""
    import torch
    rng = np.random.default_rng(rows + D)
    n_pages = rows // page + 3
    host = u.Cache(n_pages, H, D, page, rng)
    pool = dev(host.pool)
    slots = rng.permutation(n_pages * page)[:rows].astype(np.int64)
    if rows > 4:
        slots[[1, 3]] = -1, n_pages * page                               # (left out)
    x = [rows_of(rng, rows, H, D) for _ in range(2)]
    wide = torch.zeros(rows, 3 * H * D + odd, dtype=u.torch_type(kind), device="cuda")
    k, v = wide[:, odd:odd + H * D], wide[:, odd + H * D:odd + 2 * H * D]
    k.copy_(dev(x[0].reshape(rows, -1)))
    v.copy_(dev(x[1].reshape(rows, -1)))
    cache = u.cache_arg(pool, n_pages, H, D, page)
    u.write(cache, k, v, kind, dev(slots))
    for r, s in enumerate(slots):
        if 0 <= s < n_pages * page:
            host.write(int(s), as_held(x[0][r], kind), as_held(x[1][r], kind))
    assert np.array_equal(pool.cpu().numpy(), host.pool)                  # what was written, and all else as it was
    back = torch.full((2, rows, H * D + odd), 7.0, dtype=u.torch_type(kind), device="cuda")
    u.read(cache, back[0, :, odd:], back[1, :, odd:], kind, dev(slots))
    got = back.float().cpu().numpy()
    assert (got[:, :, :odd] == 7.0).all()
    for r, s in enumerate(slots):
        want = host.read(int(s)) if 0 <= s < n_pages * page else [np.zeros((H, D))] * 2
        for which in (0, 1):
            assert np.array_equal(got[which, r, odd:], as_held(want[which], kind).ravel())


@pytest.mark.parametrize("D", [64, 128])
def test_values_at_the_ends_of_the_range(D):
    """Constants, zeros of both signs, infinities, NaN, values beyond f16, groups whose scale underflows, and rounding ties."""
    rng = np.random.default_rng(5)
    x = np.zeros((12, 1, D), np.float32)
    x[1] = 3.25
    x[2] = rng.choice([0.0, -0.0], D)
    x[3], x[3, 0, 5] = rng.standard_normal(D), np.inf
    x[4], x[4, 0, 7] = rng.standard_normal(D), -np.inf
    x[5], x[5, 0, D - 1] = rng.standard_normal(D), np.nan
    x[6] = rng.standard_normal(D) * 1e30
    x[7] = rng.standard_normal(D) * 1e-8                                  # a scale below f16's smallest
    x[8] = rng.standard_normal(D) * 3e-7                                  # subnormal scales
    x[9] = rng.integers(0, 31, D) / 2.0                                   # ties: 0.5, 1.5, ..
    x[9, 0, ::64], x[9, 0, 1::64] = 0.0, 15.0
    x[10] = 1000.0 + rng.standard_normal(D) * 0.01                        # an offset that f16 holds coarsely
    x[11] = rng.standard_normal(D) * 1e-42                                # subnormal f32
    host = u.Cache(1, 1, D, 16)
    pool = dev(host.pool)
    cache = u.cache_arg(pool, 1, 1, D, 16)
    slots = np.arange(12)
    u.write(cache, dev(x[:, 0]), dev(x[::-1, 0].copy()), "f32", dev(slots))
    import torch
    back = torch.empty(2, 12, D, device="cuda")
    u.read(cache, back[0], back[1], "f32", dev(slots))
    got = back.cpu().numpy()
    for r in range(12):
        for which, row in ((0, x[r]), (1, x[11 - r])):
            assert np.array_equal(got[which, r], u.values(*u.quantise(row))[0], equal_nan=True), (r, which)
    finite = np.isfinite(x[:, 0]).all(1) & (np.abs(x[:, 0]).max(1) < 65504)
    g = x[finite, 0].reshape(-1, 64)
    step = (g.max(1) - g.min(1)) / 15
    # half a step of codes; lo, rounded to f16, 15 times the scale's rounding
    far = np.abs(got[0][finite].reshape(-1, 64) - g).max(1)
    assert (far <= step * (0.5 + 15 * 2.0 ** -11) * (1 + 1e-5) + 2 * np.abs(g).max(1) * 2.0 ** -11 + 16 * 2.0 ** -25).all()


def test_a_pool_of_more_than_two_to_the_32_bytes():
    """Offsets beyond 32 bits: the last page of a pool of 5 GB."""
    import torch
    H, D, page = 8, 128, 64
    n_pages = 5_000_000_000 // (H * page // 16 * u.tile_bytes(D))
    pool = torch.zeros(n_pages * (H * page // 16) * u.tile_bytes(D), dtype=torch.uint8, device="cuda")
    cache = u.cache_arg(pool, n_pages, H, D, page)
    rng = np.random.default_rng(1)
    x = rows_of(rng, 3, H, D)
    slots = np.array([n_pages * page - 1, 17, n_pages * page - 16], np.int64)
    u.write(cache, dev(x.reshape(3, -1)), dev(x[::-1].reshape(3, -1).copy()), "f32", dev(slots))
    back = torch.empty(2, 3, H * D, device="cuda")
    u.read(cache, back[0], back[1], "f32", dev(slots))
    assert np.array_equal(back[0].cpu().numpy().reshape(3, H, D), u.values(*u.quantise(x)))
    q = torch.from_numpy(rng.standard_normal((1, H * D)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    table[0, 0] = n_pages - 1
    one = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    u.attention(cache, q, out, "f32", H, one(0, 1), one(page), table, 0.05, u.workspace(H, H, D))
    k, v = np.zeros((H, page, D)), np.zeros((H, page, D))
    for s, i in ((0, page - 1), (2, page - 16)):
        k[:, i], v[:, i] = u.values(*u.quantise(x[s])), u.values(*u.quantise(x[::-1][s]))
    want, S, V = u.attend(q.cpu().numpy().reshape(H, D), k, v, np.ones(page, bool), 0.05)
    assert np.abs(out.cpu().numpy().reshape(H, D) - want).max() <= bound("f32", S, V, page)


# ---- the allocator -----------------------------------------------------------------------------------------------------------
def compare(step, model, want, max_rows, n_pages):
    status, start, slots, seqs, poss = want
    assert int(step.status) == status
    assert step.held_out.tolist() == model.held and int(step.n_free_out) == len(model.free)
    assert step.row_start.tolist() == start
    assert step.slots.tolist() == slots + [-9] and step.row_seq.tolist() == seqs + [-9] and step.row_pos.tolist() == poss + [-9]
    assert step.table.tolist() == model.table
    assert step.free.tolist()[:len(model.free)] == model.free


@pytest.mark.parametrize("n,page,stride,prompt", [(1, 16, 9, 40), (3, 1, 30, 9), (31, 16, 6, 33), (100, 7, 11, 20), (1024, 16, 3, 20), (1025, 64, 2, 70), (8192, 16, 2, 5)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_against_lists(n, page, stride, prompt, in_place):
    rng = np.random.default_rng(n + page)
    n_pages = max(4, n * stride * 2 // 3)
    order = [int(p) for p in rng.permutation(n_pages)]
    model = u.Pages([0] * n, [[-1] * stride for _ in range(n)], order, page)
    max_rows = n + prompt * (n // 4 + 1)
    step = u.Step(model.held, model.table, model.free, n_pages, page, max_rows, in_place)
    seen = set()
    for i in range(14 if n < 2000 else 4):
        add = rng.choice([0, 1, 1, 1, -1, prompt // 2, prompt], n, p=[.1, .3, .2, .1, .1, .1, .1] if i % 5 < 3 else [0, .1, .1, 0, .2, .3, .3])
        if i == 3:
            add[:] = 0
        if i == 6:
            add[:] = -1
        want = model.step([int(a) for a in add], max_rows, n_pages)
        step(add)
        compare(step, model, want, max_rows, n_pages)
        seen.add(want[0])
        if not in_place:      # the same step again, then the outputs become the inputs
            step()
            compare(step, model, want, max_rows, n_pages)
            step.held.copy_(step.held_out)
            step.n_free.copy_(step.n_free_out)
    assert 0 in seen


@pytest.mark.parametrize("what,status", [("pages", 1), ("table", 2), ("rows", 3), ("held", 4), ("negative", 4), ("free", 4), ("returned", 4)])
def test_a_step_that_cannot_be_taken_changes_nothing(what, status):
    held, add, max_rows, n_pages = [20, 0, 33, 5], [1, 13, -1, 0], 20, 12
    table, free = [[0, 1, -1], [-1] * 3, [2, 3, 4], [5, -1, -1]], [6, 7, 8]
    if what == "pages":
        add, free = [20, 40, 0, 0], [6, 7]
        max_rows = 99
    elif what == "table":
        add = [1, 49, 0, 0]
    elif what == "rows":
        max_rows = 13
    elif what == "held":
        held[3] = 49
    elif what == "negative":
        held[1] = -1
    step = u.Step(held, table, free, n_pages, 16, max_rows)
    if what == "free":
        step.n_free.fill_(13)
    elif what == "returned":
        step.n_free.fill_(10)                                             # and three come back: more than there are
    before = step.table.clone(), step.free.clone()
    step(add)
    assert int(step.status) == status and step.held_out.tolist() == held and int(step.n_free_out) == int(step.n_free)
    assert (step.table == before[0]).all() and (step.free == before[1]).all()
    assert step.row_start.tolist() == [0] * 5 and step.slots.tolist() == [-1] * max_rows + [-9]


def test_sums_beyond_32_bits_are_refused():
    n = 300
    step = u.Step([0] * n, [[-1]] * n, [0, 1], 2, 16, 5)
    step([2 ** 31 - 1] * n)
    assert int(step.status) == _lib.PAGES_TABLE
    step = u.Step([0] * n, [[-1] * 4] * n, [0, 1], 2, 1 << 28, 5)
    step([1 << 29] * n)                                                   # 37 bits of rows
    assert int(step.status) == _lib.PAGES_ROWS


def test_row_maps_may_be_left_out():
    step = u.Step([3, 0], [[0], [-1]], [1], 2, 16, 4)
    step.args.row_seq = step.args.row_pos = None
    step([1, 2])
    assert step.slots.tolist() == [3, 16, 17, -1, -9] and step.row_seq.tolist() == [-9] * 5


# ---- attention ---------------------------------------------------------------------------------------------------------------
def bound(kind, S, V, n, many=False):
    """Of an output's error.  S: the largest sum of |q||k| of a score; V: the largest |v|; n: keys.
    A score: at most 2^-20 S (f32 sums of sixteen terms at a time that round towards zero, 2^-23 each, eight in a row for a group, one of two terms of q;
    parameters' products), so weights twice that, in the sum and the total.  A sum of n weighted values: 2^-23 for every
    sixteen keys, and some for the sums of warps and CTAs.  Weights as operands: half a step of f16 (f32:
    of two f16), exponentials 2^-21.  many: the cache's values as f16 operands (sequences of many rows in 16-bit types), half a step each, which is 2^-11 S of a
    score, twice in the weights, and 2^-11 V.  The output's own rounding.  All relative to V, which bounds each sum of weighted values over the sum of weights."""
    weight = {"f32": 2.0 ** -21, "f16": 2.0 ** -11, "bf16": 2.0 ** -11}[kind]
    sums = (n / 16 + 16) * 2.0 ** -23
    weight += (2.0 ** -10 * S + 2.0 ** -11) * many
    return V * (2.0 ** -18 * S + 2 * sums + 2.0 ** -20 + weight) + V * HALF[kind] + 2.0 ** -25


class Batch:
    """Sequences of a cache whose pages lie anywhere, their newest rows as queries."""

    def __init__(self, lens, counts, q_heads, kv_heads, D, page, kind, seed, pad=0, spare=0, q_scale=1.0, extra=0):
        rng = self.rng = np.random.default_rng(seed)
        self.kind, self.q_heads, self.scale, self.lens, self.counts = kind, q_heads, D ** -0.5, lens, counts
        self.stride = max(1, max(-(-n // page) for n in lens)) + spare
        pages = [-(-n // page) for n in lens]
        self.host = u.Cache(sum(pages) + 2, kv_heads, D, page, rng)
        order = rng.permutation(sum(pages) + 2)
        self.table = np.full((len(lens), self.stride), 0, np.int32)
        at = 0
        for s, n in enumerate(pages):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.pool = dev(self.host.pool)
        self.cache = u.cache_arg(self.pool, self.host.n_pages, kv_heads, D, page)
        # every position that is held is written; what lies behind a sequence's last is whatever the bytes say
        slots = np.concatenate([[int(self.table[s, j // page]) * page + j % page for j in range(n)] for s, n in enumerate(lens)] + [[]]).astype(np.int64)
        if slots.size:
            k, v = (dev(rows_of(rng, slots.size, kv_heads, D).reshape(slots.size, -1)) for _ in range(2))
            u.write(self.cache, k, v, "f32", dev(slots))
            self.host.pool = self.pool.cpu().numpy()
        self.row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.n_rows = int(self.row_start[-1]) + pad
        self.q = as_held(rng.standard_normal((self.n_rows, q_heads, D)) * q_scale, kind)
        self.extra = extra
        self.ws = u.workspace(q_heads, kv_heads, D)

    def arrays(self):
        import torch
        if not hasattr(self, "dq"):
            cols = self.q.shape[1] * self.q.shape[2]
            self.dq = torch.zeros(self.n_rows, cols + self.extra, dtype=u.torch_type(self.kind), device="cuda")[:, self.extra:]
            self.dq.copy_(dev(self.q.reshape(self.n_rows, -1)))
            self.ds, self.dl, self.dt = dev(self.row_start), dev(np.array(self.lens, np.int32)), dev(self.table)
            self.outs = torch.full((self.n_rows, cols + 2 * self.extra), 7.0, dtype=u.torch_type(self.kind), device="cuda")
        return self.dq, self.outs[:, self.extra:self.extra + self.dq.shape[1]], self.ds, self.dl, self.dt

    def run(self, stream=None):
        q, out, start, lens, table = self.arrays()
        u.attention(self.cache, q, out, self.kind, self.q_heads, start, lens, table, self.scale, self.ws, stream)
        return out

    def want(self, s, i):
        """(f64 output, bound) of row i of sequence s."""
        n, page = self.lens[s], self.host.page
        seen = min(max(0, n - self.counts[s] + i + 1), self.stride * page)
        slots = [int(self.table[s, j // page]) * page + j % page if 0 <= self.table[s, j // page] < self.host.n_pages else -1 for j in range(seen)]
        key = (s, seen)
        if getattr(self, "kept", (None,))[0] != key:
            self.kept = key, self.host.rows(slots)
        k, v = self.kept[1]
        ok = np.array([x >= 0 for x in slots], bool)
        out, S, V = u.attend(self.q[self.row_start[s] + i], k, v, ok, self.scale)
        return out, bound(self.kind, S, V, seen, self.kind != "f32" and self.counts[s] * self.q_heads // self.host.heads >= 64)

    def check(self, every=1):
        out = self.run()
        got = out.float().cpu().numpy().reshape(self.n_rows, self.q_heads, -1)
        if self.extra:
            rest = self.outs.float().cpu().numpy()
            assert (rest[:, :self.extra] == 7.0).all() and (rest[:, -self.extra:] == 7.0).all()
        at = 0
        for s, c in enumerate(self.counts):
            for i in range(c):
                if at % every == 0 or i == c - 1:
                    want, most = self.want(s, i)
                    assert np.abs(got[at + 0] - want).max() <= most, (s, i, np.abs(got[at] - want).max(), most)
                at += 1
        assert (got[at:] == 0).all()
        return out


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,D,page", [(12, 2, 128, 16), (32, 8, 128, 64), (4, 2, 64, 16), (8, 1, 128, 48), (3, 3, 64, 32), (24, 1, 64, 16), (40, 1, 128, 16)])
def test_decode_steps(kind, q_heads, kv_heads, D, page):
    """One row of every sequence, of no position to some hundred; around the ends of tiles and pages."""
    lens = [1, 2, 0, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 257, 400]
    Batch(lens, [1] * len(lens), q_heads, kv_heads, D, page, kind, 3).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,D", [(12, 2, 128), (4, 2, 64), (8, 8, 128), (8, 1, 64)])
def test_ragged_rows(kind, q_heads, kv_heads, D):
    """Several rows of a sequence, none of others, more rows than positions (those see none), and rows behind the last."""
    lens, counts = [5, 70, 0, 33, 16, 3, 129, 1, 200], [5, 3, 0, 0, 16, 7, 20, 1, 9]
    Batch(lens, counts, q_heads, kv_heads, D, 16, kind, 4, pad=5, spare=1).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,counts,heads", [([300], [300], (4, 2, 64)), ([133], [133], (12, 2, 128)), ([500, 20, 90], [77, 1, 90], (4, 1, 128)), ([260], [40], (32, 8, 128))])
def test_prompts(kind, lens, counts, heads):
    Batch(lens, counts, *heads, 32, kind, 5).check(every=7)


@pytest.mark.parametrize("kind,heads,n", [("f32", (12, 2, 128), 9001), ("bf16", (8, 1, 64), 12345), ("f16", (4, 4, 128), 5000)])
def test_long_contexts_are_shared(kind, heads, n):
    """Keys of few sequences over the whole chip, between short ones."""
    Batch([7, n, 3, n // 3, 1], [1] * 5, *heads, 16, kind, 6).check()


def test_many_short_sequences():
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(0, 40, 700)]
    Batch(lens, [1] * 700, 8, 2, 64, 16, "f16", 7).check(every=13)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("extra", [1, 3])
def test_rows_that_are_not_aligned(kind, extra):
    Batch([40, 7], [3, 1], 6, 2, 64, 16, kind, 8, extra=extra).check()


def test_large_scores():
    """Queries twenty times as large: weights of one key, exponentials over a wide range."""
    for kind in ("f32", "f16", "bf16"):
        Batch([150, 33, 1000], [1, 4, 1], 8, 2, 128, 16, kind, 9, q_scale=20.0).check()


def poison(b, slots, what):
    """The pairs of K and V of these slots become `what` (NaN, infinity)."""
    for s in slots:
        for which in (0, 1):
            tile, _, _, pair = b.host._parts(int(s), which)
            tile[:, pair] = np.full(b.host.D // 32, what, np.float16).view(np.uint8)
    b.pool.copy_(dev(b.host.pool))


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_what_a_row_does_not_see_changes_nothing(kind, what):
    """NaN and infinities behind a sequence's end, and at positions that only its later rows see."""
    lens, counts, page = [37, 20, 64, 1], [1, 6, 1, 1], 16
    b = Batch(lens, counts, 6, 2, 64, page, kind, 10)
    before = b.run().clone()
    slot = lambda s, j: int(b.table[s, j // page]) * page + j % page  # noqa: E731
    poison(b, [slot(s, j) for s, n in enumerate(lens) for j in range(n, -(-n // page) * page)] + [slot(1, 17)], what)
    after = b.run()
    same = np.ones(b.n_rows, bool)
    same[4:7] = False                                                     # rows of sequence 1 at positions 17, 18, 19
    same = dev(same)
    assert (before[same] == after[same]).all()
    assert not after[~same].isfinite().any()


def test_pages_outside_the_pool_are_not_seen():
    b = Batch([70, 40, 10], [1, 2, 1], 4, 2, 128, 16, "f32", 11)
    b.table[0, 1], b.table[0, 3], b.table[1, 0], b.table[2, 0] = -1, b.host.n_pages, -2 ** 31, 2 ** 31 - 1
    b.check()                                                             # (of the last sequence: no position is left, zero)


def test_lengths_beyond_the_table_are_cut():
    b = Batch([48, 20], [1, 1], 4, 2, 64, 16, "f32", 12)
    b.lens = [2 ** 31 - 1, 20]
    b.check()
    b = Batch([48, 20], [1, 1], 4, 2, 64, 16, "f32", 12)
    b.lens = [-5, -2 ** 31]
    b.check()


def test_a_query_that_is_not_finite_spoils_its_own_heads_only():
    for kind in ("f32", "f16", "bf16"):
        b = Batch([50, 50], [2, 1], 6, 2, 64, 16, kind, 13)
        before = b.run().clone().reshape(3, 6, 64)
        b.dq[1, 64 * 4 + 3] = float("nan")
        b.dq[2, 64 * 1 + 3] = float("inf")
        after = b.run().reshape(3, 6, 64)
        keep = np.ones((3, 6), bool)
        keep[1, 4] = keep[2, 1] = False
        assert (before[keep] == after[keep]).all() and after[1, 4].isnan().all() and not after[2, 1].isfinite().any()


def test_the_same_call_gives_the_same_bits():
    b = Batch([3000, 500, 1, 77], [1, 3, 1, 1], 12, 2, 128, 16, "f32", 14)
    first = b.run().clone()
    for _ in range(20):
        assert (b.run() == first).all()


def test_calls_at_once_on_two_streams():
    import torch
    a, b = (Batch([900, 40, 2000], [1, 2, 1], 8, 2, 128, 16, "bf16", s) for s in (15, 16))
    want = a.run().clone(), b.run().clone()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(30):
        for x, s in ((a, one), (b, two)):
            x.run(s.cuda_stream)
    torch.cuda.synchronize()
    assert (a.run() == want[0]).all() and (b.run() == want[1]).all()


# ---- together ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,captured", [("f32", False), ("bf16", False), ("f16", True), ("f32", True)])
def test_a_serving_run(kind, captured):
    """Steps in place on the device: requests come, grow and end, their rows are written and attended to, all of it captured once and replayed; against a host
    that keeps lists."""
    import torch
    rng = np.random.default_rng(17)
    n, page, stride, H, QH, D, cap = 9, 16, 8, 2, 6, 64, 60
    n_pages = 30
    host = u.Cache(n_pages, H, D, page)
    pool = dev(host.pool)
    cache = u.cache_arg(pool, n_pages, H, D, page)
    model = u.Pages([0] * n, [[-1] * stride for _ in range(n)], [int(p) for p in rng.permutation(n_pages)], page)
    step = u.Step(model.held, model.table, model.free, n_pages, page, cap, in_place=True)
    qkv = torch.zeros(cap, (QH + 2 * H) * D, dtype=u.torch_type(kind), device="cuda")
    q, k, v = qkv.split([QH * D, H * D, H * D], 1)
    out, ws, slots = torch.empty(cap, QH * D, dtype=qkv.dtype, device="cuda"), u.workspace(QH, H, D), step.slots[:cap]

    def one():
        step()
        u.write(cache, k, v, kind, slots)
        u.attention(cache, q, out, kind, QH, step.row_start, step.held_out, step.table, 0.2, ws)
    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            one()                                                         # (of no rows)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            one()
    ended = 0
    for i in range(16):
        add = rng.choice([0, 1, 1, 1, -1, 7, 21], n, p=[.1, .3, .2, .1, .1, .1, .1])
        add = [int(a) if a < 1 or model.held[s] + a <= page * stride else -1 for s, a in enumerate(add)]
        want = model.step(add, cap, n_pages)
        rows = as_held(rows_of(rng, cap, QH + 2 * H, D), kind)
        qkv.copy_(dev(rows.reshape(cap, -1)))
        step.add.copy_(torch.tensor(add, dtype=torch.int32))
        if graph is not None:
            graph.replay()
        else:
            one()
        compare(step, model, want, cap, n_pages)
        ended += want[0] != 0
        live = [r for r in range(cap) if want[2][r] >= 0]
        for r in live:
            host.write(want[2][r], rows[r, QH:QH + H], rows[r, QH + H:])
        assert np.array_equal(pool.cpu().numpy(), host.pool)
        got = out.float().cpu().numpy().reshape(cap, QH, D)
        for r in live[::5] + live[-1:]:
            s, pos = want[3][r], want[4][r]
            kk, vv = host.rows([model.table[s][j // page] * page + j % page for j in range(pos + 1)])
            o, S, V = u.attend(rows[r, :QH], kk, vv, np.ones(pos + 1, bool), 0.2)
            assert np.abs(got[r] - o).max() <= bound(kind, S, V, pos + 1, kind != "f32" and add[s] * QH // H >= 64)
        assert (got[len(live):] == 0).all()
    assert ended < 16
