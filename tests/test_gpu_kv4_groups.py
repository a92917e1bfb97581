"""b200_kv4_attention where a cache's groups are of unusual magnitude: constant ones (whose minimum, rounded to f16, may lie above all of them: a negative scale), any
finite pair, and two groups of a head far from each other.  Bounds are relative to the largest value of the output's own group."""
import numpy as np
import pytest

import kv4_util as u
from test_gpu_kv4 import Batch, bound, dev, rows_of
from test_gpu_kv4_rows import Rows

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
FORMS = pytest.mark.parametrize("many", [False, True])


def batch(many, D, kind, seed, q_scale=1.0):
    """Sequences of one key to some hundred; many: beside a long prompt, so that the form for many rows has the second."""
    if many:
        return Rows([1, 150, 40], [1, 90, 1], 4, 2, D, 16, kind, seed, q_scale=q_scale)
    return Batch([1, 40, 300, 17], [1, 1, 3, 2], 4, 2, D, 16, kind, seed, q_scale=q_scale)


def refill(b, make):
    """K and V of all positions of every sequence: make(n) gives V [n, heads, D]."""
    for s in range(len(b.lens) - isinstance(b, Rows)):
        n, H, D = b.lens[s], b.host.heads, b.host.D
        slots = np.array([int(b.table[s, j // b.host.page]) * b.host.page + j % b.host.page for j in range(n)], np.int64)
        k, v = rows_of(b.rng, n, H, D), np.ascontiguousarray(make(n), np.float32)
        u.write(b.cache, dev(k.reshape(n, -1)), dev(v.reshape(n, -1)), "f32", dev(slots))
    b.host.pool = b.pool.cpu().numpy()


def check_groups(b, every=1):
    """Every output against f64, within what its own group of 64 dims allows (values of 16 bits as operands: bf16 rows of many only)."""
    out = b.run().float().cpu().numpy()
    for s in range(len(b.lens) - isinstance(b, Rows)):
        n, c, page = b.lens[s], b.counts[s], b.host.page
        many = b.kind == "bf16" and c * b.q_heads // b.host.heads >= 64
        for i in sorted(set(range(0, c, every)) | {c - 1}):
            seen = n - c + i + 1
            k, v = b.host.rows([int(b.table[s, j // page]) * page + j % page for j in range(seen)])
            r = b.row_start[s] + i
            want, S, _ = u.attend(b.q[r], k, v, np.ones(seen, bool), b.scale)
            got = out[r].reshape(want.shape)
            for g in range(0, b.host.D, 64):
                # (half of f16's smallest step, which bound() allows everywhere, is one of f16 results only)
                most = bound(b.kind, S, np.abs(v[:, :, g:g + 64]).max(), seen, many) - (2.0 ** -25 if b.kind != "f16" else 0.0)
                far = np.abs(got[:, g:g + 64] - want[:, g:g + 64]).max()
                assert far <= most, (s, i, g, far, most)


@KINDS
@FORMS
@pytest.mark.parametrize("value", [3.0012, 1000.3, 0.3, -1000.2, 3.25])
@pytest.mark.parametrize("D,which", [(64, (0,)), (128, (0, 1)), (128, (0,)), (128, (1,))])
def test_constant_groups(kind, many, value, D, which):
    b = batch(many, D, kind, 61)

    def make(n):
        v = rows_of(b.rng, n, 2, D)
        for g in which:
            v[..., 64 * g:64 * g + 64] = value
        return v
    refill(b, make)
    if value == 1000.3:                                                   # (what the case is about)
        pairs = np.ascontiguousarray(b.host._parts(int(b.table[0, 0]) * 16, 1)[0][:, 17 * D:17 * D + D // 16]).view(np.float16)
        assert pairs.reshape(2, -1, 2)[0, which[0], 0] < 0
    check_groups(b, 7)


@KINDS
@FORMS
@pytest.mark.parametrize("D", [64, 128])
def test_any_finite_pair(kind, many, D):
    """Scales of either sign with any codes, as another writer may leave them: a value is lo + scale * code whatever they are."""
    b = batch(many, D, kind, 62)
    for s in range(len(b.lens) - many):
        for j in range(b.lens[s]):
            for which in (0, 1):
                tile, _, _, pair = b.host._parts(int(b.table[s, j // 16]) * 16 + j % 16, which)
                p = np.ascontiguousarray(tile[:, pair]).view(np.float16).reshape(b.host.heads, -1, 2)
                p[..., 0] *= b.rng.choice([-1.0, -1.0, 1.0, 0.0], p.shape[:-1]).astype(np.float16)
                tile[:, pair] = p.reshape(b.host.heads, -1).view(np.uint8)
    b.pool.copy_(dev(b.host.pool))
    check_groups(b, 7)


@KINDS
@FORMS
@pytest.mark.parametrize("shift", [-20, -14, -7, 10])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("q_scale", [0.02, 1.0])
def test_groups_of_different_magnitude(kind, many, shift, which, q_scale):
    """One group of V far smaller (or larger) than the other: its outputs are as exact as they would be by themselves.  (Small queries: nearly all of the bound is weights
    and sums.)"""
    b = batch(many, 128, kind, 63, q_scale)

    def make(n):
        v = rows_of(b.rng, n, 2, 128)
        v[..., 64 * which:64 * which + 64] *= 2.0 ** shift
        return v
    refill(b, make)
    check_groups(b, 7)


@KINDS
@pytest.mark.parametrize("q_scale", [0.02, 1.0, 8.0])
def test_groups_whose_magnitude_changes_from_key_to_key(kind, q_scale):
    """Small first and large later, large first and small later, and any order: what a small group's weights were raised by has to come down again."""
    for seed in (64, 65, 66):
        b = Batch([300, 65, 700, 33], [1, 2, 1, 5], 4, 2, 128, 16, kind, seed, q_scale=q_scale)

        def make(n):
            v = rows_of(b.rng, n, 2, 128)
            x = np.linspace(-18, 10, n) if seed < 66 else b.rng.uniform(-18, 10, n)
            x = x[::-1] if seed == 65 else x
            v[..., 64 * (seed & 1):64 * (seed & 1) + 64] *= np.exp2(x).astype(np.float32)[:, None, None]
            return v
        refill(b, make)
        check_groups(b)


@pytest.mark.parametrize("D", [64, 128])
def test_how_a_group_narrower_than_its_minimums_rounding_is_held(D):
    """Where the scale is not positive every code is 0 and the value is lo, bit for bit: (values, lo, the scale's sign)."""
    rows = [(1000.3, 1000.5, -1), (3.0012, 3.001953125, -1), (-1000.2, -1000.0, -1), (3.25, 3.25, 0), (1000.2, 1000.0, 1), (65503.0, 65504.0, -1), (1e-9, 0.0, 0)]
    x = np.repeat(np.array([r[0] for r in rows], np.float32)[:, None], D, 1)
    host = u.Cache(1, 1, D, 16)
    pool = dev(host.pool)
    cache = u.cache_arg(pool, 1, 1, D, 16)
    slots = np.arange(len(rows), dtype=np.int64)
    u.write(cache, dev(x), dev(x), "f32", dev(slots))
    host.pool = pool.cpu().numpy()
    for j, (value, lo, sign) in enumerate(rows):
        for which in (0, 1):
            tile, byte, high, pair = host._parts(j, which)
            p = np.ascontiguousarray(tile[0, pair]).view(np.float16).reshape(-1, 2)
            assert (p[:, 1] == np.float16(lo)).all() and (np.sign(p[:, 0]) == sign).all(), (value, p)
            codes = tile[0, byte] >> (4 * high) & 15
            assert (codes == (15 if sign > 0 else 0)).all()
        k, _ = host.read(j)
        assert sign > 0 or (k == np.float32(lo)).all()
