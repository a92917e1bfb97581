"""b200_kv4_attention where scores are far from zero, either way, over the whole range of f32."""
import numpy as np
import pytest

import kv4_util as u
from test_gpu_kv4 import Batch, bound, dev, rows_of
from test_gpu_kv4_rows import Rows

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
FORMS = pytest.mark.parametrize("many", [False, True])


def batch(many, kind, seed):
    return Rows([1, 150, 40], [1, 90, 1], 4, 2, 64, 16, kind, seed) if many else Batch([1, 40, 300, 17], [1, 1, 3, 2], 4, 2, 64, 16, kind, seed)


def sequences(b):
    return range(len(b.lens) - isinstance(b, Rows))


def refill(b, make):
    """make(n) gives K and V [n, heads, D] of a sequence's positions."""
    for s in sequences(b):
        n = b.lens[s]
        slots = np.array([int(b.table[s, j // 16]) * 16 + j % 16 for j in range(n)], np.int64)
        k, v = (dev(np.ascontiguousarray(x, np.float32).reshape(n, -1)) for x in make(n))
        u.write(b.cache, k, v, "f32", dev(slots))
    b.host.pool = b.pool.cpu().numpy()


def rows_with_keys(b, every):
    for s in sequences(b):
        n, c = b.lens[s], b.counts[s]
        for i in sorted(set(range(0, c, every)) | {c - 1}):
            seen = n - c + i + 1
            yield b.row_start[s] + i, b.host.rows([int(b.table[s, j // 16]) * 16 + j % 16 for j in range(seen)]), c * b.q_heads // b.host.heads >= 64


@KINDS
@FORMS
@pytest.mark.parametrize("size", [1e4, 1e6, 2.0 ** 25, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28, 1e10, 1e20, 1e31])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_one_key_has_all_the_weight(kind, many, size, sign):
    """All scores of one sign, the best one ahead of the others by far more than their rounding: the output is that key's value.  Rows whose two best are nearer are left out.
    A score's error is 2^-20 of the sum of its terms' magnitudes, 2^-10 where the cache's values are f16 operands; weights of the others below e^-60.  What is left
    are the roundings of a weight and of the result, which bound(S = 0) has."""
    b = batch(many, kind, 71)
    b.scale = size / 16
    b.q = np.abs(b.q) * sign                                              # (of the type already: signs only)
    refill(b, lambda n: (4.0 + rows_of(b.rng, n, 2, 64) * 0.2, rows_of(b.rng, n, 2, 64) * (3000.0 if n == 40 else 1.0)))
    out, looked = b.run().float().cpu().numpy(), 0
    for r, (k, v), wide in rows_with_keys(b, 7):
        for h in range(4):
            q = b.q[r, h].astype(np.float64)
            s, S = k[h // 2] @ q * b.scale, (np.abs(k[h // 2]) @ np.abs(q)).max() * b.scale
            best = int(s.argmax())
            ahead = s[best] - np.delete(s, best).max() if s.size > 1 else np.inf
            if ahead < 60 + 2.0 ** (-9 if kind == "bf16" and wide else -18) * S:
                continue
            looked += 1
            want = v[h // 2, best]
            most = bound(kind, 0.0, np.abs(want).max(), 1, kind == "bf16" and wide)
            far = np.abs(out[r].reshape(4, 64)[h] - want).max()
            assert far <= most, (r, h, far, most)
    assert looked >= 12


@KINDS
@FORMS
@pytest.mark.parametrize("size", [1.0, 1e3, 2.0 ** 24, 2.0 ** 27, 2.0 ** 29, 1e12, 1e30, 1e33])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_equal_scores(kind, many, size, sign):
    """Keys that are all the same (ones, which the format holds exactly): the mean of the values, wherever the scores lie.  The same operations on the same numbers give
    the same scores, so only weights, sums and the result are rounded."""
    b = batch(many, kind, 72)
    b.scale = sign * size / 16
    refill(b, lambda n: (np.ones((n, 2, 64)), rows_of(b.rng, n, 2, 64) * (3000.0 if n == 40 else 1.0)))
    out = b.run().float().cpu().numpy()
    for r, (k, v), wide in rows_with_keys(b, 7):
        n = v.shape[1]
        far = np.abs(out[r].reshape(2, 2, 64) - v.mean(1)[:, None]).max()
        assert far <= bound(kind, 0.0, np.abs(v).max(), n, kind == "bf16" and wide), (r, n, far)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@FORMS
@pytest.mark.parametrize("q", [-1e29, 1e29, -1e35])
def test_queries_of_any_size(kind, many, q):
    b = batch(many, kind, 73)
    b.scale = 0.125
    refill(b, lambda n: (np.ones((n, 2, 64)), rows_of(b.rng, n, 2, 64)))
    b.arrays()[0].fill_(q)
    out = b.run().float().cpu().numpy()
    for r, (k, v), wide in rows_with_keys(b, 7):
        far = np.abs(out[r].reshape(2, 2, 64) - v.mean(1)[:, None]).max()
        assert far <= bound(kind, 0.0, np.abs(v).max(), v.shape[1], kind == "bf16" and wide), (r, far)
