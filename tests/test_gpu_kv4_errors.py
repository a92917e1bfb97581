"""How exact b200_kv4_attention is by root mean square, where the bounds of single outputs are too wide to tell its forms from one another."""
import numpy as np
import pytest

import kv4_util as u
from test_gpu_kv4 import Batch, bound
from test_gpu_kv4_rows import Rows

pytestmark = pytest.mark.gpu
# The rounding of a result alone: off by at most half a step, evenly, so by half a step over sqrt(3) where a value is just above a power of two, less elsewhere.
ROUNDED = {"f32": 2.0 ** -24 / 3 ** 0.5, "f16": 2.0 ** -11 / 3 ** 0.5, "bf16": 2.0 ** -8 / 3 ** 0.5}


def errors(b, last, every):
    """(rms of the error over rms of the result, largest S) over rows of the sequences before `last`; every row also within its bound, without the allowance for values
    held as 16-bit operands where the type has none."""
    out = b.run().float().cpu().numpy()
    far = size = most_S = 0.0
    for s in range(last):
        n, c, page = b.lens[s], b.counts[s], b.host.page
        for i in range(0, c, every):
            seen = n - c + i + 1
            k, v = b.host.rows([int(b.table[s, j // page]) * page + j % page for j in range(seen)])
            r = b.row_start[s] + i
            want, S, V = u.attend(b.q[r], k, v, np.ones(seen, bool), b.scale)
            off = out[r].reshape(want.shape) - want
            assert np.abs(off).max() <= bound(b.kind, S, V, seen, b.kind == "bf16" and c * b.q_heads // b.host.heads >= 64), (s, i)
            far, size, most_S = far + (off ** 2).sum(), size + (want ** 2).sum(), max(most_S, S)
    return (far / size) ** 0.5, most_S


# f32: scores of which 2^-20 S is rounded (test_gpu_kv4.py), 2^-20 for the rest.  f16: the result's rounding, a hundredth for all else: values and weights are not
# rounded to 16 bits there.  bf16: values, q and weights as f16, half a step of which is an eighth of bf16's each (2^-11 S of a score; S averages out to its root mean
# square over 64 dims and more, an eighth of it).
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,D", [(8, 2, 128), (6, 2, 64), (12, 2, 128)])
def test_sequences_of_many_rows(kind, q_heads, kv_heads, D):
    b = Rows([300, 700], [140, 100], q_heads, kv_heads, D, 16, kind, 81)
    rms, S = errors(b, 2, 5)
    limit = {"f32": 2.0 ** -20 * (1 + S), "f16": 1.01 * ROUNDED["f16"], "bf16": np.hypot(ROUNDED["bf16"], 2.0 ** -11 * (2 + S / 8))}[kind]
    assert rms <= limit, (rms, limit, S)


# Few rows: weights of 16-bit types are one f16, each off by as much as an f16 result; rows of few keys have them side by side with the result's own rounding.
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("longest", [4, 60, 600])
def test_sequences_of_few_rows(kind, longest):
    rng = np.random.default_rng(longest)
    lens = [int(x) for x in rng.integers(1, longest + 1, 40)]
    b = Batch(lens, [1] * 40, 8, 2, 128, 16, kind, 82)
    rms, S = errors(b, 40, 1)
    limit = {"f32": 2.0 ** -20 * (1 + S), "f16": 2 ** 0.5 * ROUNDED["f16"], "bf16": np.hypot(ROUNDED["bf16"], ROUNDED["f16"])}[kind]
    assert rms <= limit, (rms, limit, S)


def test_a_wait_that_gave_up_is_reported_until_the_workspace_is_zeroed():
    """The word behind the counters is what a bounded wait leaves; written from the host here."""
    import torch
    from buddy_mlir_b200 import _lib
    from gpu_util import stream
    status = _lib.load().b200_kv4_attention_status
    for b in (Batch([40, 7], [1, 3], 4, 2, 64, 16, "f32", 83), Rows([300], [140], 8, 2, 128, 16, "bf16", 84)):
        before = b.run().clone()
        assert status(b.ws.data_ptr(), stream()) == 0
        b.ws[4 * 148:4 * 149].view(torch.int32).fill_(731)
        b.run()
        assert status(b.ws.data_ptr(), stream()) == -2 and "731" in _lib.load().b200_last_error().decode()
        b.ws.zero_()
        assert (b.run() == before).all() and status(b.ws.data_ptr(), stream()) == 0


@pytest.mark.parametrize("share", [0.5, 0.6, 0.7])
def test_f16_rows_whose_weight_lies_on_few_keys(share):
    """What is left of a weight's rounding counts too where a key has a quarter of its lane's sum.  A lane of one tile has two keys, eight apart: with shares of 0.3 and
    more none is rounded.  Their values nearly cancel, so that the result's own rounding does not hide it: 2^-12 of the larger weights would be 30 times the bound."""
    from test_gpu_kv4 import dev
    b = Batch([16] * 6, [1] * 6, 2, 2, 128, 16, "f16", 85)
    b.scale = 1.0
    b.q[:] = 0.0
    b.q[:, :, 0] = 1.0
    k = np.zeros((16, 2, 128), np.float32)
    k[:8, :, :64] = np.float16(np.log(share / (1 - share)))               # (held exactly)
    for s in range(6):
        v = b.rng.standard_normal((16, 2, 128)).astype(np.float32)
        v[8:] = -share / (1 - share) * v[:8]
        slots = int(b.table[s, 0]) * 16 + np.arange(16)
        u.write(b.cache, dev(k.reshape(16, -1)), dev(v.reshape(16, -1)), "f32", dev(slots.astype(np.int64)))
    b.host.pool = b.pool.cpu().numpy()
    out = b.run().double().cpu().numpy().reshape(6, 2, 128)
    for s in range(6):
        kk, vv = b.host.rows([int(b.table[s, 0]) * 16 + j for j in range(16)])
        want, S, V = u.attend(b.q[s], kk, vv, np.ones(16, bool), 1.0)
        # scores, sums, exponentials and weights of two terms as f32 rows have them; the result's own rounding
        most = bound("f32", S, V, 16) + 2.0 ** -11 * np.abs(want)
        assert (np.abs(out[s] - want) <= most).all(), (s, np.abs(out[s] - want).max(), most.min())
