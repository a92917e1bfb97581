"""The 4-bit KV cache without a GPU: sizes, refusals (arguments are looked at before the device), and that nothing runs without one."""
import ctypes as C

import numpy as np
import pytest

import kv4_util as u
from buddy_mlir_b200 import _lib

EINVAL, ENODEV, ELIMIT = -1, -3, -5
BUF = np.zeros(1 << 16, np.uint8)
AT = (BUF.ctypes.data + 255) // 256 * 256


def cache(**kw):
    c = dict(pool=AT, n_pages=4, kv_heads=2, head_dim=128, page=16)
    return _lib.Kv4Cache(**(c | kw))


def refused(rc, code=EINVAL, word=""):
    assert rc == code and word in _lib.load().b200_last_error().decode(), (rc, _lib.load().b200_last_error())


def runs_or_has_no_device(rc):
    assert rc in (0, ENODEV)


@pytest.mark.parametrize("D", [64, 128])
def test_places_are_a_bijection_of_nibbles(D):
    for place, first in ((u.k_place, 0), (u.v_place, 8 * D)):
        byte, high = place(D)
        assert len(set((2 * byte + high).ravel())) == 16 * D and byte.min() == first and byte.max() == first + 8 * D - 1


def test_pool_bytes():
    f = _lib.load().b200_kv4_pool_bytes
    assert f(3, 2, 128, 32) == 3 * 2 * 2 * 2304 and f(1, 1, 64, 16) == 1152
    assert f(70_000, 8, 128, 4096 - 16) == 70_000 * 8 * 255 * 2304            # more than 2^32
    for bad in ((0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 96, 16), (1, 1, 64, 0), (1, 1, 64, 8), (1, 1, 64, 24), (1, 1, 64, 1 << 17), (1, 1025, 64, 16),
                (1 << 30, 2, 64, 32)):
        assert f(*bad) == EINVAL, bad


BAD_CACHES = [dict(pool=None), dict(pool=AT + 8), dict(n_pages=0), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=0), dict(page=8), dict(page=17), dict(page=-16)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_a_cache_that_none_can_be(bad):
    lib, c = _lib.load(), cache(**bad)
    refused(lib.b200_kv4_write(C.byref(c), AT, 256, AT, 256, 0, AT, 1, None))
    refused(lib.b200_kv4_read(C.byref(c), AT, 256, AT, 256, 0, AT, 1, None))
    refused(lib.b200_kv4_attention(C.byref(c), C.byref(attend()), AT, 1 << 40, None))


@pytest.mark.parametrize("call", ["b200_kv4_write", "b200_kv4_read"])
def test_rows_that_are_refused(call):
    lib, c = _lib.load(), cache()
    if call == "b200_kv4_write":
        f = lambda k=AT, kld=256, v=AT, vld=256, dtype=0, slots=AT, rows=4: lib.b200_kv4_write(C.byref(c), k, kld, v, vld, dtype, slots, rows, None)  # noqa: E731
    else:
        f = lambda k=AT, kld=256, v=AT, vld=256, dtype=0, slots=AT, rows=4: lib.b200_kv4_read(C.byref(c), k, kld, v, vld, dtype, slots, rows, None)  # noqa: E731
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(rows=-1), dict(dtype=3), dict(dtype=-1), dict(kld=255), dict(vld=255), dict(kld=-256),
               dict(k=AT + 2), dict(v=AT + 1, dtype=1), dict(slots=AT + 4)):
        refused(f(**kw))
    assert lib.b200_kv4_write(None, AT, 256, AT, 256, 0, AT, 1, None) == EINVAL
    runs_or_has_no_device(f(rows=0, k=None, v=None, slots=None))


def step(**kw):
    names = ("held", "add", "held_out", "block_table", "free_pages", "n_free", "n_free_out", "row_start", "slots", "row_seq", "row_pos", "status")
    a = dict(n_seqs=2, page=16, table_stride=4, n_pages=8, max_rows=4) | {n: AT + 256 * i for i, n in enumerate(names)}
    return _lib.PageStep(**(a | kw))


@pytest.mark.parametrize("bad", [{n: None} for n in ("held", "add", "held_out", "block_table", "free_pages", "n_free", "n_free_out", "row_start", "slots", "status")]
                         + [dict(n_seqs=0), dict(page=0), dict(page=-1), dict(table_stride=0), dict(n_pages=0), dict(max_rows=-1), dict(slots=AT + 4),
                            dict(held=AT + 2), dict(table_stride=1 << 20, page=1 << 12), dict(held_out=AT + 256)])
def test_a_step_that_is_refused(bad):
    refused(_lib.load().b200_page_step(C.byref(step(**bad)), None))


def test_a_step_of_too_many_sequences():
    refused(_lib.load().b200_page_step(C.byref(step(n_seqs=8193)), None), ELIMIT, "8193")
    assert _lib.load().b200_page_step(None, None) == EINVAL


def attend(**kw):
    a = dict(q=AT, out=AT + 4096, dtype=0, q_heads=4, q_ld=512, out_ld=512, rows=2, n_seqs=2, row_start=AT, lens=AT, block_table=AT, table_stride=4, scale=0.1)
    return _lib.Kv4Attention(**(a | kw))


@pytest.mark.parametrize("bad", [{n: None} for n in ("q", "out", "row_start", "lens", "block_table")]
                         + [dict(dtype=3), dict(dtype=-1), dict(q_heads=0), dict(q_heads=3), dict(rows=-1), dict(n_seqs=0), dict(table_stride=0), dict(q_ld=511),
                            dict(out_ld=100), dict(q=AT + 2), dict(out=AT + 4097, dtype=1), dict(lens=AT + 1), dict(out=AT), dict(table_stride=1 << 28), dict(table_stride=(1 << 26) + 1)])
def test_attention_that_is_refused(bad):
    refused(_lib.load().b200_kv4_attention(C.byref(cache()), C.byref(attend(**bad)), AT, 1 << 40, None))


def test_attention_limits_and_workspace():
    lib, c = _lib.load(), cache()
    refused(lib.b200_kv4_attention(C.byref(c), C.byref(attend(n_seqs=4097)), AT, 1 << 40, None), ELIMIT, "4097")
    need = lib.b200_kv4_attention_workspace_bytes(4, 2, 128)
    assert need > 0
    refused(lib.b200_kv4_attention(C.byref(c), C.byref(attend()), AT, need - 1, None), word="workspace")
    refused(lib.b200_kv4_attention(C.byref(c), C.byref(attend()), AT + 128, 1 << 40, None), word="workspace")
    refused(lib.b200_kv4_attention(C.byref(c), C.byref(attend()), None, 1 << 40, None))
    refused(lib.b200_kv4_attention(C.byref(c), None, AT, 1 << 40, None))
    for bad in ((0, 1, 64), (3, 2, 64), (4, 0, 64), (4, 2, 96)):
        assert lib.b200_kv4_attention_workspace_bytes(*bad) == EINVAL
    runs_or_has_no_device(lib.b200_kv4_attention(C.byref(c), C.byref(attend(rows=0, q=None, out=None)), None, 1 << 40, None))


def test_the_allocator_model_hands_pages_round():
    """The tests' own allocator: what it says is what the header says."""
    p = u.Pages([3, 5, 0], [[7, -1], [2, 4], [-1, -1]], [9, 8], 4)
    assert p.step([2, -1, 6], 9, 16)[0] == 0
    assert p.held == [5, 0, 6] and p.free == [9] and p.table == [[7, 4], [2, 4], [2, 8]]


def test_a_status_of_no_workspace():
    refused(_lib.load().b200_kv4_attention_status(None, None))


def test_a_batch_of_no_model():
    out = C.c_void_p()
    refused(_lib.load().b200_batch_create_kv4(None, 4, 16, 8, 64, C.byref(out)))
    assert not out
