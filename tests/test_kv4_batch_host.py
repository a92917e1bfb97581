"""A batch over the 4-bit cache whose kernels report failures, over the stand-in CUDA runtime: the n-th launch of a kernel writes what it would."""
import ctypes as C

import numpy as np

import fake_runtime


def test_an_allocator_that_refuses(tmp_path):
    fake_runtime.run(tmp_path, "test_kv4_batch_host", "refused_steps")


def test_an_attention_that_gives_up(tmp_path):
    fake_runtime.run(tmp_path, "test_kv4_batch_host", "waits_given_up")


def batch(fake):
    from buddy_mlir_b200 import TINY_MEGA, _lib, synthetic
    from buddy_mlir_b200.session import BatchSession, ModelSession
    _, views = synthetic.make_f32_blob(TINY_MEGA, 3)
    s = ModelSession(TINY_MEGA)
    s.load_tensors(views)
    return s, BatchSession(s, 3, 16, 16, 64, kv_bits=4), _lib


def refused_steps(fake):
    """Prefill, decode and removal each say so, and the batch is as it was: the step's status is the last word of its arguments."""
    s, b, _lib = batch(fake)
    state = {"status": 0, "adds": []}

    def launch(name, grid, args):
        if "page_step_kernel" in name:
            a = C.cast(args[0], C.POINTER(_lib.PageStep))[0]
            state["adds"].append(list((C.c_int32 * 3).from_address(a.add)))
            C.c_int32.from_address(a.status).value = state["status"]
    fake.on_launch(launch)
    q, other = b.add(), b.add()
    b.prefill(q, np.arange(20))
    b.prefill(other, np.arange(5))
    was = b.length(q), b.length(other), b.free_pages()
    assert was == (20, 5, 13)

    def fails(call):
        state["status"] = _lib.PAGES_STATE
        try:
            call()
        except _lib.B200Error as e:
            assert "allocator refused" in str(e)
        else:
            raise AssertionError("no error")
        state["status"] = 0
        assert (b.length(q), b.length(other), b.free_pages()) == was
    fails(lambda: b.prefill(q, np.arange(3)))
    fails(lambda: b.decode([other, q], [1, 2]))
    fails(lambda: b.remove(q))
    assert state["adds"][-1] == [-1, 0, 0]
    b.remove(q)
    assert b.length(q) == -1 and b.length(other) == 5 and b.free_pages() == 15
    b.decode([other], [1])
    assert state["adds"][-1] == [0, 1, 0] and b.length(other) == 6
    b.close()
    s.close()


def waits_given_up(fake):
    """The error word behind a workspace's counters makes the pass fail and is cleared, so that the next one is good; so does the status call's answer by itself."""
    s, b, _lib = batch(fake)
    state = {"code": 0, "seen": []}

    def launch(name, grid, args):
        if "kv4_attention_kernel" in name:
            counters = C.cast(args[0], C.POINTER(C.c_void_p))[20]         # Kv4Params::counters
            error = C.c_int32.from_address(counters + 4 * 148)
            state["seen"].append(error.value)
            if state["code"]:
                error.value = state["code"]
    fake.on_launch(launch)
    q = b.add()
    b.prefill(q, np.arange(20))
    for call in (lambda: b.prefill(q, np.arange(3)), lambda: b.decode([q], [1])):
        state["code"] = 731
        try:
            call()
        except _lib.B200Error as e:
            assert "code 731" in str(e)
        else:
            raise AssertionError("no error")
        state["code"] = 0
        del state["seen"][:]
        assert b.length(q) in (20, 23)
        call()
        assert state["seen"] and not any(state["seen"])
    assert b.length(q) == 24
    lib, buf = _lib.load(), np.zeros(4096, np.uint8)
    word = buf[4 * 148:4 * 149].view(np.int32)
    assert lib.b200_kv4_attention_status(buf.ctypes.data, None) == 0
    word[0] = 741
    assert lib.b200_kv4_attention_status(buf.ctypes.data, None) < 0 and "741" in lib.b200_last_error().decode()
    word[0] = 0
    assert lib.b200_kv4_attention_status(buf.ctypes.data, None) == 0
    b.close()
    s.close()
