"""Which kernels a call of b200_kv4_attention launches, over the stand-in CUDA runtime: the form for many rows by the type, the sizes and how many sequences there are."""
import ctypes as C

import fake_runtime


def test_forms(tmp_path):
    fake_runtime.run(tmp_path, "test_kv4_forms", "forms")


def forms(fake):
    import numpy as np
    from buddy_mlir_b200 import _lib
    lib, seen = _lib.load(), []
    fake.on_launch(lambda name, grid, args: seen.append(next(k for k in ("kv4_attention", "kv4_chunk", "kv4_exact") if k + "_kernel" in name)))
    buf = np.zeros(1 << 16, np.uint8)
    at = (buf.ctypes.data + 255) // 256 * 256
    cache = _lib.Kv4Cache(pool=at, n_pages=1000, kv_heads=2, head_dim=128, page=64)

    def launched(kind, rows, n_seqs, stride=128, q_heads=12):
        del seen[:]
        a = _lib.Kv4Attention(q=at, out=at + 4096, dtype=kind, q_heads=q_heads, q_ld=q_heads * 128, out_ld=q_heads * 128, rows=rows, n_seqs=n_seqs, row_start=at, lens=at,
                              block_table=at, table_stride=stride, scale=0.1)
        _lib.check(lib.b200_kv4_attention(C.byref(cache), C.byref(a), at, 1 << 40, None))
        return list(seen)
    many = {_lib.F32: "kv4_exact", _lib.F16: "kv4_exact", _lib.BF16: "kv4_chunk"}
    for kind, form in many.items():
        assert launched(kind, 24, 24) == ["kv4_attention"]                # a decode step
        assert launched(kind, 1, 1) == launched(kind, 10, 1) == ["kv4_attention"]          # fewer than 64 query vectors
        assert launched(kind, 4000, 1) == [form]                          # a prompt with enough among its own rows
        assert launched(kind, 600, 1) == [form, "kv4_attention"]          # whether there is enough is seen on the device
        assert launched(kind, 600, 30) == [form, "kv4_attention"]
        assert launched(kind, 600, 1, q_heads=258) == ["kv4_attention"]   # more heads on one than a product has rows
        assert launched(kind, 64, 1, stride=1) == ["kv4_attention"]       # nowhere near enough
    assert launched(_lib.BF16, 30000, 1501) == ["kv4_attention"]
    assert launched(_lib.F32, 30000, 801) == launched(_lib.F16, 30000, 801) == ["kv4_attention"]
