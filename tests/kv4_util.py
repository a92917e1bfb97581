"""The 4-bit KV cache in numpy, from the words of buddy_b200.h: its quantiser, its bytes, its page allocator, attention in f64; and what the
tests share to reach the library's calls."""
import ctypes as C

import numpy as np

from buddy_mlir_b200 import _lib

MOST = np.float32(65504)


def quantise(x):
    """[..., D] f32 -> codes (uint8), scale, lo (f16) of [..., D / 64]."""
    x = np.clip(np.asarray(x, np.float32), -MOST, MOST)          # (NaN stays)
    g = x.reshape(x.shape[:-1] + (-1, 64))
    with np.errstate(all="ignore"):
        lo = g.min(-1).astype(np.float16)
        scale = ((g.max(-1) - lo.astype(np.float32)) / np.float32(15)).astype(np.float16)
        s = scale.astype(np.float32)[..., None]
        q = np.clip(np.rint((g - lo.astype(np.float32)[..., None]) / s), 0, 15)
    return np.where(s > 0, q, 0).astype(np.uint8).reshape(x.shape), scale, lo


def values(codes, scale, lo):
    g = codes.reshape(codes.shape[:-1] + (-1, 64)).astype(np.float32)
    with np.errstate(all="ignore"):
        return (lo.astype(np.float32)[..., None] + scale.astype(np.float32)[..., None] * g).reshape(codes.shape)


def tile_bytes(D):
    return 16 * (D + D // 8)


def k_place(D):
    """Byte of a tile and nibble of K, [16, D]."""
    j, d = np.arange(16)[:, None], np.arange(D)
    return j * (D // 2) + d // 8 % 4 * (D // 8) + d // 32 * 4 + d % 2 * 2 + d % 8 // 4, np.broadcast_to(d // 2 % 2, (16, D))


def v_place(D):
    j, d = np.arange(16)[:, None], np.arange(D)
    return 8 * D + d // 64 * 512 + d % 8 * 64 + j % 8 // 2 * 16 + d // 16 % 4 * 4 + j % 2 * 2 + j // 8, np.broadcast_to(d // 8 % 2, (16, D))


class Cache:
    """A pool on the host: uint8 [pages, heads, page / 16, bytes]."""

    def __init__(self, n_pages, heads, D, page, rng=None):
        self.heads, self.D, self.page, self.n_pages = heads, D, page, n_pages
        shape = (n_pages, heads, page // 16, tile_bytes(D))
        self.pool = np.zeros(shape, np.uint8) if rng is None else rng.integers(0, 256, shape, dtype=np.uint8)

    def _parts(self, slot, which):
        tile = self.pool[slot // self.page, :, slot % self.page // 16]                    # [heads, bytes]
        j, D = slot % 16, self.D
        byte, high = (k_place if which == 0 else v_place)(D)
        pair = (16 + which) * D + j * (D // 16)
        return tile, byte[j], high[j], slice(pair, pair + D // 16)

    def write(self, slot, k, v):
        """k, v [heads, D]."""
        for which, x in enumerate((k, v)):
            tile, byte, high, pair = self._parts(slot, which)
            codes, scale, lo = quantise(x)
            for h in range(self.heads):
                keep = np.where(high == 1, 0x0f, 0xf0)
                for nib in (0, 1):
                    m = high == nib
                    tile[h, byte[m]] = (tile[h, byte[m]] & keep[m]) | (codes[h, m] << (4 * nib))
                tile[h, pair] = np.stack((scale[h], lo[h]), -1).reshape(-1).view(np.uint8)

    def read(self, slot):
        out = []
        for which in (0, 1):
            tile, byte, high, pair = self._parts(slot, which)
            codes = tile[:, byte] >> (4 * high) & 15
            pairs = np.ascontiguousarray(tile[:, pair]).view(np.float16).reshape(self.heads, -1, 2)
            out.append(values(codes, pairs[..., 0], pairs[..., 1]))
        return out

    def rows(self, slots):
        """f64 K and V [heads, len(slots), D]; NaN where there is no such slot."""
        k, v = (np.full((self.heads, len(slots), self.D), np.nan) for _ in range(2))
        for i, s in enumerate(slots):
            if 0 <= s < self.n_pages * self.page:
                k[:, i], v[:, i] = self.read(int(s))
        return k, v


def attend(q, k, v, seen, scale):
    """q [heads, D] of one row, k, v [kv heads, keys, D] f64, seen [keys] bool -> [heads, D] f64, and what tolerances count: the largest sum of |q||k|
    of a score, and of |v| that is seen."""
    H, G = k.shape[0], q.shape[0] // k.shape[0]
    out, S, V = np.zeros(q.shape), 0.0, 0.0
    if seen.any():
        for h in range(H):
            kk, vv, qq = k[h, seen], v[h, seen], q[h * G:(h + 1) * G].astype(np.float64)
            s = qq @ kk.T * scale
            w = np.exp(s - s.max(1, keepdims=True))
            out[h * G:(h + 1) * G] = w @ vv / w.sum(1, keepdims=True)
            S, V = max(S, float((np.abs(qq) @ np.abs(kk).T).max() * abs(scale))), max(V, float(np.abs(vv).max()))
    return out, S, V


class Pages:
    """The allocator, with lists."""

    def __init__(self, held, table, free, page):
        self.held, self.table, self.free, self.page = list(held), [list(r) for r in table], list(free), page

    def step(self, add, max_rows, n_pages):
        """(status, row_start, slots, row_seq, row_pos); does nothing where the status is not 0."""
        page, room = self.page, len(self.table[0]) * self.page
        n_rows = sum(max(0, a) for a in add)
        none = [-1] * max_rows
        pages = lambda n: -(-n // page)  # noqa: E731
        back = sum(pages(h) for h, a in zip(self.held, add) if a < 0)
        taken = sum(pages(h + a) - pages(h) for h, a in zip(self.held, add) if a > 0)
        status = 0
        if any(h < 0 or h > room for h in self.held) or len(self.free) + back > n_pages:
            status = _lib.PAGES_STATE
        elif any(h + a > room for h, a in zip(self.held, add) if a > 0):
            status = _lib.PAGES_TABLE
        elif n_rows > max_rows:
            status = _lib.PAGES_ROWS
        elif taken > len(self.free) + back:
            status = _lib.PAGES_EXHAUSTED
        if status:
            return status, [0] * (len(add) + 1), none, none, none
        for s, a in enumerate(add):
            if a < 0:
                self.free += self.table[s][:pages(self.held[s])]
                self.held[s] = 0
        start, slots, seqs, poss = [0], [], [], []
        for s, a in enumerate(add):
            for pos in range(self.held[s], self.held[s] + max(0, a)):
                if pos % page == 0:
                    self.table[s][pos // page] = self.free.pop()
                slots.append(self.table[s][pos // page] * page + pos % page)
                seqs.append(s)
                poss.append(pos)
            self.held[s] += max(0, a)
            start.append(len(slots))
        pad = [-1] * (max_rows - n_rows)
        return 0, start, slots + pad, seqs + pad, poss + pad


# ---- the library's calls -----------------------------------------------------------------------------------------------------
CODE = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def cache_arg(pool, n_pages, heads, D, page):
    return _lib.Kv4Cache(pool.data_ptr(), n_pages, heads, D, page)


def address(t):
    return None if t is None else t.data_ptr()


def write(cache, k, v, kind, slots, stream=None):
    from gpu_util import stream as current
    lib = _lib.load()
    _lib.check(lib.b200_kv4_write(C.byref(cache), address(k), k.stride(0), address(v), v.stride(0), CODE[kind], address(slots), slots.numel(),
                                  stream if stream is not None else current()))


def read(cache, k, v, kind, slots):
    from gpu_util import stream as current
    _lib.check(_lib.load().b200_kv4_read(C.byref(cache), address(k), k.stride(0), address(v), v.stride(0), CODE[kind], address(slots), slots.numel(), current()))


def workspace(q_heads, kv_heads, D):
    import torch
    return torch.zeros(_lib.load().b200_kv4_attention_workspace_bytes(q_heads, kv_heads, D), dtype=torch.uint8, device="cuda")


def attention(cache, q, out, kind, q_heads, row_start, lens, table, scale, ws, stream=None):
    from gpu_util import stream as current
    a = _lib.Kv4Attention(q=address(q), out=address(out), dtype=CODE[kind], q_heads=q_heads, q_ld=q.stride(0), out_ld=out.stride(0), rows=q.shape[0],
                          n_seqs=lens.numel(), row_start=address(row_start), lens=address(lens), block_table=address(table), table_stride=table.shape[1],
                          scale=scale)
    _lib.check(_lib.load().b200_kv4_attention(C.byref(cache), C.byref(a), address(ws), ws.numel(), stream if stream is not None else current()))


class Step:
    """Device arrays of b200_page_step."""

    def __init__(self, held, table, free, n_pages, page, max_rows, in_place=False):
        import torch
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        n = len(held)
        self.held, self.table, self.n_free = i32(held), i32(table).reshape(n, -1), i32([len(free)])
        self.free = i32(list(free) + [-7] * (n_pages - len(free)))
        self.held_out = self.held if in_place else i32([-9] * n)
        self.n_free_out = self.n_free if in_place else i32([-9])
        self.add, self.row_start, self.status = i32([0] * n), i32([-9] * (n + 1)), i32([-9])
        self.slots = torch.full((max_rows + 1,), -9, dtype=torch.int64, device="cuda")
        self.row_seq, self.row_pos = i32([-9] * (max_rows + 1)), i32([-9] * (max_rows + 1))
        self.args = _lib.PageStep(n_seqs=n, page=page, table_stride=self.table.shape[1], n_pages=n_pages, max_rows=max_rows,
                                  **{k: getattr(self, k).data_ptr() for k in ("held", "add", "held_out", "free", "n_free", "n_free_out", "row_start", "slots",
                                                                              "row_seq", "row_pos", "status") if k != "free"},
                                  block_table=self.table.data_ptr(), free_pages=self.free.data_ptr())

    def __call__(self, add=None, stream=None):
        import torch
        from gpu_util import stream as current
        if add is not None:
            self.add.copy_(torch.tensor(add, dtype=torch.int32))
        _lib.check(_lib.load().b200_page_step(C.byref(self.args), stream if stream is not None else current()))
