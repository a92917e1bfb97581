"""The operators of a KV cache held in 4 bits, case by case: their inputs, one pass, what a pass cannot do without, and their values in 64 bits.

A cache is a pool of pages.  A page holds `page` positions of every kv head; sixteen positions of a head are a tile of 16 * (D + D / 8) bytes: codes of K,
codes of V, (scale, minimum) pairs of K, those of V.  A position's K (and V) is cut into groups of 64 dims: minimum lo and scale s are rounded to f16, a
value is lo + s * code.  The operators: `tables` (b200_page_step: pages, slots and row maps from lengths), `write` (b200_kv4_write, and b200_kv4_read of what was
written), `attend` (b200_kv4_attention), and `serve`, the three in a row as a serving step has them.

Head layouts are those of this repository's configurations: 12 heads on 2 and 32 on 8 with 128 dims, 4 on 2 and others with 64.
"""
import math

import torch

own = False

GROUP = 64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of two dozen requests: every one grows by a token, a few have ended
        {"name": "tables_24", "op": "tables", "seqs": 24, "longest": 700, "prompt": 1, "page": 16},
        # a busy server's step: two thousand requests, most of them decoding, some with new prompts, some ended
        {"name": "tables_2000", "op": "tables", "seqs": 2000, "longest": 2000, "prompt": 500, "page": 64},
        # the new rows of a decode step
        {"name": "write_24", "op": "write", "rows": 24, "kv_heads": 2, "D": 128, "page": 16, "type": "f32", "prompt": False},
        # prompts on their way into the cache
        {"name": "write_16001", "op": "write", "rows": 16001, "kv_heads": 8, "D": 128, "page": 64, "type": "bf16", "prompt": True},
        # one request, a few tokens into it: nothing but latency
        {"name": "attend_first", "op": "attend", "seqs": 1, "shortest": 17, "longest": 17, "rows": 1, "q_heads": 12, "kv_heads": 2, "D": 128, "page": 16, "type": "f32"},
        # a decode step of two dozen requests of different lengths, f32 activations as the sessions have them
        {"name": "attend_24", "op": "attend", "seqs": 24, "shortest": 32, "longest": 700, "rows": 1, "q_heads": 12, "kv_heads": 2, "D": 128, "page": 16, "type": "f32"},
        # the same with many long requests: the cache's bytes are what counts
        {"name": "attend_64_4k", "op": "attend", "seqs": 64, "shortest": 2000, "longest": 4096, "rows": 1, "q_heads": 32, "kv_heads": 8, "D": 128, "page": 64, "type": "bf16"},
        # two very long documents
        {"name": "attend_2_100k", "op": "attend", "seqs": 2, "shortest": 90000, "longest": 100001, "rows": 1, "q_heads": 32, "kv_heads": 8, "D": 128, "page": 32, "type": "f16"},
        # five drafted tokens of each request are checked at once, small heads
        {"name": "attend_draft", "op": "attend", "seqs": 40, "shortest": 5, "longest": 2000, "rows": 5, "q_heads": 16, "kv_heads": 4, "D": 64, "page": 16, "type": "bf16"},
        # a chunk of a prompt behind what the cache holds of it
        {"name": "attend_chunk", "op": "attend", "seqs": 1, "shortest": 4000, "longest": 4000, "rows": 1001, "q_heads": 32, "kv_heads": 8, "D": 128, "page": 64, "type": "bf16"},
        # a session's prompt, f32, from its first token on
        {"name": "attend_prompt_f32", "op": "attend", "seqs": 1, "shortest": 1000, "longest": 1000, "rows": 1000, "q_heads": 12, "kv_heads": 2, "D": 128, "page": 16, "type": "f32"},
        # a whole step of many short requests, rows padded to what a captured graph holds
        {"name": "serve_200", "op": "serve", "seqs": 200, "shortest": 1, "longest": 600, "pad": 56, "q_heads": 32, "kv_heads": 8, "D": 128, "page": 16, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "write", "attend", "attend", "attend", "serve"])
    page, D, kind = rng.choice([16, 32, 48, 64, 128]), rng.choice([64, 128, 128]), rng.choice(["f32", "f16", "bf16"])
    if op == "tables":
        return {"op": op, "seqs": _log(rng, 1, 2000), "longest": _log(rng, 16, 2000), "prompt": _log(rng, 1, 500), "page": page}
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "write":
        return {"op": op, "rows": _log(rng, 1, 16001), "kv_heads": kv_heads, "D": D, "page": page, "type": kind, "prompt": rng.random() < 0.6}
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8] if kv_heads < 8 else [1, 2, 4])
    heads = {"q_heads": q_heads, "kv_heads": kv_heads, "D": D, "page": page, "type": kind}
    if op == "serve":
        return {"op": op, "seqs": _log(rng, 1, 200), "shortest": 1, "longest": _log(rng, 2, 2000), "pad": rng.choice([0, 0, rng.randint(1, 64)]), **heads}
    rows = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1001)])
    seqs = _log(rng, 1, 64 if rows < 9 else 2)
    # no dearer than the largest listed cases: keys of all sequences, and keys times rows
    most = max(2, min(100001, 200000 * 8 // (seqs * kv_heads), 128_000_000 // (seqs * q_heads * rows)))
    longest = min(most, max(rows, _log(rng, 2, 100001)))
    return {"op": op, "seqs": seqs, "shortest": rng.randint(1, longest), "longest": longest, "rows": rows, **heads}


# ---- the format, in elementary operations ----------------------------------------------------------------------------------
def _quantise(x):
    """[..., D] of any type -> codes (uint8), scale and minimum (f16) of [..., D / 64]: every step rounded to f32, what is stored to f16."""
    x = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, GROUP))
    lo = x.amin(-1).half()
    scale = ((x.amax(-1) - lo.float()) / torch.full_like(lo, 15.0, dtype=torch.float32)).half()
    q = (x - lo.float().unsqueeze(-1)) / scale.float().unsqueeze(-1)
    codes = torch.where(scale.unsqueeze(-1) > 0, q.round().clamp(0.0, 15.0), torch.zeros_like(q)).to(torch.uint8)
    return codes.flatten(-2), scale, lo


def _values(codes, scale, lo):
    """The f32 values that codes stand for."""
    return (lo.float().unsqueeze(-1) + scale.float().unsqueeze(-1) * codes.unflatten(-1, (-1, GROUP)).float()).flatten(-2)


def _k_bytes(c):
    """Codes [..., 16, D] of a tile -> [..., 16, D / 2]: a position's dim is 32 i + 8 t + 4 a + 2 b + h; byte [t][i][h][a] holds b = 0 and 1."""
    c = c.unflatten(-1, (-1, 4, 2, 2, 2))
    return (c[..., 0, :] | c[..., 1, :] << 4).movedim((-4, -3, -1, -2), (-3, -4, -2, -1)).flatten(-4)


def _k_codes(b):
    D = 2 * b.shape[-1]
    b = b.unflatten(-1, (4, D // 32, 2, 2)).movedim((-3, -4, -1, -2), (-4, -3, -2, -1))
    return torch.stack((b & 15, b >> 4), -2).flatten(-5)


def _v_bytes(c):
    """Codes [..., 16, D] of a tile -> [..., 8 D]: position 8 u + 2 t + h, dim 64 j + 16 i + 8 w + g; byte [j][g][t][i][h][u] holds w = 0 and 1."""
    c = c.unflatten(-1, (-1, 4, 2, 8)).unflatten(-5, (2, 4, 2))          # u t h j i w g
    b = c[..., 0, :] | c[..., 1, :] << 4                                 # u t h j i g
    return b.movedim((-3, -1, -5, -2, -4, -6), (-6, -5, -4, -3, -2, -1)).flatten(-6)


def _v_codes(b):
    D = b.shape[-1] // 8
    b = b.unflatten(-1, (D // 64, 8, 4, 4, 2, 2)).movedim((-6, -5, -4, -3, -2, -1), (-3, -1, -5, -2, -4, -6))
    return torch.stack((b & 15, b >> 4), -2).flatten(-4).flatten(-4, -2)


def _tile_bytes(D):
    return 16 * (D + D // 8)


def _pack(k, v):
    """K and V rows [..., 16, D] -> tiles [..., 16 (D + D / 8)] of bytes."""
    (kc, ks, kl), (vc, vs, vl) = _quantise(k), _quantise(v)
    pairs = [torch.stack(p, -1).contiguous().view(torch.uint8).flatten(-3) for p in ((ks, kl), (vs, vl))]
    return torch.cat([_k_bytes(kc).flatten(-2), _v_bytes(vc)] + pairs, -1)


def _parts(tiles, D):
    kb, vb, kp, vp = tiles.split([8 * D, 8 * D, D, D], -1)
    pairs = [p.contiguous().view(torch.float16).unflatten(-1, (16, D // GROUP, 2)).unbind(-1) for p in (kp, vp)]
    return (_k_codes(kb.unflatten(-1, (16, D // 2))),) + tuple(pairs[0]), (_v_codes(vb),) + tuple(pairs[1])


def _unpack(tiles, D):
    """Tiles [..., bytes] -> f32 values of K and V, [..., 16, D] each."""
    k, v = _parts(tiles, D)
    return _values(*k), _values(*v)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.empty(*shape, device="cuda").normal_(0.0, 1.0, generator=gen)


def _randint(gen, lo, hi, *shape):
    return torch.randint(lo, hi, shape, device="cuda", generator=gen, dtype=torch.int32)


def _rows(gen, *shape):
    """Rows of K or V as projections leave them: channels of different width, a few of them far out, an offset each."""
    D = shape[-1]
    width = torch.exp(0.5 * _randn(gen, D)) * torch.where(torch.rand(D, device="cuda", generator=gen) < 0.03, 6.0, 1.0)
    return _randn(gen, *shape) * width + 0.5 * _randn(gen, D)


def _ceil(a, b):
    return -(-a // b)


def _lengths(gen, case):
    """Of every sequence, with its new rows: the longest of them first."""
    n = _randint(gen, case["shortest"], case["longest"] + 1, case["seqs"])
    n[0] = case["longest"]
    return n.clamp_min(case.get("rows", 1))


def _pages(gen, lens, page, stride, n_pages):
    """A block table whose pages lie anywhere in the pool, the stack of the free ones, in any order, and how many there are."""
    need = _ceil(lens.long(), page)
    used = int(need.sum())
    order = torch.randperm(n_pages, device="cuda", generator=gen).int()
    table = torch.full((lens.numel(), stride), -1, device="cuda", dtype=torch.int32)
    table[torch.arange(stride, device="cuda") < need.unsqueeze(1)] = order[:used]
    return table, torch.cat([order[used:], torch.full_like(order[:used], -1)]), torch.tensor([n_pages - used], device="cuda", dtype=torch.int32)


def _pool(gen, n_pages, case):
    """A cache that other requests have filled."""
    H, D, page = case["kv_heads"], case["D"], case["page"]
    return _pack(_rows(gen, n_pages, H, page // 16, 16, D), _rows(gen, n_pages, H, page // 16, 16, D))


def prepare(case, seed):
    gen, op, s = _gen(seed), case["op"], dict(case)
    page = case["page"]
    if op == "tables":
        n, prompts = case["seqs"], _ceil(case["seqs"], 10)
        s["held"] = _randint(gen, 0, case["longest"] + 1, n)
        who = torch.randperm(n, device="cuda", generator=gen)
        s["add"] = torch.ones_like(s["held"])
        s["add"][who[:prompts]] = _randint(gen, 1, case["prompt"] + 1, prompts)
        s["add"][who[prompts:prompts + n // 20]] = -1                    # (requests that have ended)
        s["add"][who[prompts + n // 20:prompts + n // 10]] = 0           # (requests that wait)
        s["n_pages"] = n * (_ceil(case["longest"], page) + 1) + prompts * _ceil(case["prompt"], page)
        s["table"], s["free"], s["n_free"] = _pages(gen, s["held"], page, _ceil(case["longest"] + case["prompt"], page), s["n_pages"])
        s["cap"] = n + prompts * case["prompt"]                          # what a captured graph has room for
        return s | _table_outputs(s)
    if op == "write":
        H, D, rows = case["kv_heads"], case["D"], case["rows"]
        # slots of prompts of some hundred tokens, each behind what its page holds, or one row of a page of its own for every request
        first = _randint(gen, 1, page, rows) if not case["prompt"] else torch.arange(rows, device="cuda") + 5
        need = rows if not case["prompt"] else _ceil(rows + 5, page)
        ids = torch.randperm(need + 3, device="cuda", generator=gen)
        at = ids[torch.arange(rows, device="cuda") if not case["prompt"] else first // page]
        s["n_pages"], s["slots"] = need + 3, at.long() * page + first.long() % page
        s["pool"] = _pool(gen, need + 3, case)
        fused = torch.cat([_rows(gen, rows, H * D).to(TYPES[case["type"]]) for _ in range(3)], 1)    # q | k | v of a projection
        s["k"], s["v"] = fused[:, H * D:2 * H * D], fused[:, 2 * H * D:]
        s["back"] = torch.empty(2, rows, H * D, device="cuda")
        return s
    H, D, QH, dt = case["kv_heads"], case["D"], case["q_heads"], TYPES[case["type"]]
    lens = _lengths(gen, case)
    if op == "attend":
        n_rows = case["rows"] * case["seqs"]
        s["lens"], s["max_rows"] = lens, case["rows"]
        s["row_start"] = torch.arange(case["seqs"] + 1, device="cuda", dtype=torch.int32) * case["rows"]
        s["n_pages"] = int(_ceil(lens, page).sum()) + 3
        s["table"], _, _ = _pages(gen, lens, page, _ceil(case["longest"], page), s["n_pages"])
    else:
        n_rows = case["seqs"] + case["pad"]
        s["held"], s["add"], s["max_rows"], s["cap"] = lens - 1, torch.ones_like(lens), 1, n_rows
        s["add"][3::40] = 0                                              # (requests that wait)
        s["n_pages"] = case["seqs"] * _ceil(case["longest"], page)
        s["table"], s["free"], s["n_free"] = _pages(gen, s["held"], page, _ceil(case["longest"], page), s["n_pages"])
        s |= _table_outputs(s)
    s["pool"] = _pool(gen, s["n_pages"], case)
    width = 0.35 * torch.exp(0.3 * _randn(gen, D))
    fused = torch.cat([(_randn(gen, n_rows, QH, D) * width).flatten(1), _rows(gen, n_rows, H, D).flatten(1), _rows(gen, n_rows, H, D).flatten(1)], 1).to(dt)
    s["q"], s["k"], s["v"] = fused.split([QH * D, H * D, H * D], 1)
    s["out"] = torch.empty(n_rows, QH * D, device="cuda", dtype=dt)
    s["scale"] = 1.0 / math.sqrt(D)
    return s


def _table_outputs(s):
    """What a program keeps for the step's answers: buffers of a captured graph."""
    n, new = s["held"].numel(), lambda k, t=torch.int32: torch.empty(k, device="cuda", dtype=t)  # noqa: E731
    return {"held_out": new(n), "n_free_out": new(1), "row_start": new(n + 1), "slots": new(s["cap"], torch.int64), "row_seq": new(s["cap"]),
            "row_pos": new(s["cap"]), "status": new(1)}


# ---- one pass: the plain form ------------------------------------------------------------------------------------------------
def _plain_tables(s):
    page, n, cap, stride = s["page"], s["held"].numel(), s["cap"], s["table"].shape[1]
    held, add, n_free = s["held"].long(), s["add"].long(), s["n_free"].long()
    ends, grow = add < 0, add.clamp_min(0)
    have = _ceil(held, page)
    after = torch.where(ends, 0, held + grow)
    need = torch.where(ends, 0, _ceil(after, page) - have)
    given = torch.where(ends, have, 0)
    upto, need_to, given_to = grow.cumsum(0), need.cumsum(0), given.cumsum(0)
    total, taken, back = upto[-1], need_to[-1], given_to[-1]
    over = (after > stride * page).any()
    status = torch.where(over, 2, torch.where(total > cap, 3, torch.where(taken > n_free[0] + back, 1, 0)))
    ok = status == 0
    # the stack with the returned pages on top
    i = torch.arange(s["free"].numel(), device="cuda") - n_free
    who = torch.searchsorted(given_to, i.clamp_min(0), right=True).clamp_max(n - 1)
    returned = s["table"][who, (i - (given_to - given)[who]).clamp(0, stride - 1)]
    stack = torch.where((i >= 0) & (i < back), returned, s["free"])
    left = n_free + back - taken
    # new entries of the table: from the top of the stack down, sequence by sequence
    j = torch.arange(stride, device="cuda")
    new = (j >= have.unsqueeze(1)) & (j < (have + need).unsqueeze(1)) & ok
    place = n_free + back - 1 - ((need_to - need).unsqueeze(1) + j - have.unsqueeze(1))
    s["table"].copy_(torch.where(new, stack[place.clamp(0, stack.numel() - 1)], s["table"]))
    at = torch.arange(stack.numel(), device="cuda")
    s["free"].copy_(torch.where((at >= n_free) & (at < left) & ok, stack, s["free"]))
    r = torch.arange(cap, device="cuda")
    live = (r < total) & ok
    seq = torch.searchsorted(upto, r, right=True).clamp_max(n - 1)
    pos = held[seq] + r - (upto - grow)[seq]
    slot = s["table"][seq, (pos // page).clamp(0, stride - 1)].long() * page + pos % page
    s["slots"].copy_(torch.where(live, slot, -1))
    s["row_seq"].copy_(torch.where(live, seq, -1))
    s["row_pos"].copy_(torch.where(live, pos, -1))
    s["row_start"][0] = 0
    s["row_start"][1:].copy_(torch.where(ok, upto, 0))
    s["held_out"].copy_(torch.where(ok, after, held))
    s["n_free_out"].copy_(torch.where(ok, left, n_free))
    s["status"].copy_(status)


TABLE_OUTPUTS = ("held_out", "table", "free", "n_free_out", "row_start", "slots", "row_seq", "row_pos", "status")


def _codes_at(s, slots):
    """Where the codes and pairs of rows lie: tile numbers [rows, kv heads] and the position in the tile."""
    page, H = s["page"], s["kv_heads"]
    head = torch.arange(H, device="cuda")
    tile = ((slots // page).unsqueeze(1) * H + head) * (page // 16) + (slots % page // 16).unsqueeze(1)
    return tile, slots % 16


def _plain_write(s, slots):
    """Rows that have a slot into their tiles, byte by byte; what else a tile holds stays."""
    H, D = s["kv_heads"], s["D"]
    flat = s["pool"].view(-1)
    tile, j = _codes_at(s, slots.clamp_min(0))
    (kc, ks, kl), (vc, vs, vl) = (_quantise(x.unflatten(1, (H, D))) for x in (s["k"], s["v"]))
    base = tile.unsqueeze(-1) * _tile_bytes(D)                                         # [rows, H, 1]
    j = j.view(-1, 1, 1)
    b = torch.arange(D // 2, device="cuda")
    kb = _k_bytes(kc)
    places = [base + j * (D // 2) + b]
    # of V: a byte for dims 16 i + g and 16 i + 8 + g
    i, g = torch.arange(D // 16, device="cuda").view(-1, 1), torch.arange(8, device="cuda")
    pair = (i // 4 * 512 + g * 64 + i % 4 * 4).flatten()
    v2 = vc.unflatten(-1, (-1, 2, 8))
    vb = (v2[..., 0, :] | v2[..., 1, :] << 4).flatten(-2)                              # [rows, H, D / 2]
    places.append(base + 8 * D + pair + j % 8 // 2 * 16 + j % 2 * 2 + j // 8)
    pairs = [torch.stack(p, -1).contiguous().view(torch.uint8).flatten(-2) for p in ((ks, kl), (vs, vl))]
    p = torch.arange(D // 16, device="cuda")
    places += [base + 16 * D + j * (D // 16) + p, base + 17 * D + j * (D // 16) + p]
    at, new = torch.cat(places, -1), torch.cat([kb, vb] + pairs, -1)
    # a row without a slot writes what the first row writes (which has one)
    row = torch.where(slots < 0, 0, torch.arange(slots.numel(), device="cuda"))
    flat.scatter_(0, at[row].flatten(), new[row].flatten())


def _plain_read(s, slots):
    """f32 values of K and V of rows, [rows, kv heads * D] each."""
    D = s["D"]
    tile, j = _codes_at(s, slots)
    k, v = _unpack(s["pool"].view(-1, _tile_bytes(D))[tile], D)                         # [rows, H, 16, D]
    at = j.view(-1, 1, 1, 1).expand(-1, k.shape[1], 1, D)
    return torch.stack([x.gather(2, at).flatten(1) for x in (k, v)])


def _plain_attend(s, lens, row_start):
    """Sequences side by side, padded to the longest and to the most rows."""
    H, D, page = s["kv_heads"], s["D"], s["page"]
    n, most, G = lens.numel(), s["max_rows"], s["q_heads"] // s["kv_heads"]
    pages = _ceil(s["longest"], page)
    k, v = _unpack(s["pool"][s["table"][:, :pages].clamp_min(0).long()], D)              # [n, pages, H, page / 16, 16, D]
    k, v = (x.transpose(1, 2).flatten(2, 4) for x in (k, v))                             # [n, H, keys, D]
    count = (row_start[1:] - row_start[:-1]).long()
    i = torch.arange(most, device="cuda")
    live = i < count.unsqueeze(1)                                                        # [n, most]
    row = (row_start[:-1].long().unsqueeze(1) + i).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[row].unflatten(-1, (H, G, D)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [n, H, most * G, D]
    pos = (lens.long() - count).unsqueeze(1) + i
    seen = torch.arange(k.shape[2], device="cuda") <= pos.unsqueeze(-1)                  # [n, most, keys]
    seen = seen.repeat_interleave(G, 1, output_size=most * G).unsqueeze(1)
    w = (q @ k.transpose(-1, -2)).mul_(s["scale"]).masked_fill_(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    v = v.masked_fill(~seen.any(2).unsqueeze(-1), 0.0)
    o = (w.double() @ v.double()).float() if s["type"] == "f32" and s["longest"] > 1000 else w @ v      # (long sums)
    o = (o / torch.where(total == 0, 1.0, total)).unflatten(2, (most, G)).permute(0, 2, 1, 3, 4).flatten(2)                      # [n, most, q heads * D]
    wide = torch.zeros(s["out"].shape[0] + 1, s["out"].shape[1], device="cuda")
    wide.index_copy_(0, torch.where(live, row, s["out"].shape[0]).flatten(), o.flatten(0, 1))
    s["out"].copy_(wide[:-1])


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def _calls(s):
    """The argument blocks of the framework's calls: a program fills them once for its buffers."""
    if "calls" not in s:
        import ctypes as C
        from buddy_mlir_b200 import _lib
        lib, ptr = _lib.load(), lambda name: s[name].data_ptr()  # noqa: E731
        c = {"lib": lib, "check": _lib.check, "ref": C.byref, "stream": lambda: C.c_void_p(torch.cuda.current_stream().cuda_stream)}
        if s["op"] in ("tables", "serve"):
            c["step"] = _lib.PageStep(
                n_seqs=s["held"].numel(), page=s["page"], table_stride=s["table"].shape[1], n_pages=s["n_pages"], max_rows=s["cap"], held=ptr("held"),
                add=ptr("add"), held_out=ptr("held_out"), block_table=ptr("table"), free_pages=ptr("free"), n_free=ptr("n_free"), n_free_out=ptr("n_free_out"),
                row_start=ptr("row_start"), slots=ptr("slots"), row_seq=ptr("row_seq"), row_pos=ptr("row_pos"), status=ptr("status"))
        if s["op"] != "tables":
            c["cache"] = _lib.Kv4Cache(pool=ptr("pool"), n_pages=s["n_pages"], kv_heads=s["kv_heads"], head_dim=s["D"], page=s["page"])
            c["type"] = {"f32": _lib.F32, "f16": _lib.F16, "bf16": _lib.BF16}[s["type"]]
        if s["op"] in ("attend", "serve"):
            s["seq_lens"] = s["lens"] if s["op"] == "attend" else s["held_out"]
            c["attend"] = _lib.Kv4Attention(
                q=ptr("q"), out=ptr("out"), dtype=c["type"], q_heads=s["q_heads"], q_ld=s["q"].stride(0), out_ld=s["out"].stride(0), rows=s["q"].shape[0],
                n_seqs=s["seq_lens"].numel(), row_start=ptr("row_start"), lens=ptr("seq_lens"), block_table=ptr("table"), table_stride=s["table"].shape[1],
                scale=s["scale"])
            c["bytes"] = lib.b200_kv4_attention_workspace_bytes(s["q_heads"], s["kv_heads"], s["D"])
            s["workspace"] = torch.zeros(c["bytes"], dtype=torch.uint8, device="cuda")
        s["calls"] = c
    return s["calls"]


def _write(s):
    if own:
        c = _calls(s)
        c["check"](c["lib"].b200_kv4_write(c["ref"](c["cache"]), s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0), c["type"],
                                           s["slots"].data_ptr(), s["slots"].numel(), c["stream"]()))
    else:
        _plain_write(s, s["slots"])


def _tables(s):
    if own:
        c = _calls(s)
        c["check"](c["lib"].b200_page_step(c["ref"](c["step"]), c["stream"]()))
    else:
        _plain_tables(s)


def _attend(s):
    if own:
        c = _calls(s)
        c["check"](c["lib"].b200_kv4_attention(c["ref"](c["cache"]), c["ref"](c["attend"]), s["workspace"].data_ptr(), c["bytes"], c["stream"]()))
    else:
        _plain_attend(s, s["lens"] if s["op"] == "attend" else s["held_out"], s["row_start"])


def _read(s):
    if own:
        c = _calls(s)
        k, v = s["back"]
        c["check"](c["lib"].b200_kv4_read(c["ref"](c["cache"]), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), 0, s["slots"].data_ptr(),
                                          s["slots"].numel(), c["stream"]()))
    else:
        s["back"].copy_(_plain_read(s, s["slots"]))


def run(s):
    if s["op"] == "tables":
        _tables(s)
        return {k: s[k] for k in TABLE_OUTPUTS}
    if s["op"] == "write":
        _write(s)
        _read(s)
        return s["back"]
    if s["op"] == "attend":
        _attend(s)
        return s["out"]
    _tables(s)
    _write(s)
    _attend(s)
    return {"out": s["out"]} | {k: s[k] for k in TABLE_OUTPUTS}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def _row_bytes(case):
    """Of a position's K and V, all kv heads, in the cache."""
    return case["kv_heads"] * 2 * (case["D"] // 2 + case["D"] // 16)


def work(case):
    op = case["op"]
    if op == "tables":
        n, prompts = case["seqs"], _ceil(case["seqs"], 10)
        rows = n - prompts - n // 20 * 2 + prompts * (1 + case["prompt"]) / 2
        return {"bytes": 16 * n + 16 * (n + prompts * case["prompt"]) + 8 * rows / case["page"], "flops": 0}
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if op == "write":
        values = 2 * case["rows"] * case["kv_heads"] * case["D"]
        return {"bytes": values * (size + 4) + 2 * case["rows"] * _row_bytes(case) + 8 * case["rows"], "flops": 0}
    rows, low = case.get("rows", 1), max(case["shortest"], case.get("rows", 1))
    keys = case["longest"] + (case["seqs"] - 1) * (low + max(low, case["longest"])) / 2          # of all sequences, as they are drawn
    seen = rows * keys - case["seqs"] * rows * (rows - 1) / 2
    out = {"bytes": keys * _row_bytes(case) + 2 * size * case["seqs"] * rows * case["q_heads"] * case["D"], "flops": 4 * case["q_heads"] * case["D"] * seen}
    if op == "serve":
        out["bytes"] += case["seqs"] * (36 + 2 * size * case["kv_heads"] * case["D"])
    return out


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------------------
def _exact_group(x):
    """The values that a group of numbers is held as: what the format rounds is rounded, to the type that it names."""
    x = x.double().clamp(-65504.0, 65504.0)
    shape = x.shape
    x = x.reshape(-1, GROUP)
    lo = x.min(1).values.half().double()
    scale = ((x.max(1).values - lo).float().double() / 15.0).float().half().double()
    steps = ((x - lo[:, None]).float().double() / torch.where(scale == 0, 1.0, scale)[:, None]).float().double()
    steps = torch.where(scale[:, None] == 0, 0.0, torch.round(steps)).clamp(0, 15)
    return (lo[:, None] + scale[:, None] * steps).reshape(shape)


def _exact_rows(tiles, byte, high, pair, D):
    """f64 values of tiles [.., n, bytes] as rows [.., 16 n, D]: the nibble of each position and dim (byte, high), its pair (from byte `pair` on)."""
    j, d = torch.arange(16, device=tiles.device).view(16, 1), torch.arange(D, device=tiles.device)
    at = (pair + (j * (D // GROUP) + d // GROUP) * 4).unsqueeze(-1)
    code = (tiles[..., byte.flatten()].unflatten(-1, (16, D)).long() >> (4 * high)) & 15
    scale, lo = (tiles[..., (at + torch.tensor(o, device=tiles.device)).flatten()].view(torch.float16).unflatten(-1, (16, D)).double() for o in ((0, 1), (2, 3)))
    return (lo + scale * code).flatten(-3, -2)


def _exact_keys(tiles, D):
    """K and V in f64, from the format's map written out."""
    j, d = torch.arange(16, device=tiles.device).view(16, 1), torch.arange(D, device=tiles.device)
    k_byte = j * (D // 2) + d // 8 % 4 * (D // 8) + d // 32 * 4 + d % 2 * 2 + d % 8 // 4
    v_byte = 8 * D + d // 64 * 512 + d % 8 * 64 + j % 8 // 2 * 16 + d // 16 % 4 * 4 + j % 2 * 2 + j // 8
    return _exact_rows(tiles, k_byte, d % 4 // 2, 16 * D, D), _exact_rows(tiles, v_byte, d % 16 // 8, 17 * D, D)


def _exact_sequence(pool, pages, q, first, scale, new=None):
    """Rows q [rows, q heads, D] at positions first, first + 1, ..: their outputs in f64.  new: K and V of the last position [kv heads, D], not in the pool yet."""
    H, (rows, heads, D) = pool.shape[1], q.shape
    k, v = (x[:, :first + rows].clone() for x in _exact_keys(pool[pages].transpose(0, 1).flatten(1, 2), D))      # [H, keys, D]
    if new is not None:
        k[:, -1], v[:, -1] = _exact_group(new[0]), _exact_group(new[1])
    hidden = torch.arange(first + rows, device=q.device) > first + torch.arange(rows, device=q.device).repeat_interleave(heads // H).unsqueeze(1)
    w = q.double().unflatten(1, (H, heads // H)).transpose(0, 1).flatten(1, 2) @ k.transpose(1, 2) * scale
    return (torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v).unflatten(1, (rows, heads // H)).transpose(0, 1).flatten(1)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "tables":
        return None
    H, D, page = case["kv_heads"], case["D"], case["page"]
    if op == "write":
        return torch.stack([_exact_group(x.unflatten(1, (H, D))).flatten(1) for x in (s["k"], s["v"])])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    grow = s["add"].tolist() if op == "serve" else [case["rows"]] * case["seqs"]
    ends = [h + a for h, a in zip(s["held"].tolist(), grow)] if op == "serve" else s["lens"].tolist()
    at = 0
    free = s["free"][:int(s["n_free"])].tolist() if op == "serve" else []
    for i, (n, end) in enumerate(zip(grow, ends)):
        if n == 0:
            continue
        pages = [p for p in s["table"][i].tolist() if p >= 0]
        new = None
        if op == "serve":
            while len(pages) * page < end:
                pages.append(free.pop())
            new = [x[at].unflatten(0, (H, D)) for x in (s["k"], s["v"])]
        q = s["q"][at:at + n].unflatten(1, (case["q_heads"], D))
        out[at:at + n] = _exact_sequence(s["pool"], torch.tensor(pages[:_ceil(end, page)], device="cuda"), q, end - n, s["scale"], new)
        at += n
    return out if op == "attend" else {"out": out} | {k: None for k in TABLE_OUTPUTS}
