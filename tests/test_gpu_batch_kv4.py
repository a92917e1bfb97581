"""Batched decode over a cache held in 4 bits: every sequence against the model written out in f64 on that sequence alone, its keys and values
quantised as the cache has them; pages, order, limits."""
import numpy as np
import pytest

import kv4_util as u
from buddy_mlir_b200 import TINY_MEGA, TINY_QWEN2, TINY_QWEN3, _lib, synthetic
from buddy_mlir_b200.session import BatchSession, ModelSession

pytestmark = pytest.mark.gpu


class Plain:
    """A sequence of the model in f64; f32 weights, the cache as it is held."""

    def __init__(self, cfg, views):
        self.cfg, self.w, self.cache = cfg, {k: np.asarray(v, np.float64) for k, v in views.items()}, [([], []) for _ in range(cfg.n_layers)]

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg.eps) * w

    def rotate(self, x, pos):
        half = x.shape[-1] // 2
        th = self.w[("inv_freq", -1)].reshape(-1)[:half] * pos
        a, b = x[:, :half], x[:, half:]
        return np.concatenate([a * np.cos(th) - b * np.sin(th), b * np.cos(th) + a * np.sin(th)], -1)

    def step(self, token):
        c, w = self.cfg, self.w
        x = w[("embed", -1)].reshape(c.vocab, c.hidden)[token]
        for i in range(c.n_layers):
            h = self.norm(x, w[("in_norm", i)])
            q, k, v = (h @ w[(n, i)] + (w[(n + "_bias", i)] if c.qkv_bias else 0.0) for n in "qkv")
            q, k, v = q.reshape(c.q_heads, c.head_dim), k.reshape(c.kv_heads, c.head_dim), v.reshape(c.kv_heads, c.head_dim)
            if c.qk_norm:
                q, k = self.norm(q, w[("q_norm", i)]), self.norm(k, w[("k_norm", i)])
            keys, vals = self.cache[i]
            pos = len(keys)
            q, k = self.rotate(q, pos), self.rotate(k, pos)
            keys.append(u.values(*u.quantise(k)))
            vals.append(u.values(*u.quantise(v)))
            kk, vv = (np.stack(s, 1).astype(np.float64) for s in (keys, vals))
            o, _, _ = u.attend(q, kk, vv, np.ones(pos + 1, bool), c.head_dim ** -0.5)
            x = x + o.reshape(-1) @ w[("o", i)]
            h = self.norm(x, w[("post_norm", i)])
            g = h @ w[("gate", i)]
            x = x + (g / (1.0 + np.exp(-g)) * (h @ w[("up", i)])) @ w[("down", i)]
        return self.norm(x, w[("final_norm", -1)]) @ w[("lm_head", -1)]


def far(a, b):
    return float(np.abs(a - b).max() / np.abs(b).max())


# f32 passes are within 1e-3 of the model with an f32 cache (test_gpu_batch.py).  Here a value that lies within that rounding of the middle between two codes may
# take the other one: some 1e-5 of all values, a step in one dim of one key each, which a score sees as a few hundredths at most and a logit as a fraction of that
# over the number of keys.
FAR = 5e-3


@pytest.mark.parametrize("cfg", [TINY_QWEN2, TINY_QWEN3, TINY_MEGA])
def test_sequences_against_the_model_in_f64(cfg):
    _, views = synthetic.make_f32_blob(cfg, 71)
    s = ModelSession(cfg)
    s.load_tensors(views)
    page, n_pages = 16, 24
    bs = BatchSession(s, max_seqs=5, page_size=page, n_pages=n_pages, max_context=cfg.max_len, kv_bits=4)
    rng = np.random.default_rng(4)
    lengths = [3, 17, 32, 70, 1]
    plain, seqs, toks = [], [], []
    for n in lengths:
        m, prompt = Plain(cfg, views), rng.integers(0, cfg.vocab, n)
        for t in prompt:
            want = m.step(int(t))
        q = bs.add()
        got, nxt = bs.prefill(q, prompt)
        assert far(got, want) < FAR and nxt == int(np.argmax(got)) and bs.length(q) == n
        plain.append(m)
        seqs.append(q)
        toks.append(int(rng.integers(cfg.vocab)))
    used = lambda: sum(-(-bs.length(q) // page) for q in seqs)  # noqa: E731
    assert bs.free_pages() == n_pages - used()
    for step in range(16):      # over the ends of pages, in another order every time
        order = rng.permutation(len(seqs))
        logits, nxt = bs.decode([seqs[i] for i in order], [toks[i] for i in order])
        for r, i in enumerate(order):
            want = plain[i].step(toks[i])
            assert far(logits[r], want) < FAR, (step, i)
            assert int(nxt[r]) == int(np.argmax(logits[r]))
            toks[i] = int(rng.integers(cfg.vocab))
    assert bs.free_pages() == n_pages - used()
    # some only, without logits; then one ends, another takes its place and its pages
    _, nxt = bs.decode([seqs[3], seqs[0]], [toks[3], toks[0]], want_logits=False)
    for r, i in enumerate((3, 0)):
        assert int(nxt[r]) == int(np.argmax(plain[i].step(toks[i])))
    bs.remove(seqs[3])
    before = bs.free_pages()
    q = bs.add()
    assert q == seqs[3]
    m, prompt = Plain(cfg, views), rng.integers(0, cfg.vocab, 40)
    for t in prompt:
        want = m.step(int(t))
    got, _ = bs.prefill(q, prompt[:25])
    got, _ = bs.prefill(q, prompt[25:])
    assert far(got, want) < FAR and bs.free_pages() == before - 3
    plain[3] = m
    logits, _ = bs.decode(seqs, toks)
    for i in range(len(seqs)):
        assert far(logits[i], plain[i].step(toks[i])) < FAR
    bs.close()
    s.close()


def test_limits_are_reported_and_change_nothing():
    cfg = TINY_QWEN2
    _, views = synthetic.make_f32_blob(cfg, 72)
    s = ModelSession(cfg)
    s.load_tensors(views, quantize_to="w8")
    for bad in (dict(page_size=8), dict(page_size=24), dict(n_pages=0), dict(max_seqs=5000)):
        with pytest.raises(_lib.B200Error):
            BatchSession(s, **(dict(max_seqs=2, page_size=16, n_pages=4, max_context=48, kv_bits=4) | bad))
    with pytest.raises(ValueError):
        BatchSession(s, 2, 16, 4, 48, kv_bits=8)
    bs = BatchSession(s, max_seqs=2, page_size=16, n_pages=3, max_context=48, kv_bits=4)
    a, b = bs.add(), bs.add()
    rng = np.random.default_rng(1)
    first = rng.integers(0, cfg.vocab, 31)
    bs.prefill(a, first)
    for tokens in (rng.integers(0, cfg.vocab, 17), ):
        with pytest.raises(_lib.B200Error, match="exhausted"):
            bs.prefill(b, tokens)
    with pytest.raises(_lib.B200Error, match="context limit"):
        bs.prefill(a, rng.integers(0, cfg.vocab, 18))
    bs.prefill(b, first[:16])
    assert bs.free_pages() == 0
    with pytest.raises(_lib.B200Error, match="exhausted"):
        bs.decode([b, a], [1, 2])                      # b has no page left; a would have room
    assert bs.length(a) == 31 and bs.length(b) == 16
    got, _ = bs.decode([a], [5])
    other = BatchSession(s, max_seqs=1, page_size=16, n_pages=3, max_context=48, kv_bits=4)
    q = other.add()
    other.prefill(q, first)
    want, _ = other.decode([q], [5])
    assert np.array_equal(got, want)                   # what was refused left no trace
    other.close()
    bs.close()
    s.close()
