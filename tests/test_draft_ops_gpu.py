"""Drafted tokens over a cache on the GPU: the 8-bit K/V cache, tree attention
and RoPE on several axes against plain formulas in 64 bits.

Tolerances count roundings (u = 2^-24 for f32, 2^-11 for f16, at most half a
step each):

* the 8-bit cache: scales and codes are decided exactly, so values read back
  are equal (f16: the RNE of them);
* RoPE: two products and a sum of them, 2 u (|x0 c| + |x1 s|);
* attention, per element: a score's dh products and sums are off by (dh + 4)
  u sum |q_d k_d| scale, its exponent by 4 u max|s| more and the exponential
  by 4 u, so a weight by twice their sum (its own, and the total's); the
  weighted sum and the total add n u each; f16 results half a step, weights
  held in f16 (f16 caches, f16 activations) half a step of each, 2^-11; 8-bit
  caches with f16 activations 2^-15 for weights of 16 bits."""

import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
LOG2E = 1.4426950408889634


# ------------------------------------------------------------ 8-bit cache


def stands_for(x):
    """What rows x [.., dh] (f32 or f16 values) are in the cache, in f64."""
    x = np.asarray(x, dtype=np.float64)
    top = np.abs(x).max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        least = np.maximum(top / 127.0, 2.0 ** -100)
        m, e = np.frexp(least)
        s = np.ldexp(np.ceil(m * 256.0) / 256.0, e)
        v = s * np.rint(x / s)
    return np.where(np.isfinite(x).all(-1, keepdims=True), v, np.nan)


def rows_of(rng, n, width, kind):
    x = rng.standard_normal((n, width)) * np.exp(2 * rng.standard_normal((n, 1)))
    if kind == "ties":  # values on the halves of a step: the scale is exactly 2^-3
        x = rng.integers(-253, 254, (n, width)) / 16.0
        x[:, ::64] = 127.0 / 8.0
    if kind == "edges":
        x[0::5] = 0.0
        x[1::5] *= 1e-38
        x[2::5] *= 1e30
        x[3::5, 1::2] *= 1e-6
    return x.astype(np.float32)


def read_back(ta, ex, cache, f16, positions, first=0, t_dst=None):
    t = t_dst or cache.t_max
    kt = ex.tensor_from(np.full((cache.kv_heads, cache.head_dim, t), 7.0, np.float32), f16=f16)
    v = ex.tensor_from(np.full((cache.kv_heads, t, cache.head_dim), 7.0, np.float32), f16=f16)
    ex.q8_cache_read(cache, kt, v, ta.Q8ReadDesc(positions, first))
    return ex.download(kt), ex.download(v)


def same(got, ref, f16):
    ref = ref.astype(np.float16) if f16 else ref.astype(np.float32)
    return np.array_equal(np.asarray(got, np.float32), ref.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dh,heads,tokens,pos,t_max,kind", [
    (64, 4, 1, 0, 1, "plain"), (64, 1, 1, 63, 64, "plain"), (128, 3, 32, 32, 96, "ties"), (64, 2, 33, 31, 70, "ties"),
    (128, 5, 200, 7, 211, "edges"), (64, 8, 129, 127, 257, "edges"), (128, 2, 64, 0, 64, "plain")])
def test_q8_write_and_read(ta, ex, f16, dh, heads, tokens, pos, t_max, kind):
    if f16 and kind == "edges":
        kind = "plain"
    rng = np.random.default_rng(dh + tokens)
    k, v = (rows_of(rng, tokens, heads * dh, kind) for _ in range(2))
    if f16:
        k, v = (np.clip(x, -6e4, 6e4).astype(np.float16).astype(np.float32) for x in (k, v))
    cache = ex.q8_cache(heads, dh, t_max)
    assert cache.size_bytes == 2 * heads * ((t_max + 31) // 32 * 32) * (dh + 2)
    ex.q8_cache_write(ex.tensor_from(k, f16=f16), ex.tensor_from(v, f16=f16), cache, ta.Q8WriteDesc(tokens, pos))
    want_k, want_v = (stands_for(x.reshape(tokens, heads, dh)) for x in (k, v))
    got_k, got_v = read_back(ta, ex, cache, False, t_max)
    new = slice(pos, pos + tokens)
    assert same(got_k[:, :, new], want_k.transpose(1, 2, 0), False)
    assert same(got_v[:, new], want_v.transpose(1, 0, 2), False)
    # the other positions stay zeros
    for a, axis in ((got_k, 2), (got_v, 1)):
        assert not np.delete(a, np.arange(pos, pos + tokens), axis).any()
    # the f16 form, of these positions alone, leaves what it does not read
    with np.errstate(over="ignore"):
        h_k, h_v = read_back(ta, ex, cache, True, tokens, pos, t_max + 3)
        assert same(h_k[:, :, new], want_k.transpose(1, 2, 0), True)
        assert same(h_v[:, new], want_v.transpose(1, 0, 2), True)
    for a, axis in ((h_k, 2), (h_v, 1)):
        assert (np.delete(a, np.arange(pos, pos + tokens), axis) == 7.0).all()


def test_q8_every_scale_boundary(ta, ex):
    """Largest magnitudes on, just under and just over 127 times every number
    of 8 bits: the scale is that number, or the next."""
    m = np.arange(128, 256, dtype=np.float32) * 127.0
    top = np.concatenate([m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(1e9))])
    x = np.zeros((top.size, 64), np.float32)
    x[:, 5] = -top
    x[:, 6] = top / 2
    for shift in (0, -130, 90):
        y = np.ldexp(x, shift).astype(np.float32)
        cache = ex.q8_cache(1, 64, top.size)
        t = ex.tensor_from(y)
        ex.q8_cache_write(t, t, cache, ta.Q8WriteDesc(top.size))
        k, v = read_back(ta, ex, cache, False, top.size)
        assert same(k[0].T, stands_for(y), False) and same(v[0], stands_for(y), False)


def test_q8_every_tie(ta, ex):
    """Values on every half step of every scale, and the f32 numbers next to
    them: to even on it, to the nearer code beside it."""
    s = np.arange(128, 256, dtype=np.float32)[:, None]
    tie = s * (np.arange(127, dtype=np.float32) + 0.5)  # 16 bits: exact
    rows = [tie, np.nextafter(tie, np.float32(0)), np.nextafter(tie, np.float32(1e9))]
    x = np.concatenate([np.concatenate([127 * s, np.minimum(r, 127 * s)], 1) for r in rows])
    x[:, 1::2] *= -1
    for shift in (0, -105, 95):
        y = np.ldexp(x, shift).astype(np.float32)
        cache = ex.q8_cache(1, 128, len(y))
        t = ex.tensor_from(y)
        ex.q8_cache_write(t, t, cache, ta.Q8WriteDesc(len(y)))
        k, v = read_back(ta, ex, cache, False, len(y))
        assert same(k[0].T, stands_for(y), False) and same(v[0], stands_for(y), False)


def test_q8_rows_not_finite(ta, ex):
    x = np.random.default_rng(5).standard_normal((40, 128)).astype(np.float32)
    x[3, 7], x[11, 0], x[33, 127], x[34, 60] = np.inf, -np.inf, np.nan, np.nan
    x[34, 61] = np.inf
    cache = ex.q8_cache(1, 128, 40)
    t = ex.tensor_from(x)
    ex.q8_cache_write(t, t, cache, ta.Q8WriteDesc(40))
    k, v = read_back(ta, ex, cache, False, 40)
    assert same(v[0], stands_for(x), False) and same(k[0].T, stands_for(x), False)
    assert np.isnan(v[0]).any(-1).sum() == 4


def test_q8_strided_and_overwritten(ta, ex):
    """Rows inside a fused QKV tensor; later writes replace earlier ones and
    nothing else."""
    rng = np.random.default_rng(9)
    heads, dh, n = 3, 64, 50
    width = (6 + 2 * heads) * dh + 5
    qkv = rng.standard_normal((n, width)).astype(np.float32)
    cache = ex.q8_cache(heads, dh, 100)
    t = ex.tensor_from(qkv)
    desc = dict(k_offset=6 * dh, k_stride=width, v_offset=(6 + heads) * dh, v_stride=width)
    ex.q8_cache_write(t, t, cache, ta.Q8WriteDesc(n, 11, **desc))
    again = rng.standard_normal((7, heads * dh)).astype(np.float32)
    a = ex.tensor_from(again)
    ex.q8_cache_write(a, a, cache, ta.Q8WriteDesc(7, 30))
    k = qkv[:, 6 * dh:(6 + heads) * dh].reshape(n, heads, dh).copy()
    v = qkv[:, (6 + heads) * dh:(6 + 2 * heads) * dh].reshape(n, heads, dh).copy()
    k[19:26] = v[19:26] = again.reshape(7, heads, dh)
    got_k, got_v = read_back(ta, ex, cache, False, n, 11)
    assert same(got_k[:, :, 11:61], stands_for(k).transpose(1, 2, 0), False)
    assert same(got_v[:, 11:61], stands_for(v).transpose(1, 0, 2), False)


def test_q8_write_at_a_cell(ta, ex):
    """A position cell moves a prepared write; rows past the cache are not
    written."""
    rng = np.random.default_rng(2)
    heads, dh, n, t_max = 2, 128, 5, 67
    pos = ex.create_pos_buffer()
    x = rng.standard_normal((n, heads * dh)).astype(np.float32)
    t = ex.tensor_from(x)
    cache = ex.q8_cache(heads, dh, t_max)
    step = ex.prepare_exec_ops([ta.ExecOp.q8_cache_write(t, t, cache, ta.Q8WriteDesc(
        n, 1, pos_addr=pos.device_address))])
    want = np.zeros((heads, t_max, dh))
    for at in (0, 28, 60, 63, 66, 5000, 0xFFFFFFFF):
        pos.set(at)
        step.run()
        for i in range(n):
            if 1 + at + i < t_max:
                want[:, 1 + at + i] = stands_for(x[i].reshape(heads, dh))
        assert same(read_back(ta, ex, cache, False, t_max)[1], want, False), at


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("dh,first", [(64, 0), (128, 3)])
def test_q8_rows_that_f16_holds_read_back_finite(ta, ex, f16, dh, first):
    """The scale of a row whose largest magnitude is among f16's top eight is
    516, and 127 times that is past f16's largest: it reads back as that one.
    Rows past f16 read back as infinities still, rows with a NaN as NaN."""
    tops = np.arange(65280, 65505, 32, dtype=np.float32)
    n = 2 * tops.size + 3
    x = np.random.default_rng(dh).standard_normal((n, dh)).astype(np.float32)
    x[:tops.size, 7], x[tops.size:2 * tops.size, dh - 1] = tops, -tops
    x[-1, 5] = np.nan
    if f16:
        x = x.astype(np.float16).astype(np.float32)
    else:
        x[-2, 9], x[-3, 9] = 7e4, -1e9
    want = stands_for(x)
    assert (np.abs(want[:2 * tops.size]).max(-1) == 65532).all()
    cache = ex.q8_cache(1, dh, n)
    t = ex.tensor_from(x, f16=f16)
    ex.q8_cache_write(t, t, cache, ta.Q8WriteDesc(n))
    k, v = read_back(ta, ex, cache, True, n - first, first)
    want = np.where(np.abs(want) == 65532, np.sign(want) * 65504, want)[first:]
    with np.errstate(over="ignore"):
        assert same(k[0, :, first:].T, want, True) and same(v[0, first:], want, True)
    assert np.isfinite(v[0, first:2 * tops.size]).all() and np.isinf(v[0]).any() == (not f16)


# ------------------------------------------------------------------- RoPE


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("tokens,heads,head_dim,sections", [
    (1, 1, 2, [1]), (16, 32, 64, [32]), (5, 3, 128, [16, 24, 24]), (777, 9, 80, [7, 13]), (33, 2, 48, [4, 4, 8, 8]),
    (3, 1, 7, [1, 2]), (2100, 4, 64, [5, 3, 20]), (20000, 1, 8, [1, 1, 2])])
def test_rope_axes(ta, ex, f16, tokens, heads, head_dim, sections):
    rng = np.random.default_rng(tokens)
    pairs = sum(sections)
    x = rng.standard_normal((tokens, heads, head_dim)).astype(np.float32)
    if f16:
        x = x.astype(np.float16).astype(np.float32)
    rows = 500
    theta = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(pairs) / pairs)
    table = np.stack([np.cos(theta), np.sin(theta)], -1).astype(np.float32)
    pos = rng.integers(0, rows - 20, (len(sections), tokens))
    pos[:, 0] = 600  # past the table: its last row
    cell = ta.U32Cell(ex.ctx, pos.size + 1)
    cell.write(pos.reshape(-1))
    base = ex.create_pos_buffer()
    base.set(7)
    t, out = ex.tensor_from(x, f16=f16), ex.tensor(x.shape, f16)
    desc = ta.RopeAxesDesc(heads, head_dim, 2 * pairs, sections, pos_base=3, pos_addr=base.device_address)
    ex.rope_axes(t, ex.tensor_from(table), cell, out, desc)
    axis = np.repeat(np.arange(len(sections)), sections)
    cs = table[np.minimum(pos + 10, rows - 1)[axis].T, np.arange(pairs)].astype(np.float64)[:, None]
    a, b = x[..., 0:2 * pairs:2].astype(np.float64), x[..., 1:2 * pairs:2].astype(np.float64)
    ref, size = x.astype(np.float64).copy(), np.zeros(x.shape)
    ref[..., 0:2 * pairs:2] = a * cs[..., 0] - b * cs[..., 1]
    ref[..., 1:2 * pairs:2] = a * cs[..., 1] + b * cs[..., 0]
    size[..., 0:2 * pairs:2] = np.abs(a * cs[..., 0]) + np.abs(b * cs[..., 1])
    size[..., 1:2 * pairs:2] = np.abs(a * cs[..., 1]) + np.abs(b * cs[..., 0])
    got = ex.download(out)
    tol = 2 * U32 * size + (2.0 ** -11 * np.abs(ref) + 2.0 ** -25 if f16 else 0.0)
    assert (np.abs(got - ref) <= tol * 1.001).all()
    # in place
    ex.rope_axes(t, ex.tensor_from(table), cell, t, desc)
    assert np.array_equal(ex.download(t), got)


def test_rope_axes_equals_rope(ta, ex):
    """Positions 0, 1, 2 .. on one axis: ta_rope's bits."""
    rng = np.random.default_rng(3)
    x = ex.tensor_from(rng.standard_normal((40, 8, 64)).astype(np.float32))
    table = ex.tensor_from(rng.standard_normal((60, 24, 2)).astype(np.float32))
    a, b = ex.tensor([40, 8, 64]), ex.tensor([40, 8, 64])
    cell = ta.U32Cell(ex.ctx, 40)
    cell.write(range(40))
    ex.rope(x, table, a, 8, 64, 48, pos_base=11)
    ex.rope_axes(x, table, cell, b, ta.RopeAxesDesc(8, 64, 48, [24], pos_base=11))
    assert np.array_equal(ex.download(a), ex.download(b))


# ---------------------------------------------------------- tree attention


def tree_masks(rng, tokens):
    words = []
    for t in range(tokens):
        parent = int(rng.integers(-1, t)) if t else -1
        words.append((words[parent] if parent >= 0 else 0) | 1 << t)
    return words


def mask_cell(ta, ex, words):
    c = ta.U32Cell(ex.ctx, 2 * len(words))
    c.write([w >> s & 0xFFFFFFFF for w in words for s in (0, 32)])
    return c


def reference(q, k, v, words, n0, scale):
    """q [T, H, dh], k and v [n, H_kv, dh], all f64.  (out, per-element sum of
    weight * |v|, per-row score error without the 4 u, n seen)."""
    t, h, dh = q.shape
    group = h // k.shape[1]
    out, mag, eps = np.zeros(q.shape), np.zeros(q.shape), np.zeros((t, h, 1))
    for i in range(t):
        seen = np.array([True] * n0 + [bool(words[i] >> j & 1) for j in range(t)])
        for a in range(h):
            kk, vv = k[seen, a // group], v[seen, a // group]
            if not len(kk):
                continue
            s = kk @ q[i, a] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, a], mag[i, a] = p @ vv, p @ np.abs(vv)
            eps[i, a] = (np.abs(kk) @ np.abs(q[i, a])).max() * abs(scale) * (dh + 4) * U32 + 4 * U32 * np.abs(s).max()
    return out, mag, eps


def check(got, ref, f16, q8, n):
    out, mag, eps = ref
    tol = mag * (2 * (eps + 4 * U32) + 2 * n * U32) + 1e-37
    if f16:
        tol = tol + 2.0 ** -11 * np.abs(out) + 2.0 ** -25 + (2.0 ** -15 * mag if q8 else 2.0 ** -11 * mag)
    err = np.abs(got - out)
    assert np.isfinite(got).all() and (err <= tol).all(), float((err / tol).max())


class Case:
    """Inputs of one attention: a dense cache (f32, f16) or an 8-bit one."""

    def __init__(self, ta, ex, cache, f16, dh, heads, group, tokens, n0, extra=0, seed=0, fused=0, spread=1.0,
                 words=None):
        rng = np.random.default_rng(seed + 31 * tokens + n0)
        self.ta, self.ex, self.f16, self.kind = ta, ex, f16, cache
        self.t, self.n0, self.n, self.dh = tokens, n0, n0 + tokens, dh
        self.h, self.hkv, self.t_max = heads * group, heads, n0 + tokens + extra
        self.scale = 1.0 / np.sqrt(dh)
        self.words = tree_masks(rng, tokens) if words is None else words
        self.fused = fused
        width = self.h * dh + fused
        q = rng.standard_normal((tokens, width)).astype(np.float32) * spread
        if f16:
            q = q.astype(np.float16).astype(np.float32)
        self.q = q
        self.k = rng.standard_normal((self.t_max, heads, dh)).astype(np.float32)
        self.v = rng.standard_normal((self.t_max, heads, dh)).astype(np.float32)
        if cache == "f16":
            self.k, self.v = (x.astype(np.float16).astype(np.float32) for x in (self.k, self.v))

    def put(self):
        ta, ex = self.ta, self.ex
        self.tq = ex.tensor_from(self.q, f16=self.f16)
        self.out = ex.tensor([self.t, self.h, self.dh], self.f16)
        if self.kind == "q8":
            self.cache = ex.q8_cache(self.hkv, self.dh, self.t_max)
            k, v = (ex.tensor_from(x.reshape(self.t_max, -1)) for x in (self.k, self.v))
            ex.q8_cache_write(k, v, self.cache, ta.Q8WriteDesc(self.t_max))
        else:
            f16 = self.kind == "f16"
            self.kt = ex.tensor_from(np.ascontiguousarray(self.k.transpose(1, 2, 0)), f16=f16)
            self.tv = ex.tensor_from(np.ascontiguousarray(self.v.transpose(1, 0, 2)), f16=f16)
        return self

    def desc(self, **kw):
        kw = {"kv_len": self.n0, **kw}
        return self.ta.TreeAttentionDesc(tokens=self.t, scale=self.scale,
                                         q_stride=self.q.shape[1] if self.fused else 0, **kw)

    def op(self, mask, desc=None):
        d = desc or self.desc()
        if self.kind == "q8":
            return self.ta.ExecOp.q8_tree_attention(self.tq, self.cache, self.out, d, mask)
        return self.ta.ExecOp.tree_attention(self.tq, self.kt, self.tv, self.out, d, mask)

    def run(self, mask=True, desc=None):
        m = mask_cell(self.ta, self.ex, self.words) if mask is True else mask
        d = desc or self.desc()
        if self.kind == "q8":
            self.ex.q8_tree_attention(self.tq, self.cache, self.out, d, m)
        else:
            self.ex.tree_attention(self.tq, self.kt, self.tv, self.out, d, m)
        return self.ex.download(self.out)

    def values(self):
        if self.kind == "q8":
            return stands_for(self.k), stands_for(self.v)
        return self.k.astype(np.float64), self.v.astype(np.float64)

    def ref(self, n0=None, words=None, k=None, v=None):
        n0 = self.n0 if n0 is None else n0
        vk, vv = self.values()
        k, v = vk if k is None else k, vv if v is None else v
        q = self.q[:, :self.h * self.dh].astype(np.float64).reshape(self.t, self.h, self.dh)
        return reference(q, k[:n0 + self.t], v[:n0 + self.t], self.words if words is None else words, n0, self.scale)

    def check(self, got, ref=None):
        check(got, ref or self.ref(), self.f16, self.kind == "q8", self.n)


KINDS = [("f32", False), ("f16", False), ("f16", True), ("q8", False), ("q8", True)]


@pytest.mark.parametrize("cache,f16", KINDS)
@pytest.mark.parametrize("dh,heads,group,tokens,n0,extra", [
    (64, 1, 1, 1, 0, 0), (128, 1, 1, 1, 1, 0), (64, 2, 1, 1, 63, 1), (128, 2, 8, 1, 300, 3), (64, 4, 8, 8, 1016, 7),
    (128, 3, 3, 5, 31, 0), (128, 2, 4, 64, 129, 0), (64, 5, 2, 33, 95, 62), (128, 1, 1, 64, 2000, 1),
    (64, 1, 12, 3, 64, 0), (64, 2, 4, 16, 0, 5)])
def test_tree_attention(ta, ex, cache, f16, dh, heads, group, tokens, n0, extra):
    c = Case(ta, ex, cache, f16, dh, heads, group, tokens, n0, extra).put()
    got = c.run()
    c.check(got)
    assert np.array_equal(got, c.run())  # the same bits every time


@pytest.mark.parametrize("cache,f16", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("heads,group,tokens", [(2, 4, 4), (1, 17, 1), (2, 8, 4), (1, 8, 5), (2, 4, 16), (1, 3, 22),
                                                (1, 8, 12), (1, 4, 33), (1, 5, 64)])
@pytest.mark.parametrize("n0,t_max", [(700, 840), (0, 72), (1111, 1176)])
def test_tree_attention_every_row_count(ta, ex, cache, f16, dh, heads, group, tokens, n0, t_max):
    """16, 17, 32, 40, 64, 66, 96, 132 and 320 rows of a head, on caches of
    whole 16-byte pieces that end inside a tile or before it."""
    c = Case(ta, ex, cache, f16, dh, heads, group, tokens, n0, t_max - n0 - tokens).put()
    assert c.t_max % 8 == 0
    c.check(c.run())


@pytest.mark.parametrize("cache,f16", KINDS)
@pytest.mark.parametrize("dh,heads,group,tokens,t_max", [(64, 1, 16, 1, 4800), (128, 1, 8, 4, 4807), (128, 2, 4, 12, 4744),
                                                         (64, 1, 8, 14, 4736)])
def test_tree_attention_many_chunks(ta, ex, cache, f16, dh, heads, group, tokens, t_max):
    """Chunks to the cap of every row count, the last ones ragged."""
    c = Case(ta, ex, cache, f16, dh, heads, group, tokens, 4700, t_max - 4700 - tokens).put()
    c.check(c.run())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("heads,group,tokens,t_max", [(1, 3, 22, 16000), (1, 3, 22, 15999), (1, 8, 33, 3976),
                                                      (2, 4, 64, 4154), (1, 16, 64, 1088), (1, 16, 64, 1091)])
@pytest.mark.parametrize("n0", [0, 700, -1])
def test_tree_attention_many_rows_and_positions(ta, ex, f16, dh, heads, group, tokens, t_max, n0):
    """Four row tiles of an f16 cache to a workgroup (2^20 rows x positions),
    the last of them in part, on a cache of either kind of rows; few committed
    positions named by a cell, and all that fit."""
    full = t_max - tokens - 1
    at = full if n0 < 0 else n0
    c = Case(ta, ex, "f16", f16, dh, heads, group, tokens, at, t_max - at - tokens).put()
    assert tokens * group * (t_max - 1) >= 2**20
    if n0 < 0:
        c.check(c.run())
        return
    cell = ex.create_pos_buffer()
    cell.write([at])
    c.check(c.run(desc=c.desc(kv_len=0, pos_addr=cell.device_address)))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("dh,tokens,t_max", [(128, 64, 1088), (128, 64, 1091), (64, 64, 1088), (64, 64, 1091),
                                             (128, 4, 1088), (128, 4, 1091), (64, 4, 1091)])
def test_tree_attention_masked_values_in_many_rows(ta, ex, f16, bad, dh, tokens, t_max):
    """NaN and infinities in a draft that one row sees, and behind the drafts,
    at every number of row tiles to a workgroup."""
    words = [1 << t for t in range(tokens)]
    at = t_max - tokens - 3
    c = Case(ta, ex, "f16", f16, dh, 1, 16, tokens, at, 3, words=words)
    k, v = c.values()
    for x in (c.k, c.v):
        x[at + 2, 0, 5] = bad  # draft 2
        x[at + tokens:, :, ::3] = bad
    c.put()
    got = c.run()
    rows = [t for t in range(tokens) if t != 2]
    check(got[rows], tuple(x[rows] for x in c.ref(k=k, v=v)), f16, False, c.n)
    assert not np.isfinite(got[2]).all(-1).any()


@pytest.mark.parametrize("cache,f16", KINDS)
def test_tree_attention_long(ta, ex, cache, f16):
    """Many chunks, and a group of rows past one tile."""
    c = Case(ta, ex, cache, f16, 128, 2, 4, 9, 9001, 3, spread=3.0).put()
    c.check(c.run())


@pytest.mark.parametrize("cache,f16", KINDS)
def test_tree_attention_fused_q(ta, ex, cache, f16):
    """q as part of a fused product's rows, from an odd element on."""
    c = Case(ta, ex, cache, f16, 64, 2, 3, 7, 70, fused=257)
    q = c.q.copy()
    c.q = np.concatenate([np.full((c.t, 1), 9e4 if not f16 else 9.0, np.float32), q[:, :-1]], 1)
    c.put()
    got = c.run(desc=c.desc(q_offset=1))
    c.q = q[:, :-1]
    c.check(got)


@pytest.mark.parametrize("cache,f16", KINDS)
def test_tree_attention_chain(ta, ex, cache, f16):
    """No mask: drafts see those before them, all 64."""
    c = Case(ta, ex, cache, f16, 64, 1, 2, 64, 10).put()
    c.check(c.run(mask=None), c.ref(words=[(1 << t + 1) - 1 for t in range(64)]))


@pytest.mark.parametrize("cache,f16", KINDS)
@pytest.mark.parametrize("n0", [0, 40])
def test_tree_attention_rows_that_see_nothing(ta, ex, cache, f16, n0):
    words = [0, 1, 1 << 5, 0, 0b111, 1 << 63 | 1 << 4]  # bits past the drafts name nothing
    c = Case(ta, ex, cache, f16, 128, 2, 2, 6, n0, words=words).put()
    got = c.run()
    c.check(got, c.ref(words=[w & 63 for w in words]))
    if n0 == 0:
        assert not got[0].any() and not got[3].any()


@pytest.mark.parametrize("cache,f16", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_tree_attention_masked_values_do_not_matter(ta, ex, cache, f16, bad):
    """NaN and infinities in drafts that a row does not see, and behind the
    drafts, in K and in V."""
    words = [1 << t for t in range(6)]  # every draft sees itself alone
    c = Case(ta, ex, cache, f16, 128, 2, 4, 6, 100, 40, words=words)
    k, v = c.values()
    for x in (c.k, c.v):
        x[102, 0, 5] = bad  # draft 2, head 0
        x[106:, :, ::3] = bad
    c.put()
    got = c.run()
    rows = [0, 1, 3, 4, 5]
    ref = c.ref(k=k, v=v)
    check(got[rows], tuple(x[rows] for x in ref), f16, cache == "q8", c.n)
    check(got[2:3, 4:], tuple(x[2:3, 4:] for x in ref), f16, cache == "q8", c.n)
    if not np.isfinite(bad) and cache == "q8":
        assert np.isnan(got[2, :4]).all()  # such a row stands for NaN


@pytest.mark.parametrize("cache,f16", [k for k in KINDS if k[0] != "q8"])
def test_tree_attention_infinite_values_seen(ta, ex, cache, f16):
    """An infinity that rows do see comes out as the formula has it: in V in
    its column, in K as a weight of zero or a NaN."""
    c = Case(ta, ex, cache, f16, 64, 1, 2, 4, 90, 3, words=[15] * 4)
    c.v[17, 0, 9] = np.inf
    c.v[93, 0, 30] = -np.inf
    c.put()
    got = c.run()
    with np.errstate(invalid="ignore"):
        out = c.ref()[0]
    assert (got[..., 9] == np.inf).all() and (got[..., 30] == -np.inf).all()
    rest = [d for d in range(64) if d not in (9, 30)]
    k, v = c.values()
    v[17, 0, 9] = v[93, 0, 30] = 0.0
    ref = c.ref(k=k, v=v)
    check(got[..., rest], tuple(x[..., rest] if x.shape[-1] > 1 else x for x in ref), f16, False, c.n)
    # K: q of one sign against it
    c = Case(ta, ex, cache, f16, 64, 1, 2, 4, 90, 3, words=[15] * 4)
    c.q[:2] = -np.abs(c.q[:2])
    c.q[2:] = np.abs(c.q[2:])
    k, v = c.values()
    c.k[40, 0, 3] = np.inf
    c.put()
    got = c.run()
    keep = np.r_[0:40, 41:c.t_max]
    ref = reference(c.q.astype(np.float64).reshape(4, 2, 64), k[keep][:93], v[keep][:93], c.words, 89, c.scale)
    check(got[:2], tuple(x[:2] for x in ref), f16, False, c.n)
    assert np.isnan(got[2:]).all()


@pytest.mark.parametrize("cache,f16", [("f32", False), ("f16", False), ("q8", False)])
@pytest.mark.parametrize("spread", [1e-30, 1e-6, 60.0])
def test_tree_attention_q_ranges(ta, ex, cache, f16, spread):
    """Tiny and large f32 q: uniform weights, and weights far apart."""
    c = Case(ta, ex, cache, f16, 64, 2, 2, 5, 200, spread=spread).put()
    c.check(c.run())


@pytest.mark.parametrize("cache,f16", KINDS)
def test_tree_attention_small_weights_count(ta, ex, cache, f16):
    """Values that only keys of small weight have keep f32's precision: V is
    zero where the weights are large."""
    c = Case(ta, ex, cache, f16, 64, 1, 1, 1, 255)
    c.q[:] = 0.0
    c.q[0, 0] = 16.0
    c.k[:] = 0.0
    c.k[:128, 0, 0] = 8.0  # weight ratio 2^(-16 * 8 / 8 * log2 e) = 2^-23
    c.k[:, 0, 1] = 1.0
    c.v[:128] = 0.0
    c.put()
    c.check(c.run())


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_tree_attention_q8_scales_far_apart(ta, ex, cache):
    """Rows of very different size side by side."""
    c = Case(ta, ex, cache, False, 64, 1, 2, 3, 300)
    size = np.exp(np.random.default_rng(1).uniform(-6, 3, (c.t_max, 1, 1)))
    c.v = (c.v * size).astype(np.float32)
    if cache == "f16":
        c.v = c.v.astype(np.float16).astype(np.float32)
    c.put()
    c.check(c.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-45, 1e-30])
@pytest.mark.parametrize("cache,f16", KINDS)
def test_tree_attention_scales(ta, ex, cache, f16, scale):
    c = Case(ta, ex, cache, f16, 64, 2, 2, 3, 77).put()
    c.scale = float(np.float32(scale))
    c.check(c.run())


@pytest.mark.parametrize("cache,f16", KINDS)
def test_tree_attention_follows_a_cell(ta, ex, cache, f16):
    """A prepared attention replayed at other lengths and masks, among eager
    work of the same executor; the length is kept within the cache."""
    c = Case(ta, ex, cache, f16, 64, 2, 4, 6, 500).put()
    pos = ex.create_pos_buffer()
    mask = mask_cell(ta, ex, c.words)
    step = ex.prepare_exec_ops([c.op(mask, c.desc(kv_len=3, pos_addr=pos.device_address))])
    for at, words in ((0, c.words), (497, [63] * 6), (29, c.words), (100, [0] * 6), (4000, c.words)):
        pos.set(at)
        mask.write([w >> s & 0xFFFFFFFF for w in words for s in (0, 32)])
        step.run()
        got = ex.download(c.out)
        n0 = min(3 + at, 500)
        c.check(got, c.ref(n0=n0, words=words))
        eager = c.run(mask=mask, desc=c.desc(kv_len=n0))
        c.check(eager, c.ref(n0=n0, words=words))
        step.run()
        assert np.array_equal(ex.download(c.out), got)


def test_tree_attention_two_graphs_and_threads(ta, ex):
    """Two prepared graphs in flight together, and eager calls from several
    threads, each with scratch of its own: the bits of lone calls."""
    cs = [Case(ta, ex, "q8", False, 128, 2, 4, 4, 6000, seed=s).put() for s in range(4)]
    cs.append(Case(ta, ex, "f16", True, 64, 4, 8, 64, 3000).put())
    want = [c.run() for c in cs]
    masks = [mask_cell(ta, ex, c.words) for c in cs]
    steps = [ex.prepare_exec_ops([c.op(m)]) for c, m in zip(cs, masks)]
    for _ in range(5):
        for s in steps:
            s.submit()
        for s in steps:
            s.wait()
        for c, w in zip(cs, want):
            assert np.array_equal(ex.download(c.out), w)
    bad = []

    def work(i):
        for _ in range(5):
            if not np.array_equal(cs[i].run(mask=masks[i]), want[i]):
                bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(cs))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_far_positions_of_the_8_bit_cache(ta, ex):
    """Offsets past 32 bits: drafts behind 2^25 - 4 positions of zeros, whose
    weights and values are whole numbers and zeros, so they add no rounding."""
    rng = np.random.default_rng(4)
    t, dh, t_max = 4, 64, 1 << 25
    cache = ex.q8_cache(2, dh, t_max)
    assert cache.size_bytes > 1 << 33
    q, k, v = (rng.standard_normal((t, 2, dh)).astype(np.float32) * s for s in (3.0, 8.0, 1e6))
    ex.q8_cache_write(ex.tensor_from(k.reshape(t, -1)), ex.tensor_from(v.reshape(t, -1)), cache,
                      ta.Q8WriteDesc(t, t_max - t))
    out = ex.tensor([t, 2, dh])
    ex.q8_tree_attention(ex.tensor_from(q), cache, out, ta.TreeAttentionDesc(t_max - t, t, 1 / 8))
    got, lk, lv = ex.download(out), stands_for(k), stands_for(v)
    for i in range(t):
        for h in range(2):
            s = lk[:i + 1, h] @ q[i, h].astype(np.float64) / 8
            w = np.exp(s)
            ref, mag = w @ lv[:i + 1, h] / (t_max - t + w.sum()), w @ np.abs(lv[:i + 1, h]) / (t_max - t + w.sum())
            eps = (np.abs(lk[:i + 1, h]) @ np.abs(q[i, h])).max() / 8 * (dh + 4) * U32 + 4 * U32 * np.abs(s).max()
            assert (np.abs(got[i, h] - ref) <= mag * (2 * (eps + 4 * U32) + 2 * 600 * U32)).all()


def test_tree_attention_without_scratch(ta, ctx, monkeypatch):
    """Scratch that cannot be had is an error, and the next call runs."""
    ex1 = ta.Executor(ctx, n_slots=1, tune=False)
    c = Case(ta, ex1, "q8", False, 64, 1, 2, 2, 3000).put()
    monkeypatch.setenv("TA_SCRATCH_LIMIT", "1000")
    with pytest.raises(ta.TensorAshError, match="out of memory"):
        c.run()
    with pytest.raises(ta.TensorAshError, match="out of memory"):
        ex1.prepare_exec_ops([c.op(None)])
    monkeypatch.delenv("TA_SCRATCH_LIMIT")
    c.check(c.run())


# The sizes pick every kernel over f16 caches: 32, 64 (dh 128) and 128 rows to
# a workgroup, rows of K in whole 16-byte pieces or not; the last two take the
# 128-row kernel for the cache's capacity, the length being named by a cell.
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("group,tokens,t_max,cell", [
    (1, 1, 256, False), (1, 1, 257, False), (8, 8, 256, False), (8, 8, 257, False), (64, 64, 256, False),
    (64, 64, 257, False), (4, 64, 4104, True), (4, 64, 4103, True)])
def test_tree_attention_f16_weights_in_two_pieces(ta, ex, dh, group, tokens, t_max, cell):
    """f16 activations over an f16 cache hold weights in two f16 pieces, in a
    prepared step as in an eager call: within 2^-22, counted twice (its own,
    and the total's).  Half of the keys have the row's largest weight, which
    f16 holds, the others one that it misses by nearly half a step, and V makes
    their sums cancel, so that the result's own step is far below that."""
    n = 256
    c = Case(ta, ex, "f16", True, dh, 1, group, tokens, n - tokens, t_max - n, words=[(1 << tokens) - 1] * tokens)
    d = np.arange(1, 512) / 64.0
    w = np.exp(-4.0 * d * c.scale)
    off = np.abs((w * 2048).astype(np.float16).astype(np.float64) / (w * 2048) - 1) * (w > 0.25) * (w < 0.9)
    at = int(off.argmax())
    assert off[at] > 0.75 * 2.0 ** -11
    c.q[:] = 0.0
    c.q.reshape(tokens, -1, dh)[..., 0] = 4.0
    c.k[:] = 0.0
    c.k[1::2, :, 0] = -d[at]
    c.v[0::2] = 1.0
    c.v[1::2] = np.float32(np.float16(-1.0 / w[at]))
    c.put()
    pos = ex.create_pos_buffer()
    pos.set(n - tokens)
    got = c.run(desc=c.desc(kv_len=0, pos_addr=pos.device_address) if cell else None)
    out, mag, eps = c.ref()
    tol = mag * (2 * (eps + 4 * U32) + 2 * n * U32 + 2.0 ** -21) + 2.0 ** -11 * np.abs(out) + 2.0 ** -25
    # one piece would be off by that step of half of mag
    assert (2 * tol < mag * off[at] / 2).all()
    assert (np.abs(got - out) <= tol).all(), float((np.abs(got - out) / tol).max())


@pytest.mark.parametrize("cache,f16", KINDS)
@pytest.mark.parametrize("dh,group,tokens,n0,extra", [(64, 2, 6, 100, 40), (128, 4, 3, 300, 2), (128, 8, 16, 240, 1)])
def test_tree_attention_bits_without_what_lies_behind(ta, ex, cache, f16, dh, group, tokens, n0, extra):
    """Memory behind the drafts may hold anything: not a bit of the result,
    nor the way it is taken, depends on it."""
    got = []
    for bad in (0.0, 1.0, np.inf, np.nan):
        c = Case(ta, ex, cache, f16, dh, 2, group, tokens, n0, extra)
        c.k[c.n:] = c.v[c.n:] = bad
        got.append(c.put().run())
    c.check(got[0])
    for g in got[1:]:
        assert np.array_equal(got[0], g)


@pytest.mark.parametrize("cache,f16", [("f32", False), ("q8", False), ("q8", True)])
@pytest.mark.parametrize("group", [2, 20])
@pytest.mark.parametrize("scale", [0.0, 1e-45, 1e-40, -1e-38])
def test_tree_attention_small_scales_of_large_scores(ta, ex, cache, f16, group, scale):
    """A scale of zero, or below f32's smallest normal, over q . k near f32's
    largest: what the formula has.  (scale log2 e then has an error of its own
    of 2^-150; times |q . k| < 2^123 that is below the exponential's 4 u.)"""
    c = Case(ta, ex, cache, f16, 64, 2, group, 5, 120)
    if not f16:
        c.q *= 1e15
    c.k *= np.float32(1e36 if f16 else 1e21)
    c.put()
    c.scale = float(np.float32(scale))
    q = c.q.astype(np.float64).reshape(5, 2, group, 64)
    top = np.abs(np.einsum("tgad,ngd->tgan", q, c.values()[0])).max()
    assert 2.0 ** 118 < top < 2.0 ** 126
    c.check(c.run())


@pytest.mark.parametrize("group", [2, 20])
def test_tree_attention_q8_largest_q(ta, ex, group):
    """|q| * 127 * dh close under f32's largest, against a row of K whose codes
    are all 127, and V whose sum with weights of 16 is close under it too."""
    c = Case(ta, ex, "q8", False, 64, 2, group, 5, 120)
    c.q *= np.float32(4.1e34) / np.abs(c.q).max()
    c.q[0] = 4.1e34
    c.k *= np.float32(1e-29)
    c.k[3] = 127.0 * 2.0 ** -100
    c.v *= np.float32(3.3e38 / 16) / np.abs(c.v).sum(0).max()
    c.put()
    c.scale = float(np.float32(1e-7))
    assert (c.values()[0][3] == 127.0 * 2.0 ** -100).all()
    c.check(c.run())


# ------------------------------------------------------------- used together


@pytest.mark.parametrize("quantised", [True, False])
def test_verifying_drafts_in_one_graph(ta, ex, quantised):
    """A tree of drafts through one attention layer, prepared once and
    replayed at two lengths: QKV product, rotation by depth, write into the
    cache, attention, output product; against the formulas in 64 bits on the
    GPU's own projections."""
    rng = np.random.default_rng(17)
    hid, h, hkv, dh, t, t_max = 256, 4, 2, 64, 10, 400
    kv, width = hkv * dh, (h + 2 * hkv) * dh
    words = tree_masks(rng, t)
    depth = [bin(w).count("1") - 1 for w in words]
    theta = np.arange(t_max)[:, None] * 10000.0 ** (-np.arange(dh // 2) / (dh // 2))
    table = np.stack([np.cos(theta), np.sin(theta)], -1).astype(np.float32)
    x = ex.tensor_from(rng.standard_normal((t, hid)).astype(np.float32))
    wqkv = ex.tensor_from((rng.standard_normal((hid, width)) * 0.06).astype(np.float32))
    wo = ex.tensor_from((rng.standard_normal((h * dh, hid)) * 0.06).astype(np.float32))
    old_k, old_v = (rng.standard_normal((t_max, hkv, dh)).astype(np.float32) for _ in range(2))
    qkv, y, attn = ex.tensor([t, width]), ex.tensor([t, hid]), ex.tensor([t, h * dh])
    turned = ex.tensor([t, width])
    tt, pos = ex.tensor_from(table), ex.create_pos_buffer()
    depths, mask = ta.U32Cell(ex.ctx, t), mask_cell(ta, ex, words)
    depths.write(depth)
    E, at = ta.ExecOp, pos.device_address
    # q and k heads turn, v heads pass through a second op that keeps them
    ops = [E.matmul(ta.MatmulOp(x, wqkv, qkv)),
           E.rope_axes(qkv, tt, depths, turned, ta.RopeAxesDesc(h + 2 * hkv, dh, dh, [dh // 2], pos_addr=at))]
    desc = ta.TreeAttentionDesc(0, t, 1 / np.sqrt(dh), q_stride=width, pos_addr=at)
    k, v = (ex.tensor_from(a.reshape(t_max, kv)) for a in (old_k, old_v))
    if quantised:
        cache = ex.q8_cache(hkv, dh, t_max)
        ex.q8_cache_write(k, v, cache, ta.Q8WriteDesc(t_max))
        # K from the turned rows, V from the product
        ops += [E.q8_cache_write(turned, qkv, cache, ta.Q8WriteDesc(
                    t, 0, k_offset=h * dh, k_stride=width, v_offset=h * dh + kv, v_stride=width, pos_addr=at)),
                E.q8_tree_attention(turned, cache, attn, desc, mask)]
    else:
        kt = ex.tensor_from(np.ascontiguousarray(old_k.transpose(1, 2, 0)))
        vc = ex.tensor_from(np.ascontiguousarray(old_v.transpose(1, 0, 2)))
        ops += [E.copy_strided(turned, kt, ta.CopyDesc((dh, hkv, t), (1, dh, width), (t_max, dh * t_max, 1),
                                                       src_offset=h * dh, pos_addr=at, pos_scale=1)),
                E.copy_strided(qkv, vc, ta.CopyDesc((dh, hkv, t), (1, dh, width), (1, t_max * dh, dh),
                                                    src_offset=h * dh + kv, pos_addr=at, pos_scale=dh)),
                E.tree_attention(turned, kt, vc, attn, desc, mask)]
    ops.append(E.matmul(ta.MatmulOp(attn, wo, y)))
    step = ex.prepare_exec_ops(ops)
    lk, lv = old_k.astype(np.float64), old_v.astype(np.float64)
    if quantised:
        lk, lv = stands_for(lk), stands_for(lv)
    for n0 in (300, 33, 390):
        pos.set(n0)
        step.run()
        rows = ex.download(qkv).astype(np.float64)
        cs = table[np.array(depth) + n0].astype(np.float64)[:, None]
        z = rows.reshape(t, -1, dh)
        rot = np.empty_like(z)
        rot[..., 0::2] = z[..., 0::2] * cs[..., 0] - z[..., 1::2] * cs[..., 1]
        rot[..., 1::2] = z[..., 0::2] * cs[..., 1] + z[..., 1::2] * cs[..., 0]
        got_rot = ex.download(turned).reshape(t, -1, dh).astype(np.float64)
        assert np.abs(got_rot - rot).max() <= 4 * U32 * np.abs(z).max() * 2
        new_k, new_v = got_rot[:, h:h + hkv], z[:, h + hkv:]
        if quantised:
            new_k, new_v = stands_for(new_k), stands_for(new_v)
        lk[n0:n0 + t], lv[n0:n0 + t] = new_k, new_v
        ref = reference(got_rot[:, :h], lk[:n0 + t], lv[:n0 + t], words, n0, 1 / np.sqrt(dh))
        check(ex.download(attn).reshape(t, h, dh), ref, False, quantised, n0 + t)
        a = ex.download(attn).astype(np.float64)
        w = ex.download(wo).astype(np.float64)
        assert np.abs(ex.download(y) - a @ w).max() <= (hid + 4) * U32 * (np.abs(a) @ np.abs(w)).max()


def test_chunked_prompt_over_the_8_bit_cache(ta, ex):
    """A prompt in two chunks: each is quantised as it comes, and the whole
    cache is read back for the prefill attention."""
    rng = np.random.default_rng(23)
    h, hkv, dh, n = 4, 2, 64, 150
    q = rng.standard_normal((n, h, dh)).astype(np.float32)
    k, v = (rng.standard_normal((n, hkv, dh)).astype(np.float32) for _ in range(2))
    cache = ex.q8_cache(hkv, dh, n)
    kt, vc = ex.tensor([hkv, dh, n]), ex.tensor([hkv, n, dh])
    got = []
    for lo, hi in ((0, 64), (64, n)):
        tk, tv = (ex.tensor_from(x[lo:hi].reshape(hi - lo, -1)) for x in (k, v))
        tq = ex.tensor_from(np.ascontiguousarray(q[lo:hi].transpose(1, 0, 2)))
        out = ex.tensor([h, hi - lo, dh])
        ex.run_exec_ops([ta.ExecOp.q8_cache_write(tk, tv, cache, ta.Q8WriteDesc(hi - lo, lo)),
                         ta.ExecOp.q8_cache_read(cache, kt, vc, ta.Q8ReadDesc(hi)),
                         ta.ExecOp.flash_attn(tq, kt, vc, out, ta.FlashAttentionDesc(hi, lo, 1 / np.sqrt(dh)))])
        got.append(ex.download(out).transpose(1, 0, 2))
    got = np.concatenate(got)
    lk, lv = stands_for(k), stands_for(v)
    for i in (0, 63, 64, 100, n - 1):
        ref = reference(q[i:i + 1].astype(np.float64), np.r_[lk[:i + 1], lk[:0]], lv[:i + 1], [1], i, 1 / np.sqrt(dh))
        check(got[i:i + 1], ref, False, True, i + 1)


# ------------------------------------------------------------------ refusals


def test_refusals(ta, ctx, ex):
    """What the entry points refuse on the device's side of the checks (the
    shapes' own are unit-tested without a GPU)."""
    other = ta.Context()
    ex2 = ta.Executor(other, n_slots=1, tune=False)
    q, out = ex.tensor([4, 2, 64]), ex.tensor([4, 2, 64])
    kt, v = ex.tensor([2, 64, 32]), ex.tensor([2, 32, 64])
    cache, d = ex.q8_cache(2, 64, 32), ta.TreeAttentionDesc(8, 4, 0.125)
    mask = ta.U32Cell(ctx, 8)

    def refuses(match, f):
        with pytest.raises(ta.TensorAshError, match=match):
            f()

    refuses("q and out must be different", lambda: ex.q8_tree_attention(q, cache, q, d, mask))
    refuses("kt and out must be different", lambda: ex.tree_attention(q, kt, v, kt, d, mask))
    refuses("different HIP context", lambda: ex.q8_tree_attention(q, ex2.q8_cache(2, 64, 32), out, d, mask))
    refuses("different", lambda: ex.q8_tree_attention(q, cache, out, d, ta.U32Cell(other, 8)))
    refuses("mask holds", lambda: ex.q8_tree_attention(q, cache, out, d, ta.U32Cell(ctx, 7)))
    refuses("kt and v must be different", lambda: ex.q8_cache_read(cache, kt, kt, ta.Q8ReadDesc(4)))
    refuses("different HIP context",
            lambda: ex.q8_cache_write(q, q, ex2.q8_cache(2, 64, 32), ta.Q8WriteDesc(4)))
    refuses("unsupported", lambda: ex.q8_cache(2, 32, 32))
    refuses("nonzero", lambda: ex.q8_cache(0, 64, 32))
    table, pos = ex.tensor([40, 32, 2]), ta.U32Cell(ctx, 4)
    refuses("table and output", lambda: ex.rope_axes(table, table, pos, table, ta.RopeAxesDesc(1, 64, 64, [32])))
    refuses("positions hold", lambda: ex.rope_axes(q, table, pos, q, ta.RopeAxesDesc(2, 64, 64, [16, 16])))
    refuses("needs ta_exec_op_v2", lambda: ta._check(ta.lib.ta_run_exec_ops(
        ex.handle, ta.C.byref(ta._ExecOp(kind=ta.EXEC_TREE_ATTENTION)), 1, None)))
    refuses("cache is null", lambda: ex.run_exec_ops(
        [ta.ExecOp(ta.EXEC_Q8_CACHE_WRITE, inp=[q, q], more=dict(q8_write=ta.Q8WriteDesc(4)._raw()))]))
    refuses("both set", lambda: ex.run_exec_ops(
        [ta.ExecOp(ta.EXEC_TREE_ATTENTION, inp=[q, kt, v], out=out, more=dict(q8=cache.handle, tree=d._raw()))]))
    bad = d._raw()
    bad.reserved = 1
    refuses("reserved", lambda: ta._check(ta.lib.ta_q8_tree_attention(
        ex.handle, q.handle, cache.handle, None, out.handle, ta.C.byref(bad), None)))
    ex.q8_tree_attention(q, cache, out, d, mask)  # and the good call still runs
