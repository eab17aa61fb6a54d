"""Paged caches (xtg_hip_paged_append, _read and _attention) against plain forms in 64 bits (tests/kv4_oracle.py), element by
element, within what their roundings allow: every cache dtype and head size, sequences of any length, rows of one token and
of many, rotation and norms, strided rows, windows, pages that are reused, missing or shared, left-out sequences."""
import ctypes
import types

import numpy as np
import pytest

import kv4_oracle as o

pytestmark = pytest.mark.gpu

HEADS = {64: (16, 8), 128: (8, 2), 256: (4, 2)}
DTYPES = ["bf16", "fp8", "nvfp4"]


def unit(rng, shape):
    x = rng.standard_normal(shape).astype(np.float32)
    return x / np.linalg.norm(x, axis=-1, keepdims=True)


def stored_fp8(x):
    """E4M3 codes of x / scale with scale amax * (1 / 448) per (row, head), in FP32 (o.stored_fp8 has the quotient)."""
    x = np.asarray(x, np.float32)
    amax = np.fmax.reduce(np.abs(x), axis=-1, keepdims=True, initial=np.float32(0))
    s = np.where(amax >= np.float32(448 * 2.0 ** -126), amax * (np.float32(1) / np.float32(448)), np.float32(1)).astype(np.float32)
    y = (x * (np.float32(1) / s)).astype(np.float64)
    return np.minimum(o.nearest(np.abs(y), 4, 2.0 ** -9), 448.0) * np.sign(y) * s.astype(np.float64)


def stored_pair(k, v, dtype, globals_=(1.0, 1.0)):
    return (stored_fp8(k), stored_fp8(v)) if dtype == "fp8" else o.stored_pair(k, v, dtype, globals_)


class Pool:
    """A pool and some sequences in it: their pages in no order, and what each of their positions holds, in FP32."""

    def __init__(self, hip, rng, dtype, kvh, d, lengths, page=32, spare=3, globals_=None):
        self.hip, self.rng, self.dtype, self.kvh, self.d, self.page = hip, rng, dtype, kvh, d, page
        need = [max(1, -(-n // page)) for n in lengths]
        self.n_pages, self.max_pages = sum(need) + spare, max(need)
        self.cache = hip.paged_cache(kvh, d, self.n_pages, page, o.KV[dtype])
        self.globals_ = globals_ or (1.0, 1.0)
        if globals_:
            self.cache.globals(*globals_)
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lengths), self.max_pages), -1, np.int32)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = order[at:at + m]
            at += m
        self.spare = order[at:]
        shape = lambda n: (n, kvh, d)   # noqa: E731
        self.k = [np.zeros(shape(n), np.float32) for n in lengths]
        self.v = [np.zeros(shape(n), np.float32) for n in lengths]
        self.dev = []

    def device(self, a, dtype=np.int32):
        self.dev.append(self.hip.array(np.ascontiguousarray(a, dtype)))
        return self.dev[-1]

    def rows(self, pos, n, table=None, n_rows=None, one_each=False):
        """The call's rows: n[s] of sequence s at pos[s] and on."""
        starts = np.concatenate([[0], np.cumsum(n)])
        return self.hip.paged_rows(self.device(pos), self.device(self.table if table is None else table),
                                   int(starts[-1]) if n_rows is None else n_rows, None if one_each else self.device(starts))

    def put(self, pos, n, k, v, x_dtype=o.F32, **kw):
        """Appends rows as they are, and remembers them."""
        a = [self.hip.array(o.rows(x, x_dtype)[0]) for x in (k, v)]
        self.cache.append(self.rows(pos, n, **kw), a[0], a[1], x_dtype)
        at = 0
        for s, (p, m) in enumerate(zip(pos, n)):
            if p >= 0:
                self.k[s][p:p + m], self.v[s][p:p + m] = (o.rows(x, x_dtype)[1][at:at + m] for x in (k, v))
            at += m
        self.hip.finish()
        for x in a:
            x.free()

    def fill(self, lengths=None):
        """Unit keys and values of order one in the first positions of each sequence."""
        n = [len(k) for k in self.k] if lengths is None else lengths
        self.put([0] * len(n), n, unit(self.rng, (sum(n), self.kvh, self.d)),
                 self.rng.standard_normal((sum(n), self.kvh, self.d)).astype(np.float32))

    def held(self, s, n):
        """The stored values of sequence s's first n positions, in 64 bits."""
        return stored_pair(self.k[s][:n], self.v[s][:n], self.dtype, self.globals_)

    def read(self, pos, n, x_dtype=o.F32, **kw):
        shape = (sum(n), self.kvh, self.d)
        a = [self.hip.array(np.full(shape, 0x7fc1 if x_dtype else np.nan, np.uint16 if x_dtype else np.float32)) for _ in "kv"]
        self.cache.read(self.rows(pos, n, **kw), a[0], a[1], x_dtype)
        got = [x.numpy() for x in a]
        for x in a:
            x.free()
        return [o.bf16_values(g) if x_dtype else g for g in got]

    def attend(self, pos, n, heads, x_dtype=o.BF16, spread=1.0, q=None, rows=None, stride=0, before=None, **kw):
        """The call's outputs, with what they should be and how far they may be off."""
        total = sum(n)
        if q is None:
            q = unit(self.rng, (total, heads, self.d)) * np.float32(self.d * spread)
        given, means = o.rows(q, x_dtype)
        means = o.bf16(means)
        if stride:
            wide = np.zeros((total, stride), given.dtype)
            wide[:, :heads * self.d] = given.reshape(total, -1)
            given = wide
        dq = self.hip.array(given)
        out = self.hip.array(np.full((total + 3, heads, self.d), 0x7fc1 if x_dtype else 12345.0, np.uint16 if x_dtype else np.float32))
        rows = rows or self.rows(pos, n)
        self.cache.attention(rows, dq, out, heads, x_dtype, q_stride=stride, **kw)
        got = out.numpy()
        dq.free()
        out.free()
        got = o.bf16_values(got) if x_dtype else got
        assert (got[total:] == 12345.0).all() if not x_dtype else np.isnan(got[total:]).all()   # rows behind the last
        want, tol, at = np.zeros((total, heads, self.d)), np.zeros((total, heads, self.d)), 0
        scale = kw.get("scale")
        more = {x: kw[x] for x in ("window", "softcap") if x in kw}
        for s, (p, m) in enumerate(zip(pos, n)):
            if p >= 0 and m:
                k, v = self.held(s, p + m)
                if before is not None:
                    k, v = before(s, k, v)
                w, size, most = o.attend(means[at:at + m], k, v, np.arange(p + m), p, self.d ** -0.5 if scale is None else scale, **more)
                want[at:at + m] = w
                tol[at:at + m] = o.tolerance(w, size, most, self.d, 11 if self.dtype == "nvfp4" else 8, x_dtype)
            at += m
        return got[:total], want, tol

    def check(self, *a, **kw):
        same(*self.attend(*a, **kw))

    def free(self):
        self.hip.finish()
        for x in self.dev:
            x.free()
        self.cache.destroy()


def same(got, want, tol):
    finite = np.isfinite(want)
    np.testing.assert_array_equal(got[~finite], want[~finite].astype(np.float32))
    off = np.abs(got.astype(np.float64)[finite] - want[finite])
    bad = ~(off <= tol[finite])
    assert not bad.any(), "%d of %d off by up to %.3g of %.3g" % (bad.sum(), bad.size, np.nanmax(off[bad]), tol[finite][bad].max())


# --------------------------------------------------------------------------------------------- rows in and back


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("x_dtype", [o.F32, o.BF16])
def test_rows_appended_and_read_back(hip, d, dtype, x_dtype):
    """Rows of several sequences, in pieces that begin and end inside tiles and pages: exactly what a cache of this dtype
    holds of them, and nothing else is touched."""
    rng = np.random.default_rng(d + x_dtype)
    lengths = [1, 33, 32, 100, 0, 71]
    p = Pool(hip, rng, dtype, 3, d, lengths, page=64)
    done = [0] * len(lengths)
    while any(a < b for a, b in zip(done, lengths)):
        n = [min(b - a, int(rng.choice([0, 1, 1, 3, 31, 50]))) for a, b in zip(done, lengths)]
        shape = (sum(n), 3, d)
        size = np.float32(2.0) ** rng.integers(-3, 4, (shape[0], 3, 1)).astype(np.float32)
        p.put(done, n, rng.standard_normal(shape).astype(np.float32) * size, rng.standard_normal(shape).astype(np.float32) / size,
              x_dtype)
        done = [a + m for a, m in zip(done, n)]
    want = [p.held(s, m) for s, m in enumerate(lengths)]
    for x in (o.F32, o.BF16):
        for i, got in enumerate(p.read([0] * len(lengths), lengths, x)):
            w = np.concatenate([y[i] for y in want]).astype(np.float32)
            np.testing.assert_array_equal(got, o.bf16(w) if x else w)
    # a span in the middle of each
    pos, n = [0, 5, 31, 40, 0, 33], [1, 9, 1, 33, 0, 38]
    for i, got in enumerate(p.read(pos, n)):
        w = np.concatenate([y[i][a:a + m] for y, a, m in zip(want, pos, n)]).astype(np.float32)
        np.testing.assert_array_equal(got, w)
    p.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_decode_step_of_many_sequences(hip, d, dtype):
    """One row each, more sequences than a wave has lanes, some left out; twice, so that slots of a word are filled by
    different calls."""
    rng = np.random.default_rng(d)
    lengths = [int(x) for x in rng.integers(3, 90, 70)]
    p = Pool(hip, rng, dtype, 2, d, lengths)
    for back in (3, 2, 1):
        pos = [m - back if s % 7 else -1 for s, m in enumerate(lengths)]
        shape = (len(lengths), 2, d)
        p.put(pos, [1] * len(lengths), rng.standard_normal(shape).astype(np.float32), rng.standard_normal(shape).astype(np.float32),
              one_each=True)
    for i, got in enumerate(p.read([m - 3 for m in lengths], [3] * len(lengths))):
        w = np.concatenate([p.held(s, m)[i][m - 3:] for s, m in enumerate(lengths)]).astype(np.float32)
        np.testing.assert_array_equal(got, w)
    p.free()


def rotated(x, at, theta):
    """x [n][heads][d] turned by positions at, in 64 bits, and the sum of the terms' magnitudes."""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    angle = np.asarray(at, np.float64)[:, None, None] * np.float64(np.float32(theta)) ** (-np.arange(half) / half)
    c, s, a, b = np.cos(angle), np.sin(angle), x[..., :half], x[..., half:]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([size, size], -1)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("x_dtype", [o.F32, o.BF16])
@pytest.mark.parametrize("theta,norm,scaled", [(1e4, False, False), (1e7, True, True), (0.0, True, False), (1.0, False, True)])
def test_rotation_and_norm(hip, d, dtype, x_dtype, theta, norm, scaled):
    """q and k turned by their rows' positions, far ones among them, and normalised per head, q scaled. Bounds: sine and
    cosine are within 2^-23 and products and sums round by 2^-24 each, so a turned value is within 2^-21 of its terms; the
    norm's sum of d squares and its root add (d + 8) * 2^-24 of the value; a row type or a cache rounds once more."""
    rng = np.random.default_rng(d + x_dtype)
    heads, kvh = HEADS[d]
    pos, n, page = [0, 1000, 65000, 40], [3, 40, 2, 1], 4096
    p = Pool(hip, rng, dtype, kvh, d, [5, 1100, 65010, 50], page=page)
    total = sum(n)
    q, k, v = (rng.standard_normal((total, h, d)).astype(np.float32) for h in (heads, kvh, kvh))
    qscale = rng.uniform(0.5, 1.5, heads * d).astype(np.float32)
    given = [hip.array(o.rows(x, x_dtype)[0]) for x in (q, k, v)]
    out, sc = hip.array(np.zeros_like(o.rows(q, x_dtype)[0])), hip.array(qscale)
    rows = p.rows(pos, n)
    p.cache.append(rows, given[1], given[2], x_dtype, given[0], out, heads, theta, norm, sc if scaled else None)
    at = np.concatenate([a + np.arange(m) for a, m in zip(pos, n)])

    def exact(x, scale=None):
        x = o.rows(x, x_dtype)[1].astype(np.float64)
        y, size = rotated(x, at, theta) if theta else (x, np.abs(x))
        tol = size * 2.0 ** -21
        if norm:
            f = 1.0 / np.sqrt((y * y).sum(-1, keepdims=True) + 1e-6)
            y, tol = y * f, tol * f + np.abs(y * f) * ((d + 8) * 2.0 ** -24)
        if scale is not None:
            s = scale.astype(np.float64).reshape(1, -1, d)
            y, tol = y * s, tol * s + np.abs(y * s) * 2.0 ** -24
        return y, tol
    y, tol = exact(q, qscale if scaled else None)
    got = out.numpy()
    got = o.bf16_values(got) if x_dtype else got
    off = np.abs(got - y)
    bound = tol + (np.abs(y) + tol) * (2.0 ** -8 if x_dtype else 2.0 ** -24)
    assert (off <= bound).all(), (off / bound).max()
    y, tol = exact(k)
    amax = np.abs(y).max(-1, keepdims=True)
    if dtype == "bf16":
        bound = tol + (np.abs(y) + tol) * 2.0 ** -8
    elif dtype == "fp8":   # half a step of the code, 2^-4 of it or 2^-10 of the scale, which is off by as much as amax
        bound = 2 * tol + np.maximum(np.abs(y) * 2.0 ** -4, amax / 448 * 2.0 ** -10) * (1 + 2.0 ** -4) + amax * 2.0 ** -20
    else:   # a block's scale is its amax / 6 to within 2^-4; the widest step is 2 of it
        block = np.abs(y).reshape(*y.shape[:-1], d // 16, 16).max(-1, keepdims=True)
        block = np.broadcast_to(block, (*block.shape[:-1], 16)).reshape(y.shape)
        bound = 2 * tol + block / 6 * (1 + 2.0 ** -4) + 2.0 ** -10
    got_k, got_v = p.read(pos, n)
    off = np.abs(got_k - y)
    assert (off <= bound).all(), (off / bound).max()
    np.testing.assert_array_equal(got_v, stored_pair(o.rows(v, x_dtype)[1], o.rows(v, x_dtype)[1], dtype)[1].astype(np.float32))
    for x in given + [out, sc]:
        x.free()
    p.free()


def test_strided_rows_and_q_in_place(hip):
    """q, k and v as parts of one wide row each, q turned where it lies; what is between the rows stays."""
    rng = np.random.default_rng(8)
    heads, kvh, d, n = 8, 2, 128, 37
    wide = (heads + 2 * kvh) * d + 8
    p = Pool(hip, rng, "bf16", kvh, d, [60], page=32)
    x = rng.standard_normal((n, wide)).astype(np.float32)
    bits = o.bf16_bits(x)
    a = hip.array(bits)
    rows = p.rows([20], [n])
    p.cache.append(rows, a.ptr + 2 * heads * d, a.ptr + 2 * (heads + kvh) * d, o.BF16, a.ptr, a.ptr, heads, 1e4,
                   q_stride=wide, k_stride=wide, v_stride=wide)
    after = a.numpy()
    np.testing.assert_array_equal(after[:, heads * d:], bits[:, heads * d:])
    x = o.bf16(x)
    y, size = rotated(x[:, :heads * d].reshape(n, heads, d), 20 + np.arange(n), 1e4)
    off = np.abs(o.bf16_values(after[:, :heads * d]).reshape(n, heads, d) - y)
    assert (off <= size * 2.0 ** -21 + np.abs(y) * 2.0 ** -8 * 1.0001).all()
    k, v = p.read([20], [n])
    y, size = rotated(x[:, heads * d:(heads + kvh) * d].reshape(n, kvh, d), 20 + np.arange(n), 1e4)
    assert (np.abs(k - y) <= size * 2.0 ** -21 + np.abs(y) * 2.0 ** -8 * 1.0001).all()
    np.testing.assert_array_equal(v, x[:, (heads + kvh) * d:-8].reshape(n, kvh, d))
    a.free()
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_page(hip, dtype):
    """Positions whose table entry is no page, or behind the table, are not stored and read as zeros; q is turned all the
    same. Rows behind the last sequence, and a left-out sequence's, are left as they were."""
    rng = np.random.default_rng(4)
    kvh, d, heads = 2, 64, 4
    p = Pool(hip, rng, dtype, kvh, d, [64, 64, 64], page=32, spare=2)
    p.fill()
    before = p.read([0, 0, 0], [64, 64, 64])
    table = p.table.copy()
    table[0, 1], table[1, 0] = -1, p.n_pages   # the first's second page, the second's first
    pos, n = [30, 31, -1], [4, 40, 5]          # the second's rows 64 .. 70 are behind its table
    total = sum(n)
    q, k, v = (rng.standard_normal((total + 6, h, d)).astype(np.float32) for h in (heads, kvh, kvh))
    dev = [hip.array(x) for x in (q, k, v)]
    rows = p.rows(pos, n, table=table, n_rows=total + 6)
    p.cache.append(rows, dev[1], dev[2], o.F32, dev[0], dev[0], heads, 1e4)
    got = dev[0].numpy()
    live = total - 5
    at = np.concatenate([30 + np.arange(4), 31 + np.arange(40)])
    y, size = rotated(q[:live], at, 1e4)
    assert (np.abs(got[:live] - y) <= size * 2.0 ** -20).all()
    np.testing.assert_array_equal(got[live:], q[live:])
    after = p.read([0, 0, 0], [64, 64, 64])
    for x, b in zip(after, before):   # the first's 30, 31 and the second's 32 .. 63 are new
        new = np.zeros(192, bool)
        new[[30, 31]] = True
        new[64 + 32:128] = True
        np.testing.assert_array_equal(x[~new], b[~new])
        assert (x[new] != b[new]).any(axis=(1, 2)).all()
    out = [hip.array(np.full((total + 6, kvh, d), 7.0, np.float32)) for _ in "kv"]
    p.cache.read(rows, out[0], out[1])
    for x, b in zip(out, after):
        x = x.numpy()
        want = np.zeros((live, kvh, d), np.float32)
        want[:2], want[4 + 1:4 + 33] = b[30:32], b[64 + 32:128]
        np.testing.assert_array_equal(x[:live], want)
        assert (x[live:] == 7.0).all()
    for x in dev + out:
        x.free()
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite(hip, dtype):
    """A row with a NaN reads back as a cache of this dtype reads it; its neighbours in the same words are as they were."""
    rng = np.random.default_rng(5)
    kvh, d = 2, 128
    p = Pool(hip, rng, dtype, kvh, d, [64], page=32)
    k, v = (rng.standard_normal((64, kvh, d)).astype(np.float32) for _ in "kv")
    k[10, 0, 3], v[17, 1, 100] = np.nan, np.nan
    p.put([0], [64], k, v)
    for got, w in zip(p.read([0], [64]), p.held(0, 64)):
        np.testing.assert_array_equal(got, w.astype(np.float32))
    p.free()


def test_globals_of_a_pool(hip, pkg):
    rng = np.random.default_rng(6)
    p = Pool(hip, rng, "nvfp4", 2, 64, [50, 20], globals_=(2.0 ** -6, 8.0))
    p.fill()
    for i, got in enumerate(p.read([0, 0], [50, 20])):
        np.testing.assert_array_equal(got, np.concatenate([p.held(s, m)[i] for s, m in enumerate((50, 20))]).astype(np.float32))
    p.check([49, 19], [1, 1], 8)
    with pytest.raises(pkg.XtgError, match="has been written"):
        p.cache.globals(1.0, 1.0)
    p.free()


# ------------------------------------------------------------------------------------------------- attention


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(), dict(window=40), dict(softcap=20.0, spread=4.0), dict(softcap=9.0, window=1, spread=4.0)])
def test_one_token_each(hip, d, dtype, kw):
    """A decode step: lengths of one to some hundred positions, left-out sequences among them."""
    rng = np.random.default_rng(d)
    lengths = [1, 2, 31, 32, 33, 64, 65, 700, 5, 300]
    p = Pool(hip, rng, dtype, HEADS[d][1], d, lengths, page=64)
    p.fill()
    pos = [m - 1 for m in lengths]
    pos[8] = -1
    rows = p.rows(pos, [1] * len(pos), one_each=True)
    p.check(pos, [1] * len(pos), HEADS[d][0], rows=rows, **kw)
    p.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(), dict(window=50), dict(softcap=20.0, spread=4.0)])
def test_rows_of_any_number(hip, d, dtype, kw):
    """Decoded tokens, verify steps, turns and prompts in one call; sequences without rows and left-out ones."""
    rng = np.random.default_rng(d + 1)
    n = [1, 8, 0, 37, 1, 130, 3, 1, 90]
    pos = [200, 0, 50, 33, 0, 70, -1, 511, -7]
    p = Pool(hip, rng, dtype, HEADS[d][1], d, [max(0, a) + m for a, m in zip(pos, n)], page=32)
    p.fill()
    p.check(pos, n, HEADS[d][0], **kw)
    p.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_long_sequence_is_split(hip, d, dtype):
    """One token over 9000 positions, alone and beside short ones; rows of a verify step over as many."""
    rng = np.random.default_rng(d + 2)
    p = Pool(hip, rng, dtype, HEADS[d][1], d, [9000, 40, 1, 3000], page=128)
    p.fill()
    heads = HEADS[d][0]
    p.check([8999, 39, 0, 2999], [1, 1, 1, 1], heads)
    p.check([8990, 38, 0, 2900], [5, 1, 1, 30], heads)
    p.check([8990, 38, 0, 2900], [5, 1, 1, 30], heads, window=4000, softcap=30.0, spread=3.0)
    p.free()


@pytest.mark.parametrize("heads,kvh", [(1, 1), (3, 1), (6, 2), (17, 1), (40, 2), (128, 1), (5, 5)])
def test_head_groups(hip, heads, kvh):
    rng = np.random.default_rng(heads)
    p = Pool(hip, rng, "fp8", kvh, 64, [500, 70, 9], page=32)
    p.fill()
    p.check([499, 69, 8], [1, 1, 1], heads, rows=p.rows([499, 69, 8], [1, 1, 1], one_each=True))
    p.check([480, 0, 1], [19, 70, 8], heads)
    p.free()


@pytest.mark.parametrize("d,page", [(64, 32), (64, 64), (128, 32), (128, 4096), (256, 32), (256, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_over_pages_of_any_size(hip, d, page, dtype):
    """Blocks of 128 q-cols whose tiles of 64 keys are one page's or two's, from the first position on and after some; FP32
    rows too, whose output is turned in two passes."""
    rng = np.random.default_rng(d + page)
    n, pos = [260, 33, 1], [0, 95, 40]
    p = Pool(hip, rng, dtype, HEADS[d][1], d, [a + m for a, m in zip(pos, n)], page=page)
    p.fill()
    p.check(pos, n, HEADS[d][0])
    p.check(pos, n, HEADS[d][0], x_dtype=o.F32, window=70)
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_prompt_chunk_over_a_long_context(hip, dtype, d):
    """Blocks of many q-cols whose keys are split over work-groups, and joined."""
    rng = np.random.default_rng(d + 3)
    heads, kvh = {64: 8, 128: 8, 256: 4}[d], 1
    p = Pool(hip, rng, dtype, kvh, d, [5000, 600], page=64)
    p.fill()
    p.check([4980, 599], [20, 1], heads)
    p.check([4980, 560], [20, 40], heads, softcap=15.0, spread=3.0)
    p.free()


def test_prompt_blocks_with_rows_that_end_in_different_tiles(hip):
    """A group of one q head: a block of 128 q-cols is 128 rows, over four tiles' diagonals."""
    rng = np.random.default_rng(19)
    p = Pool(hip, rng, "bf16", 2, 64, [700, 300])
    p.fill()
    p.check([300, 0], [400, 300], 2)
    p.check([300, 0], [400, 300], 2, window=33)
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e4, 1e8, 1e10])
@pytest.mark.parametrize("n", [1, 40])
def test_scores_beyond_the_integers_of_fp32(hip, dtype, scale, n):
    """Scores so large that one key takes all the weight: its value comes back. Keys whose scores are further from the best
    than its rounding (2^-24 of it and more) count for nothing."""
    rng = np.random.default_rng(int(scale) % 1000 + n)
    p = Pool(hip, rng, dtype, 2, 64, [200 + n])
    p.fill()
    q = unit(rng, (n, 8, 64)) * np.float32(64)
    got, want, _ = p.attend([200], [n], 8, q=q, scale=scale, x_dtype=o.F32)
    k, v = p.held(0, 200 + n)
    for i in range(n):
        for h in range(8):
            s = k[:201 + i, h // 4] @ o.bf16(q[i, h]).astype(np.float64)
            top = np.sort(s)[-2:]
            if (top[1] - top[0]) * scale > 200 + abs(top[1]) * scale * 2.0 ** -18:
                assert np.abs(got[i, h] - v[s.argmax(), h // 4]).max() <= np.abs(v[s.argmax(), h // 4]).max() * 2.0 ** -8
    assert np.isfinite(got).all()
    p.free()


def test_more_sequences_than_lanes(hip):
    """200 sequences of any length, most of one token: the prefix sums go over several waves' widths."""
    rng = np.random.default_rng(9)
    pos = [int(x) for x in rng.integers(-1, 300, 200)]
    n = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 9], 200)]
    p = Pool(hip, rng, "bf16", 2, 64, [max(0, a) + m for a, m in zip(pos, n)])
    p.fill()
    p.check(pos, n, 8)
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_fp32_rows_and_strides(hip, dtype):
    rng = np.random.default_rng(10)
    p = Pool(hip, rng, dtype, 2, 128, [90, 300])
    p.fill()
    p.check([80, 299], [10, 1], 8, x_dtype=o.F32)
    p.check([80, 299], [10, 1], 8, x_dtype=o.F32, stride=8 * 128 + 4)
    p.check([80, 299], [10, 1], 8, stride=12 * 128)
    p.check([80, 299], [10, 1], 8, scale=-0.3)
    p.check([80, 299], [10, 1], 8, scale=0.0)
    p.free()


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_reused_pages_hold_nothing_of_their_past(hip, d, dtype):
    """Every page full of rows that are NaN and infinite; then sequences begin in them and grow."""
    rng = np.random.default_rng(d)
    heads, kvh = HEADS[d]
    p = Pool(hip, rng, dtype, kvh, d, [100, 100, 100], page=64, spare=0)
    old = np.full((384, kvh, d), np.nan, np.float32)
    old[::2, :, ::3] = np.inf
    a = hip.array(old)
    whole = np.arange(p.n_pages, dtype=np.int32).reshape(1, -1)
    p.cache.append(hip.paged_rows(p.device([0]), p.device(whole), 384, p.device([0, 384])), a, a)
    hip.finish()
    a.free()
    p.fill([1, 37, 64])
    p.check([0, 36, 63], [1, 1, 1], heads)
    p.check([0, 20, 60], [1, 17, 4], heads)
    p.check([0, 20, 60], [1, 17, 4], heads, window=10)
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx,heads", [(40, 8), (3000, 8), (40, 64)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(hip, dtype, ctx, heads):
    rng = np.random.default_rng(ctx)
    n, kvh, d = 12, 2, 64
    p = Pool(hip, rng, dtype, kvh, d, [ctx + n, 90])
    p.fill()
    k, v = (x[0][ctx + 5:ctx + 6].copy() for x in (p.k, p.v))
    v[0, 1, 7] = np.nan
    p.put([ctx + 5, -1], [1, 0], k, v)
    got, want, tol = p.attend([ctx, 60], [n, 30], heads)
    if dtype == "fp8":   # a NaN among an FP8 row's values is one element's
        assert np.isnan(want[5:n, heads // 2:, 7]).all()
    assert np.isfinite(got[:5]).all() and np.isfinite(got[:n, :heads // 2]).all()
    seen = np.isnan(want)
    assert np.isnan(got[seen]).all() and np.isfinite(want[n:]).all()
    same(got[~seen], want[~seen], tol[~seen])
    # behind a window it is nobody's
    p.check([ctx + 9, 60], [3, 30], heads, window=3)
    p.free()


def test_scores_of_minus_infinity_alone_are_nan(hip):
    rng = np.random.default_rng(12)
    p = Pool(hip, rng, "bf16", 1, 64, [50, 50])
    p.fill()
    p.put([0, -1], [50, 0], np.full((50, 1, 64), 1e38, np.float32), rng.standard_normal((50, 1, 64)).astype(np.float32))
    q = np.full((4, 1, 64), 1.0, np.float32)
    q[:2] = -3e38
    got, want, tol = p.attend([48, 48], [2, 2], 1, q=q)
    assert np.isnan(got[:2]).all()
    same(got[2:], want[2:], tol[2:])
    p.free()


def test_positions_without_a_page_are_nan(hip):
    """... for the rows that see them: not behind a window, and not where nothing of the page is seen."""
    rng = np.random.default_rng(13)
    kvh, d, heads = 2, 128, 8
    p = Pool(hip, rng, "bf16", kvh, d, [300, 300, 40], page=32)
    p.fill()
    table = p.table.copy()
    table[0, 2], table[1, 1] = -1, 10 ** 6
    pos, n = [290, 20, 30], [9, 60, 3]
    got, want, tol = p.attend(pos, n, heads, rows=p.rows(pos, n, table=table))
    assert np.isnan(got[:9]).all()
    assert np.isnan(got[9 + 12:9 + 60]).all()   # from position 32 on
    clear = np.r_[9:21, 69:72]
    same(got[clear], want[clear], tol[clear])
    got, want, tol = p.attend(pos, n, heads, rows=p.rows(pos, n, table=table), window=16)
    clear = np.r_[0:9, 9:21, 9 + 64 - 20 + 15:9 + 60, 69:72]
    assert np.isnan(got[9 + 12:9 + 44]).all()
    same(got[clear], want[clear], tol[clear])
    # rows behind the table's last position
    short = np.ascontiguousarray(p.table[:, :2])
    got, want, tol = p.attend(pos, n, heads, rows=p.rows(pos, n, table=short))
    assert np.isnan(got[:9]).all() and np.isnan(got[9 + 44:69]).all()
    same(got[9:9 + 44], want[9:9 + 44], tol[9:9 + 44])
    # sixteen and more parts, one of them without its page
    p.free()
    p = Pool(hip, rng, "bf16", kvh, d, [9000, 9000], page=32)
    p.fill()
    table = p.table.copy()
    table[0, 100] = -1
    got, want, tol = p.attend([8999, 8999], [1, 1], heads, rows=p.rows([8999, 8999], [1, 1], table=table))
    assert np.isnan(got[0]).all()
    same(got[1:], want[1:], tol[1:])
    p.free()


def test_shared_pages(hip):
    """Two sequences over one prefix, whose pages are in both tables."""
    rng = np.random.default_rng(14)
    p = Pool(hip, rng, "fp8", 2, 64, [96, 96], page=32)
    p.fill()
    p.table[1, :2] = p.table[0, :2]
    p.k[1][:64], p.v[1][:64] = p.k[0][:64], p.v[0][:64]
    p.check([95, 95], [1, 1], 8)
    p.check([60, 64], [30, 32], 8)
    p.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_follows_its_arrays(hip, dtype):
    """A decode step of append and attention captured once and replayed as the sequences grow, end, and begin in reused
    pages: each replay is bit for bit the step run eagerly."""
    rng = np.random.default_rng(15)
    kvh, heads, d, s = 2, 8, 64, 5
    p = Pool(hip, rng, dtype, kvh, d, [120] * s, page=32, spare=6)
    p.fill([40, 64, 31, 90, 1])
    pos, table = p.device([0] * s), p.device(p.table)
    rows = hip.paged_rows(pos, table)
    shape = lambda h: (s, h, d)   # noqa: E731
    dev = [hip.array(np.zeros(shape(h), np.uint16)) for h in (heads, kvh, kvh, heads, heads)]

    def step():
        p.cache.append(rows, dev[1], dev[2], o.BF16, dev[0], dev[3], heads, 1e4, True)
        p.cache.attention(rows, dev[3], dev[4], heads, o.BF16, 50)
    step()   # sizes scratch
    hip.finish()
    hip.graph_begin()
    step()
    g = hip.graph_end("paged step")
    at = np.array([40, 64, 31, -1, 1])
    for turn in range(6):
        if turn == 3:   # the third ends; its page begins another sequence
            at[2] = 0
            p.table[2] = p.table[2][::-1]
            table.upload(p.table)
        pos.upload(at.astype(np.int32))
        for x, h in zip(dev[:3], (heads, kvh, kvh)):
            x.upload(o.bf16_bits(rng.standard_normal(shape(h))))
        hip.graph_launch(g)
        got = dev[3].numpy(), dev[4].numpy()
        for x in dev[3:]:
            x.upload(np.zeros(shape(heads), np.uint16))
        step()   # the same rows to the same places
        for a, b, live in zip(got, (dev[3].numpy(), dev[4].numpy()), (at >= 0, at >= -1)):
            np.testing.assert_array_equal(a[live], b[live])
        assert np.isfinite(o.bf16_values(got[1])).all() and (got[1][3] == 0).all()
        at[at >= 0] += 1
    hip.graph_destroy(g)
    for x in dev:
        x.free()
    p.free()


def test_two_captured_graphs_share_the_scratch(hip):
    rng = np.random.default_rng(16)
    p = Pool(hip, rng, "bf16", 2, 128, [5000, 4000], page=64)
    p.fill()
    calls = []
    for pos, n in (([4999, 3999], [1, 1]), ([4900, 3000], [20, 3])):
        q = hip.array(o.bf16_bits(unit(rng, (sum(n), 8, 128)) * np.float32(100)))
        out = hip.array(shape=(sum(n), 8, 128), dtype=np.uint16)
        rows = p.rows(pos, n)
        p.cache.attention(rows, q, out, 8, o.BF16)
        calls.append((rows, q, out, out.numpy()))
    graphs = []
    for rows, q, out, _ in calls:
        hip.graph_begin()
        p.cache.attention(rows, q, out, 8, o.BF16)
        graphs.append(hip.graph_end("attention"))
    for turn in range(3):
        for _, _, out, _ in calls:
            out.upload(np.zeros(out.shape, np.uint16))
        for g in graphs if turn % 2 else graphs[::-1]:
            hip.graph_launch(g)
        for _, _, out, want in calls:
            np.testing.assert_array_equal(out.numpy(), want)
    for g in graphs:
        hip.graph_destroy(g)
    for _, q, out, _ in calls:
        q.free()
        out.free()
    p.free()


def test_a_run_of_steps_is_attention_over_the_whole(hip):
    """Prompts appended and attended in one call, then steps of one token: each row sees what came before, turned and
    normalised as one pass in 64 bits does it."""
    rng = np.random.default_rng(17)
    kvh, heads, d, theta = 2, 8, 128, 1e6
    total = [45, 70, 33]
    p = Pool(hip, rng, "bf16", kvh, d, total, page=32)
    q, k, v = ([rng.standard_normal((m, h, d)).astype(np.float32) for m in total] for h in (heads, kvh, kvh))

    def normed(x, at):
        y = rotated(o.bf16(x), at, theta)[0]
        return y / np.sqrt((y * y).sum(-1, keepdims=True) + 1e-6)
    keys = [normed(x, np.arange(len(x))) for x in k]
    done, scale = [0, 0, 0], float(d) ** 0.5
    for n in ([40, 65, 28], [1, 1, 1], [1, 1, 1], [3, 3, 3]):
        part = [np.concatenate([x[a:a + m] for x, a, m in zip(y, done, n)]) for y in (q, k, v)]
        dev = [hip.array(o.bf16_bits(x)) for x in part] + [hip.array(shape=part[0].shape, dtype=np.uint16) for _ in "qo"]
        rows = p.rows(done, n)
        p.cache.append(rows, dev[1], dev[2], o.BF16, dev[0], dev[3], heads, theta, True)
        p.cache.attention(rows, dev[3], dev[4], heads, o.BF16, scale=scale)
        got, at = o.bf16_values(dev[4].numpy()), 0
        for s, (a, m) in enumerate(zip(done, n)):
            # q and k are rounded to BF16 after the norm: each score is then off by up to 2 * 2^-8 of |q| |k| * scale
            w, size, _ = o.attend(normed(q[s][a:a + m], a + np.arange(m)), keys[s][:a + m], o.bf16(v[s][:a + m]), np.arange(a + m), a, scale)
            e = 2 * 2.0 ** -8 * scale * 1.01 + 2.0 ** -8
            assert (np.abs(got[at:at + m] - w) <= size[0] * (np.exp(2 * e) - 1) + np.abs(w) * 2.0 ** -7 + 1e-6).all()
            at += m
        done = [a + m for a, m in zip(done, n)]
        for x in dev:
            x.free()
    p.free()


def test_offsets_beyond_32_bits(hip):
    """A pool of more than 2^32 bytes and elements of K: pages at its end."""
    rng = np.random.default_rng(18)
    kvh, d, page = 8, 256, 4096
    pages = 2 ** 32 // (kvh * d * page) + 2
    c = hip.paged_cache(kvh, d, pages, page, o.KV["fp8"])
    n = 40
    k, v = unit(rng, (n, kvh, d)), rng.standard_normal((n, kvh, d)).astype(np.float32)
    dev = [hip.array(x) for x in (k, v)]
    arrays = [hip.array(np.array(x, np.int32)) for x in ([0], [[pages - 1]], [0, n], [n - 1], [[0]])]
    rows = hip.paged_rows(arrays[0], arrays[1], n, arrays[2])
    c.append(rows, dev[0], dev[1])
    out = [hip.array(shape=(n, kvh, d)) for _ in "kv"]
    c.read(rows, out[0], out[1])
    want = stored_pair(k, v, "fp8")
    for x, w in zip(out, want):
        np.testing.assert_array_equal(x.numpy(), w.astype(np.float32))
    q = unit(rng, (1, 16, d)) * np.float32(d)
    dq, y = hip.array(o.bf16_bits(q)), hip.array(shape=(1, 16, d), dtype=np.uint16)
    c.attention(hip.paged_rows(arrays[3], arrays[1]), dq, y, 16, o.BF16)
    w, size, most = o.attend(o.bf16(q), *want, np.arange(n), n - 1, d ** -0.5)
    same(o.bf16_values(y.numpy()), w, o.tolerance(w, size, most, d, 8, o.BF16))
    c.read(hip.paged_rows(arrays[0], arrays[4], n, arrays[2]), out[0], out[1])   # page 0 is as it was
    assert all((x.numpy() == 0).all() for x in out)
    for x in dev + out + arrays + [dq, y]:
        x.free()
    c.destroy()


def test_refusals(hip, pkg):
    kvh, d = 2, 64
    with pytest.raises(pkg.XtgError, match="power of two"):
        hip.paged_cache(kvh, d, 4, 48)
    with pytest.raises(pkg.XtgError, match="power of two"):
        hip.paged_cache(kvh, d, 4, 16)
    with pytest.raises(pkg.XtgError, match="head_dim 96"):
        hip.paged_cache(kvh, 96, 4)
    with pytest.raises(pkg.XtgError, match="pages"):
        hip.paged_cache(kvh, d, 0)
    with pytest.raises(pkg.XtgError, match="unknown KV dtype"):
        hip.paged_cache(kvh, d, 4, dtype=5)
    c = hip.paged_cache(kvh, d, 4, 32)
    with pytest.raises(pkg.XtgError, match="not an NVFP4"):
        c.globals(1.0, 1.0)
    pos, table, starts = (hip.array(np.array(x, np.int32)) for x in ([0, 0], [[0, 1], [2, 3]], [0, 3, 5]))
    k, q = hip.array(shape=(5, kvh, d)), hip.array(shape=(5, 8, d))
    rows = hip.paged_rows(pos, table, 5, starts)
    with pytest.raises(pkg.XtgError, match="without starts"):
        c.append(hip.paged_rows(pos, table, 5), k, k)
    with pytest.raises(pkg.XtgError, match=r"\[n_seqs\]\[max_pages\]"):
        hip.paged_rows(pos, pos)
    with pytest.raises(pkg.XtgError, match="pos has 2 elements"):
        hip.paged_rows(pos, hip_table(hip, 3))
    with pytest.raises(pkg.XtgError, match="not of the call's int32"):
        hip.paged_rows(k, table)
    with pytest.raises(pkg.XtgError, match="k has"):
        c.append(rows, hip.array(shape=(4, kvh, d)), k)
    with pytest.raises(pkg.XtgError, match="not of the call's row type BF16"):
        c.append(rows, k, k, pkg.X_BF16)
    with pytest.raises(pkg.XtgError, match="both, or neither"):
        c.append(rows, k, k, q=q, heads=8)
    with pytest.raises(pkg.XtgError, match="scale without q"):
        c.append(rows, k, k, qscale=q)
    with pytest.raises(pkg.XtgError, match="theta 0.5"):
        c.append(rows, k, k, theta=0.5)
    with pytest.raises(pkg.XtgError, match="stride of 100"):
        c.append(rows, q, k, k_stride=100)
    with pytest.raises(pkg.XtgError, match="multiple of 16 bytes"):
        c.append(rows, q, k, k_stride=130)
    with pytest.raises(pkg.XtgError, match="16-byte aligned"):
        c.append(rows, k.ptr + 4, k.ptr)
    with pytest.raises(pkg.XtgError, match="over 2 KV heads"):
        c.attention(rows, q, q, 5)
    with pytest.raises(pkg.XtgError, match="softcap"):
        c.attention(rows, q, q, 8, softcap=2000.0)
    with pytest.raises(pkg.XtgError, match="scale"):
        c.attention(rows, q, q, 8, scale=float("nan"))
    with pytest.raises(pkg.XtgError, match="out has"):
        c.attention(rows, q, k, 8)
    with pytest.raises(pkg.XtgError, match="is not in device memory"):
        c.read(rows, np.zeros((5, kvh, d), np.float32), k)
    wide = hip.array(np.zeros((1, 2 ** 20), np.int32))
    big = hip.paged_cache(1, 64, 1, 4096)
    with pytest.raises(pkg.XtgError, match="2\\^30 positions"):
        big.read(hip.paged_rows(pos, wide), k, k)
    # a pool that does not fit leaves no error behind for the next call
    with pytest.raises(pkg.XtgError, match="hipMalloc"):
        hip.paged_cache(8, 256, 200000, 4096)
    hip.add_norm(k, None, k, 1, 64)
    gone = hip.array(np.zeros(2, np.int32))
    late = hip.paged_rows(gone, table, 2)
    gone.free()
    with pytest.raises(pkg.XtgError, match="have been freed"):
        c.read(late, k, k)
    other = hip.paged_rows(pos, table)
    other.b = types.SimpleNamespace(device=hip.device + 1)
    with pytest.raises(pkg.XtgError, match="not in the memory of the backend's device"):
        c.read(other, k, k)
    # nothing to do is done
    none = hip.paged_rows(pos, table, 0, hip.array(np.zeros(3, np.int32)))
    c.append(none, k, k)
    c.read(none, k, k)
    c.attention(none, q, q, 8)
    c.destroy()
    with pytest.raises(pkg.XtgError, match="NULL argument"):
        c.read(rows, k, k)
    big.destroy()
    for x in (pos, table, starts, k, q, wide):
        x.free()


def hip_table(hip, n):
    return hip.array(np.zeros((n, 2), np.int32))


def test_scratch_is_refused_during_a_capture(pkg):
    b = pkg.HipBackend(0)
    try:
        c = b.paged_cache(1, 64, 4, 32)
        pos, table = b.array(np.zeros(2, np.int32)), b.array(np.array([[0], [1]], np.int32))
        q = b.array(shape=(2, 4, 64))
        out = b.array(shape=(2, 4, 64))
        rows = b.paged_rows(pos, table)
        b.graph_begin()
        with pytest.raises(pkg.XtgError, match="during graph capture"):
            c.attention(rows, q, out, 4)
        with pytest.raises(pkg.XtgError, match="before a graph capture"):
            c.append(rows, q, q, theta=1e4)
        g = b.graph_end("nothing")
        b.graph_destroy(g)
        c.attention(rows, q, out, 4)
        b.graph_begin()
        c.attention(rows, q, out, 4)
        b.graph_destroy(b.graph_end("attention"))
    finally:
        b.close()


def test_the_profiler_names_the_kernels(hip):
    c = hip.paged_cache(2, 64, 16, 32)
    pos, table = hip.array(np.array([300, 7], np.int32)), hip.array(np.arange(32, dtype=np.int32).reshape(2, 16) % 16)
    rows = hip.paged_rows(pos, table)
    kv, q = hip.array(np.zeros((2, 2, 64), np.float32)), hip.array(np.zeros((2, 8, 64), np.float32))
    out = hip.array(shape=(2, 8, 64))
    hip.profile()
    c.append(rows, kv, kv)
    c.read(rows, kv, kv)
    c.attention(rows, q, out, 8)
    names = hip.profile_report()
    hip.profile(False)
    assert {n.split("<")[0]: x["calls"] for n, x in names.items()} == {
        "paged_append_kernel": 1, "paged_read_kernel": 1, "paged_attn_kernel": 1, "paged_merge_kernel": 1}
    c.destroy()
    for x in (pos, table, kv, q, out):
        x.free()


@pytest.mark.parametrize("x_dtype", [1, 0])
def test_fp8_rows_midway_between_codes_and_tiny_ones(hip, x_dtype):
    """Rows whose values lie on the midpoints of their codes (amax 7 u, values M u), which the scale's last bit decides, and
    rows whose scale would be no normal number."""
    kvh, d = 2, 128
    rng = np.random.default_rng(11)
    u = np.repeat([1.0, 3.0, 5.0, 7.0], 2)[:, None, None]
    x = rng.integers(8, 16, (8, kvh, d)) * 2 + 1
    x = (x * u * 2.0 ** -rng.integers(3, 9, (8, kvh, d)) * rng.choice([-1, 1], (8, kvh, d))).astype(np.float32)
    x[..., 5] = 7.0 * u[..., 0]
    x[1] *= np.float32(2.0 ** -130)
    x[3] *= np.float32(2.0 ** -118)
    c = hip.paged_cache(kvh, d, 1, 32, o.KV["fp8"])
    pos, starts, table = (hip.array(np.array(y, np.int32)) for y in ([0], [0, 8], [[0]]))
    rows = hip.paged_rows(pos, table, 8, starts)
    a, want = o.rows(x, x_dtype)
    dev, k, v = hip.array(a), hip.array(shape=x.shape), hip.array(shape=x.shape)
    c.append(rows, dev, dev, x_dtype)
    c.read(rows, k, v)
    hip.finish()
    for got in (k.numpy(), v.numpy()):
        np.testing.assert_array_equal(got, stored_fp8(want).astype(np.float32))
    c.destroy()
    for y in (pos, starts, table, dev, k, v):
        y.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 5, 40])
def test_a_nan_far_below_the_best_score_is_seen_however_the_keys_are_cut(hip, dtype, n):
    """Scores of the first half are 460 base-2 units below the second's, so that a part's factor, and a weight, is zero in
    FP32: a NaN value there is one of every row that sees it, in a call whose blocks are cut into parts as in a call whose
    600 sequences are one part each."""
    rng = np.random.default_rng(20 + n)
    ctx, d, heads = 6000, 64, 4
    p = Pool(hip, rng, dtype, 1, d, [ctx + n], page=64)
    u = unit(rng, (d,))
    k = np.where(np.arange(ctx + n)[:, None, None] < ctx // 2, np.float32(-20) * u, np.float32(20) * u).astype(np.float32)
    v = rng.standard_normal((ctx + n, 1, d)).astype(np.float32)
    v[100, 0, 7] = np.nan
    p.put([0], [ctx + n], k, v)
    q = np.broadcast_to(u * np.float32(d), (n, heads, d)).astype(np.float32)
    got, want, tol = p.attend([ctx], [n], heads, q=q)
    gone = np.isnan(want)
    assert gone.all() if dtype == "nvfp4" else (gone == (np.arange(d) == 7)).all()
    same(got, want, tol)
    many = 600
    dq, out = hip.array(o.bf16_bits(np.tile(q, (many, 1, 1)))), hip.array(shape=(many * n, heads, d), dtype=np.uint16)
    p.cache.attention(p.rows([ctx] * many, [n] * many, table=np.repeat(p.table, many, 0)), dq, out, heads, o.BF16)
    got = o.bf16_values(out.numpy()).reshape(many, n, heads, d)
    same(got[0], want, tol)
    np.testing.assert_array_equal(got, np.broadcast_to(got[:1], got.shape))
    dq.free()
    out.free()
    p.free()


@pytest.mark.parametrize("x_dtype", [o.F32, o.BF16])
def test_queries_at_positions_without_a_page_are_turned_by_them(hip, x_dtype):
    """Up to the last 32-bit position and behind it. An angle is a product of a position and a frequency, both rounded in 64 bits,
    here as in the reference: of 2^31 radians each is off by a few times 2^-22, together by less than 2^-19."""
    rng = np.random.default_rng(21)
    heads, d, theta = 4, 128, 1e4
    pos, n = [2 ** 30 - 2, 2 ** 30 + 12345, 2 ** 31 - 3], [4, 3, 5]
    p = Pool(hip, rng, "bf16", 1, d, [40, 40, 40])
    total = sum(n)
    q, k = (rng.standard_normal((total, h, d)).astype(np.float32) for h in (heads, 1))
    given, means = o.rows(q, x_dtype)
    dev = [hip.array(given), hip.array(o.rows(k, x_dtype)[0])]
    p.cache.append(p.rows(pos, n), dev[1], dev[1], x_dtype, dev[0], dev[0], heads, theta)
    got = dev[0].numpy()
    got = o.bf16_values(got) if x_dtype else got
    y, size = rotated(means, np.concatenate([a + np.arange(m) for a, m in zip(pos, n)]), theta)
    tol = size * 2.0 ** -19
    assert (np.abs(got - y) <= tol + (np.abs(y) + tol) * (2.0 ** -8 if x_dtype else 2.0 ** -24)).all()
    assert all((x == 0).all() for x in p.read([0] * 3, [40] * 3))   # nothing is stored
    for x in dev:
        x.free()
    p.free()


def test_memory_that_is_not_there_is_no_error_of_the_next_call(hip, pkg):
    """What fails is told once: by the call that failed, not by the next launch as well."""
    k = hip.array(np.ones((5, 64), np.float32))
    for _ in range(2):
        with pytest.raises(pkg.XtgError, match="hipMalloc"):
            hip.alloc(1 << 46)
        hip.add_norm(k, None, k, 5, 64)
    with pytest.raises(pkg.XtgError, match="hipMalloc"):
        hip.paged_cache(8, 256, 200000, 4096)
    hip.add_norm(k, None, k, 5, 64)
    np.testing.assert_allclose(k.numpy(), 1 / 8, rtol=1e-5)
    k.free()


def test_more_sequences_than_a_call_takes_are_refused(hip, pkg):
    """Every work-group looks for its piece among all sequences, so a call's time grows with the square of their number."""
    n = 2 ** 14
    c = hip.paged_cache(1, 64, 2, 32)
    arrays = [hip.array(np.zeros(s, np.int32)) for s in ((n + 1,), (n + 1, 1), (n + 2,))]
    x, out = hip.array(np.ones((4, 1, 64), np.float32)), hip.array(shape=(4, 1, 64))
    rows = hip.paged_rows(arrays[0], arrays[1], 4, arrays[2])
    for call in (lambda: c.append(rows, x, x), lambda: c.read(rows, out, out), lambda: c.attention(rows, x, out, 1)):
        with pytest.raises(pkg.XtgError, match="4 rows of 16385 sequences"):
            call()
    # as many as it takes, the last of them with rows
    arrays[2].upload(np.where(np.arange(n + 2) < n, 0, 4).astype(np.int32))
    rows = hip.paged_rows(arrays[0], arrays[1], 4, arrays[2])
    rows.args.n_seqs = n
    c.append(rows, x, x)
    c.attention(rows, x, out, 1)
    np.testing.assert_allclose(out.numpy(), 1.0, rtol=2.0 ** -13)
    c.destroy()
    for a in arrays + [x, out]:
        a.free()


def test_fp8_rows_at_the_least_scale(hip):
    """From an amax of 448 * 2^-126 on rows have a scale, a normal number; below it they are zeros. A code's value there is the
    nearest of FP32's subnormal numbers to its product with the scale."""
    kvh, d = 2, 64
    x = np.random.default_rng(22).uniform(-1, 1, (4, kvh, d)).astype(np.float64)
    x[..., 9] = 1.0
    least = np.float32(448 * 2.0 ** -126)
    amax = np.array([least, np.nextafter(least, np.float32(0)), np.float32(2.0 ** -117), np.float32(2.0 ** -118)])
    x = (x * amax.astype(np.float64)[:, None, None]).astype(np.float32)
    c = hip.paged_cache(kvh, d, 1, 32, o.KV["fp8"])
    arrays = [hip.array(np.array(y, np.int32)) for y in ([0], [[0]], [0, 4])]
    rows = hip.paged_rows(arrays[0], arrays[1], 4, arrays[2])
    dev, k, v = hip.array(x), hip.array(shape=x.shape), hip.array(shape=x.shape)
    c.append(rows, dev, dev)
    c.read(rows, k, v)
    want = stored_fp8(x)
    assert (want[[1, 3]] == 0).all() and (want[[0, 2]] != 0).any(axis=(1, 2)).all()
    for got in (k.numpy(), v.numpy()):
        np.testing.assert_array_equal(got, want.astype(np.float32))
    c.destroy()
    for y in arrays + [dev, k, v]:
        y.free()


def attend_all(q, k, v, pos, scale):
    """o.attend for many rows at once, without a window or a cap: (outputs, the sums of |weight * value| and 2^-32 of the
    |value|s', the largest sum of |q.k| * scale)."""
    n, heads, d = q.shape
    kvh, group = k.shape[1], heads // k.shape[1]
    out, size, floor, most = *(np.zeros((n, heads, d)) for _ in "osf"), 0.0
    hide = np.arange(len(k))[None, None] > (pos + np.arange(n))[:, None, None]
    for h in range(kvh):
        kh, vh, at = k[:, h], v[:, h], slice(h * group, (h + 1) * group)
        x = q[:, at].astype(np.float64).reshape(n * group, d)
        part = np.where(hide, 0, (np.abs(x) @ np.abs(kh).T).reshape(n, group, -1) * scale)
        most = max(most, part.max())
        s = np.where(hide, -np.inf, (x @ kh.T).reshape(n, group, -1) * scale)
        p = np.exp(s - s.max(-1, keepdims=True))
        p = (p / p.sum(-1, keepdims=True)).reshape(n * group, -1)
        out[:, at] = (p @ vh).reshape(n, group, d)
        size[:, at] = (p @ np.abs(vh)).reshape(n, group, d)
        floor[:, at] = (np.where(hide, 0.0, 1.0)[:, 0] @ np.abs(vh))[:, None] * 2.0 ** -32
    return out, (size, floor), most


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,ctx", [(260, 4000), (40, 4000)])
def test_a_chunk_beside_single_tokens_is_joined_by_any_merge(hip, d, dtype, rows, ctx):
    """A chunk over some thousand positions, whose blocks are cut into several parts, beside single tokens: more than 8192
    q-cols (a wave of the merge joins several) and more than 1024 (one each). Then a value in the chunk's last rows is NaN: the
    rows that see it have one, and the others of its tiles, computed again behind the merge, do not."""
    rng = np.random.default_rng(d + rows)
    heads, kvh = 32, 4
    pos, n = [ctx, 900, 30, 2000], [rows, 1, 1, 1]
    p = Pool(hip, rng, dtype, kvh, d, [a + m for a, m in zip(pos, n)], page=64)
    p.fill()
    q = unit(rng, (sum(n), heads, d)) * np.float32(d)
    means = o.bf16(q)
    given, out = hip.array(o.bf16_bits(q)), hip.array(shape=q.shape, dtype=np.uint16)
    call = p.rows(pos, n)

    def attended(last):
        p.cache.attention(call, given, out, heads, o.BF16)
        got, at = o.bf16_values(out.numpy()), 0
        for s, (a, m) in enumerate(zip(pos, n)):
            k, v = (np.nan_to_num(x) for x in p.held(s, a + m))
            w, size, most = attend_all(means[at:at + m], k, v, a, d ** -0.5)
            tol = o.tolerance(w, size, most, d, 11 if dtype == "nvfp4" else 8, o.BF16)
            if s == 0 and last is not None:   # NVFP4: the whole row is NaN for its KV head
                w[last:, heads // 2:heads // 2 + heads // kvh, slice(None) if dtype == "nvfp4" else 7] = np.nan
            same(got[at:at + m], w, tol)
            at += m
    attended(None)
    k, v = (x[0][ctx + rows - 9:ctx + rows - 8].copy() for x in (p.k, p.v))
    v[0, 2, 7] = np.nan
    p.put([ctx + rows - 9, -1, -1, -1], [1, 0, 0, 0], k, v)
    attended(rows - 9)
    given.free()
    out.free()
    p.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
def test_weights_of_single_tokens_have_15_bits(hip, d, dtype):
    """Over BF16 and FP8 pages a weight of a sequence of up to 16 q-cols is a sum of two BF16 values: what the first, which is
    cut, leaves of it, 2^-7, is rounded by 2^-8 of that, and has 2^-17 of the weight more: together less than 2^-14.6."""
    rng = np.random.default_rng(d + 23)
    heads, kvh = HEADS[d]
    lengths = [1, 2, 33, 700, 3000, 500, 64]
    p = Pool(hip, rng, dtype, kvh, d, lengths, page=64)
    p.fill()
    for n, one_each in (([1] * 7, True), ([1, 2, 1, 3, 1, 4, 2], False)):
        pos = [m - x for m, x in zip(lengths, n)]
        q = unit(rng, (sum(n), heads, d)) * np.float32(d)
        given, out = hip.array(q), hip.array(shape=q.shape)
        p.cache.attention(p.rows(pos, n, one_each=one_each), given, out, heads)
        got, at = out.numpy(), 0
        for s, (a, m) in enumerate(zip(pos, n)):
            w, size, most = attend_all(o.bf16(q[at:at + m]), *p.held(s, a + m), a, d ** -0.5)
            same(got[at:at + m], w, o.tolerance(w, size, most, d, 14.6, o.F32))
            at += m
        given.free()
        out.free()
    p.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ctx", [50, 5000])
def test_infinite_values_are_infinite_outputs(hip, d, ctx):
    """Infinities of both signs among BF16 values: an output that one of them takes part in is that infinity, whichever bits its
    weight has; for single tokens, few rows and many."""
    rng = np.random.default_rng(d + ctx)
    heads, kvh = HEADS[d]
    p = Pool(hip, rng, "bf16", kvh, d, [ctx + 40, ctx + 40], page=64)
    p.fill()
    k, v = (x[0][3:43].copy() for x in (p.k, p.v))
    at = rng.integers(0, 40, d - 10)   # dims 10 and on: each one key's
    v[at, 0, np.arange(10, d)] = np.where(rng.integers(0, 2, d - 10), np.inf, -np.inf)
    p.put([3, -1], [40, 0], k, v)
    for n in (1, 2, 40):
        got, want, tol = p.attend([ctx, ctx], [n, 1], heads)
        assert np.isinf(want[:n, 0, 10:]).all()
        same(got, want, tol)
    p.free()
