"""xtg_hip_attention_ext against attention in 64 bits (tests/kv4_oracle.py), element by element, within what its
roundings allow: caches of every dtype, rings, windows, documents, prefixes, rows that see nothing, capped scores, a
distance bias, BF16 and FP32 rows, one row to several hundred."""
import numpy as np
import pytest

import kv4_oracle as o

pytestmark = pytest.mark.gpu


class Call:
    """A cache filled to ctx, the rows of a call, and what the call's keys are in 64 bits."""

    def __init__(self, hip, rng, dtype, n, ctx, heads, kvh, d, ring=0, x_dtype=o.BF16, spread=1.0, own=True, slots=None):
        self.hip, self.n, self.ctx, self.heads, self.kvh, self.d, self.x = hip, n, ctx, heads, kvh, d, x_dtype
        self.dtype, self.own = dtype, own
        kc, vc = self.unit(rng, (ctx, kvh, d)), rng.standard_normal((ctx, kvh, d)).astype(np.float32)
        q = self.unit(rng, (n, heads, d)) * np.float32(d * spread)
        k, v = self.unit(rng, (n, kvh, d)), rng.standard_normal((n, kvh, d)).astype(np.float32)
        self.cache = None
        p0 = max(0, ctx - ring) if ring else 0
        if dtype != "none":
            self.cache = hip.kv_cache(kvh, d, slots or ctx + n, ring, o.KV[dtype])
            if ctx:
                self.fill(p0, kc[p0:], vc[p0:])
        self.set(p0, kc[p0:], vc[p0:], q, k, v)

    @staticmethod
    def unit(rng, shape):
        x = rng.standard_normal(shape).astype(np.float32)
        return x / np.linalg.norm(x, axis=-1, keepdims=True)

    def fill(self, p, k, v):
        a = [self.hip.array(np.ascontiguousarray(x, np.float32)) for x in (k, v)]
        self.cache.write(p, len(k), a[0], a[1])
        self.hip.finish()
        for x in a:
            x.free()

    def set(self, p0, kc, vc, q, k, v):
        """The cached rows (from position p0) and the call's rows, FP32; q, k and v mean their BF16 values."""
        cached = o.stored_pair(kc, vc, self.dtype) if self.cache is not None else (kc[:0].astype(np.float64), vc[:0])
        if self.own:
            keys = [np.concatenate([c, o.bf16(x)]) for c, x in zip(cached, (k, v))]
            self.at = np.concatenate([p0 + np.arange(len(cached[0])), self.ctx + np.arange(self.n)])
        else:
            keys, self.at = cached, p0 + np.arange(len(cached[0]))
        self.q, self.keys = o.bf16(q), keys
        self.dev = [self.hip.array(o.rows(x, self.x)[0]) for x in (q, k, v)]
        self.out = self.hip.array(shape=q.shape, dtype=np.uint16 if self.x else np.float32)

    def queue(self, pos0=None, window=0, scale=None, softcap=0.0, slopes=None, first=None, end=None):
        self.extra = [self.hip.array(np.ascontiguousarray(x, t)) if x is not None else None
                      for x, t in ((slopes, np.float32), (first, np.int32), (end, np.int32))]
        k, v = self.dev[1:] if self.own else (None, None)
        self.hip.attention_ext(self.cache, self.dev[0], k, v, self.out, self.n, self.ctx if pos0 is None else pos0,
                               self.heads, self.kvh, self.d, self.x, window, scale, softcap, *self.extra)

    def result(self):
        y = self.out.numpy()
        return o.bf16_values(y) if self.x else y

    def run(self, **kw):
        self.out.upload(np.full(self.out.shape, 0x7fc1 if self.x else np.nan, self.out.dtype))
        self.queue(**kw)
        return self.result()

    def check(self, pos0=None, scale=None, **kw):
        got = self.run(pos0=pos0, scale=scale, **kw)
        out, size, most = o.attend(self.q, *self.keys, self.at, self.ctx if pos0 is None else pos0,
                                   self.d ** -0.5 if scale is None else scale, **kw)
        bits = 11 if self.dtype == "nvfp4" and not self.own else 8
        finite = np.isfinite(out)
        np.testing.assert_array_equal(got[~finite], out[~finite].astype(np.float32))
        off = np.abs(got.astype(np.float64)[finite] - out[finite])
        tol = o.tolerance(out, size, most, self.d, bits, self.x)[finite]
        assert (off <= tol).all(), "off by %.3g of %.3g" % (off[off > tol].max(), tol[off > tol].max())
        return got

    def free(self):
        for x in self.dev + [self.out] + [e for e in getattr(self, "extra", []) if e is not None]:
            x.free()
        if self.cache is not None:
            self.cache.destroy()


HEADS = {64: (16, 8), 128: (8, 2), 256: (4, 2)}
# over 768 (row, q head of a KV head) pairs the call's work-groups share tiles; these groups of heads bring few rows there
MANY = {64: (32, 1), 128: (64, 2), 256: (32, 1)}


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("n,ctx", [(1, 0), (1, 1), (1, 31), (1, 700), (2, 33), (5, 1), (8, 300), (17, 64), (37, 1001),
                                   (130, 257), (64, 3)])
def test_plain_scores(hip, d, dtype, n, ctx):
    c = Call(hip, np.random.default_rng(n * 1000 + ctx + d), dtype, n, ctx if dtype != "none" else 0, *HEADS[d], d)
    c.check()
    c.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("n,ctx", [(25, 1), (26, 64), (33, 80), (40, 321), (130, 33)])
def test_plain_scores_of_many(hip, d, dtype, n, ctx):
    """The cache ends with the context: for 64 and 128 dims also in the middle of a tile of 64 keys."""
    c = Call(hip, np.random.default_rng(n * 1000 + ctx + d), dtype, n, ctx if dtype != "none" else 0, *MANY[d], d,
             slots=ctx)
    c.check()
    c.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(slopes=True), dict(slopes=True, softcap=30.0, window=70)])
def test_changed_scores_of_many(hip, d, dtype, kw):
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = np.linspace(0.01, 0.5, MANY[d][0])
    c = Call(hip, np.random.default_rng(d), dtype, 30, 200 if dtype != "none" else 0, *MANY[d], d, spread=5.0)
    c.check(**kw)
    c.free()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8"])
@pytest.mark.parametrize("n,ctx", [(1, 3000), (2, 8200)])
def test_more_than_sixteen_records(hip, d, dtype, n, ctx):
    """A decoded token over a long cache, whose records several groups of lanes join."""
    c = Call(hip, np.random.default_rng(ctx + d), dtype, n, ctx, *HEADS[d], d)
    hip.profile()
    c.check()
    names = hip.profile_report()
    hip.profile(False)
    assert "ext_merge_kernel<%d, %d, %d>" % (d, o.KV[dtype], 1024 // d) in names, names
    c.check(softcap=8.0, slopes=np.linspace(0.001, 0.01, c.heads))
    c.check(first=np.full(n, ctx - 40))   # most records saw nothing
    c.free()


@pytest.mark.parametrize("n,heads", [(1, 8), (7, 8), (45, 8), (50, 64)])
def test_weights_over_an_nvfp4_cache_keep_eleven_bits(hip, n, heads):
    """FP32 rows out and no keys of the call's own: half a step of f16's weights is the bound that decides."""
    c = Call(hip, np.random.default_rng(n), "nvfp4", n, 600, heads, 2, 128, x_dtype=o.F32, own=False)
    c.check(pos0=600 - n)
    c.check(pos0=500, softcap=9.0, window=100)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("n,heads", [(1, 8), (20, 8), (45, 64)])
def test_the_first_and_last_key_of_a_span(hip, dtype, n, heads):
    """The keys at both ends of what a row sees and beside them outweigh all others, so that one too many or too few shows."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 0 if dtype == "none" else 3000, 2, 128
    n = n if dtype != "none" else n + 3000
    c = Call(hip, rng, dtype, n, ctx, heads, kvh, d, slots=ctx)
    u = c.unit(rng, (1, 1, d))
    kc, vc = c.unit(rng, (ctx, kvh, d)), rng.standard_normal((ctx, kvh, d)).astype(np.float32)
    k, v = c.unit(rng, (n, kvh, d)), rng.standard_normal((n, kvh, d)).astype(np.float32)
    q = np.repeat(np.repeat(u * d, n, 0), heads, 1).astype(np.float32)
    both, vals = np.concatenate([kc, k]), np.concatenate([vc, v])
    spans = [(1023, 2048), (1000, 1001), (31, 2977)] + ([(2990, 3000)] if ctx else [])
    for lo, hi in spans:
        for p in (lo - 1, lo, hi - 1, hi):
            both[p] = u
        vals[lo - 1], vals[hi] = 50.0, -50.0
    if ctx:
        c.fill(0, both[:ctx], vals[:ctx])
    for x in c.dev + [c.out]:
        x.free()
    c.set(0, both[:ctx], vals[:ctx], q, both[ctx:], vals[ctx:])
    if dtype == "none":   # (rows enough for any kernel; a few of them are looked at)
        c.q = c.q[-3:]
    for lo, hi in spans:
        if ctx:
            c.check(first=np.full(n, lo), end=np.full(n, hi))
        else:
            got = c.run(first=np.full(n, lo), end=np.full(n, hi))[-3:]
            out, size, most = o.attend(c.q, *c.keys, c.at, n - 3, d ** -0.5, first=np.full(3, lo), end=np.full(3, hi))
            assert (np.abs(got - out) <= o.tolerance(out, size, most, d, 8, c.x)).all()
    c.free()


def test_key_splits_of_many(hip):
    """Enough tiles to be split over work-groups, with a window and documents that leave some of them without keys."""
    c = Call(hip, np.random.default_rng(5), "nvfp4", 32, 3000, 64, 2, 128)
    c.check()
    c.check(window=500)
    c.check(first=np.full(32, 2990), softcap=5.0)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("n,ctx", [(1, 500), (6, 129), (45, 400)])
@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(softcap=3.0, window=50), dict(slopes=True), dict(window=16),
                                dict(slopes=True, softcap=30.0, window=100)])
def test_changed_scores(hip, dtype, n, ctx, kw):
    d, kw = 128, dict(kw)
    heads, kvh = 12, 4
    if kw.get("slopes"):
        kw["slopes"] = 2.0 ** (-8.0 * (np.arange(heads) + 1) / heads)
    c = Call(hip, np.random.default_rng(n + ctx), dtype, n, ctx if dtype != "none" else 0, heads, kvh, d, spread=5.0)
    c.check(**kw)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "fp8"])
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_changed_scores_other_heads(hip, dtype, d, n):
    c = Call(hip, np.random.default_rng(d + n), dtype, n, 333, *HEADS[d], d, spread=5.0)
    c.check(softcap=15.0, slopes=np.linspace(0.01, 0.5, HEADS[d][0]))
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "none"])
@pytest.mark.parametrize("n,heads", [(3, 8), (90, 8), (300, 8), (26, 64), (150, 64)])
def test_documents_prefixes_and_padding(hip, dtype, n, heads):
    """first / end as packed documents, prefixes seen both ways, padding rows (nothing), ends before the row, and
    values outside of every position."""
    rng = np.random.default_rng(n)
    ctx = 150 if dtype != "none" else 0
    c = Call(hip, rng, dtype, n, ctx, heads, 2, 128)
    cuts = np.sort(rng.integers(0, n, 4))
    start = np.array([max([0] + [ctx + x for x in cuts if x <= i and x > 0]) for i in range(n)])
    c.check(first=start)
    end = np.maximum(ctx + np.arange(n) + 1, ctx + n // 2)
    c.check(end=end)
    c.check(first=start, end=end, window=40, softcap=9.0)
    lo, hi = rng.integers(-5, ctx + n, n), rng.integers(-5, ctx + n + 50, n)
    lo[n // 2:], hi[n // 2:] = 0, 0   # padding
    got = c.check(first=lo, end=hi)
    assert not got[n // 2:].any()
    lo[:] = 2 ** 31 - 1
    assert not c.check(first=lo).any()
    hi[:] = -2 ** 31
    assert not c.check(end=hi).any()
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8"])
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("n,ctx,ring,window", [(1, 500, 96, 90), (8, 77, 96, 64), (8, 1000, 103, 0), (60, 400, 160, 100),
                                               (1, 95, 96, 0), (26, 150, 90, 70)])
def test_rings(hip, dtype, heads, n, ctx, ring, window):
    c = Call(hip, np.random.default_rng(ctx), dtype, n, ctx, heads, 2, 128, ring=ring)
    c.check(window=window)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8"])
@pytest.mark.parametrize("n,heads", [(1, 8), (7, 8), (50, 8), (50, 64)])
def test_rows_already_stored(hip, dtype, n, heads):
    """k and v NULL: the call's rows are among the cached ones, also at positions from pos0 on."""
    c = Call(hip, np.random.default_rng(n), dtype, n, 200, heads, 2, 128, own=False)
    c.check(pos0=200 - n)
    c.check(pos0=100)   # rows in the middle: later positions are masked
    c.check(pos0=100, end=np.full(n, 150), softcap=5.0)
    c.free()


def test_stale_slots_are_not_seen(hip):
    """Slots at or past pos0 (a rewound session) and slots never written."""
    c = Call(hip, np.random.default_rng(3), "nvfp4", 4, 300, 8, 2, 128, slots=500)
    keep = (c.at < 180) | (np.arange(len(c.at)) >= 300)
    c.keys, c.at = [k[keep] for k in c.keys], c.at[keep]
    c.at[180:] = 180 + np.arange(4)
    c.check(pos0=180)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16"])
@pytest.mark.parametrize("n,heads", [(2, 8), (33, 8), (33, 64)])
def test_fp32_rows(hip, dtype, n, heads):
    c = Call(hip, np.random.default_rng(n), dtype, n, 210, heads, 2, 128, x_dtype=o.F32)
    c.check()
    c.check(softcap=4.0, window=60)
    c.free()


@pytest.mark.parametrize("heads,kvh", [(1, 1), (3, 1), (40, 2), (32, 1), (5, 5)])
@pytest.mark.parametrize("n", [1, 19])
def test_head_groups(hip, heads, kvh, n):
    c = Call(hip, np.random.default_rng(heads), "nvfp4", n, 100, heads, kvh, 128)
    c.check()
    c.free()


@pytest.mark.parametrize("scale", [4.0, -0.3, 0.0])
@pytest.mark.parametrize("n,heads", [(1, 8), (40, 8), (40, 64)])
def test_scales_and_sharp_softmaxes(hip, scale, n, heads):
    c = Call(hip, np.random.default_rng(8), "nvfp4", n, 300, heads, 2, 128)
    c.check(scale=scale)
    c.check(scale=scale, softcap=50.0)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("scale", [1e4, 1e6, 1e8, 1e10, 1e30])
@pytest.mark.parametrize("n,heads", [(2, 8), (45, 8), (26, 64), (150, 64)])
def test_scores_beyond_the_integers_of_fp32(hip, dtype, scale, n, heads):
    """Scores up to 1e32 of either sign, whose last bits are worth far more than an exponential's range: one key stands out
    by half of them, and its value is the output."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 0 if dtype == "none" else 300, 2, 128
    c = Call(hip, rng, dtype, n, ctx, heads, kvh, d)
    u = c.unit(rng, (1, 1, d))
    q = np.repeat(np.repeat(u * d, n, 0), heads, 1).astype(np.float32)
    vc, v = (rng.standard_normal((m, kvh, d)).astype(np.float32) for m in (ctx, n))
    for sign in (1, -1):   # the best key: the largest score, or the one least below zero
        kc, k = (np.repeat(np.repeat((0.5 if sign > 0 else -1.0) * u, m, 0), kvh, 1).astype(np.float32) for m in (ctx, n))
        (kc if ctx else k)[0] = (1.0 if sign > 0 else -0.5) * u
        if ctx:
            c.fill(0, kc, vc)
        for x in c.dev + [c.out]:
            x.free()
        c.set(0, kc, vc, q, k, v)
        want = np.repeat(c.keys[1][0], heads // kvh, 0)
        for kw in (dict(), dict(slopes=np.full(heads, 0.01)), dict(window=n + 200 if ctx else 0, first=np.zeros(n))):
            got = c.run(scale=scale, **kw)
            if kw.get("window"):   # the best key is out of the window: all are alike
                assert np.isfinite(got).all() and (np.abs(got) <= np.abs(c.keys[1]).max()).all()
            else:   # half a step of a weight of 8 bits (or of its product with an FP8 value's scale), and of a BF16 output
                assert (np.abs(got - want) <= np.abs(want) * (2.0 ** -7 + 2.0 ** -14)).all()
    c.free()


@pytest.mark.parametrize("cap", [1e-38, 1e-3, 1024.0])
@pytest.mark.parametrize("n,heads", [(2, 8), (26, 64)])
def test_tiny_and_large_caps(hip, cap, n, heads):
    c = Call(hip, np.random.default_rng(n), "nvfp4", n, 300, heads, 2, 128)
    c.check(softcap=cap)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8", "none"])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 40])
@pytest.mark.parametrize("n,heads", [(2, 8), (45, 8), (26, 64)])
def test_a_tiny_cap_with_large_queries_and_keys_of_zeros(hip, dtype, size, n, heads):
    """What a product is multiplied by passes FP32 and has to stay finite: a key of zeros has a score of zero. All scores
    are within 1e-38 of it, so the weights are equal (tolerances count no error of a score)."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 0 if dtype == "none" else 120, 2, 128
    c = Call(hip, rng, dtype, n, ctx, heads, kvh, d)
    kc, vc = c.unit(rng, (ctx, kvh, d)), rng.standard_normal((ctx, kvh, d)).astype(np.float32)
    q = c.unit(rng, (n, heads, d)) * np.float32(d * size)
    k, v = c.unit(rng, (n, kvh, d)), rng.standard_normal((n, kvh, d)).astype(np.float32)
    kc[::3], k[::2] = 0.0, 0.0
    if ctx:
        c.fill(0, kc, vc)
    for x in c.dev + [c.out]:
        x.free()
    c.set(0, kc, vc, q, k, v)
    got = c.run(softcap=1e-38)
    out, weight, _ = o.attend(c.q, *c.keys, c.at, ctx, d ** -0.5, softcap=1e-38)
    off = np.abs(got.astype(np.float64) - out)
    assert (off <= o.tolerance(out, weight, 0.0, d, 8, c.x)).all()
    c.free()


@pytest.mark.parametrize("x_dtype", [o.F32, o.BF16])
@pytest.mark.parametrize("globs", [(2.0 ** 60, 2.0 ** -60), (2.0 ** -60, 2.0 ** 60), (0.25, 8.0)])
@pytest.mark.parametrize("n,heads", [(2, 8), (40, 8), (50, 64)])
def test_globals(hip, x_dtype, globs, n, heads):
    """Keys and values at an NVFP4 cache's globals, the call's rows among them; the scale undoes the keys'."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 300, 2, 128
    c = Call(hip, rng, "nvfp4", n, 0, heads, kvh, d, own=False, slots=ctx, x_dtype=x_dtype)
    kc, vc = (x.astype(np.float32) for x in (c.unit(rng, (ctx, kvh, d)) * globs[0],
                                              rng.standard_normal((ctx, kvh, d)) * globs[1]))
    c.cache.globals(*globs)
    c.fill(0, kc, vc)
    c.keys, c.at = o.stored_pair(kc, vc, "nvfp4", globs), np.arange(ctx)
    c.check(pos0=ctx - n, scale=d ** -0.5 / globs[0])
    c.check(pos0=100, scale=-0.5 / globs[0], softcap=5.0, window=80)
    c.free()


@pytest.mark.parametrize("size", [2.0 ** -127, 2.0 ** -100, 2.0 ** 40])
@pytest.mark.parametrize("n,heads", [(2, 8), (26, 64)])
def test_tiny_and_huge_queries(hip, size, n, heads):
    """Queries near both ends of BF16's exponents: scores that vanish, and scores of one at a scale that undoes them."""
    c = Call(hip, np.random.default_rng(n), "nvfp4", n, 300, heads, 2, 128, spread=size)
    c.check(scale=128 ** -0.5 if size < 1 else 2.0 ** -46)
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("up", [114, -114])
@pytest.mark.parametrize("n,heads", [(2, 8), (45, 8), (26, 64)])
def test_huge_queries_over_small_keys(hip, dtype, up, n, heads):
    """Queries and keys near opposite ends of BF16's exponents, whose products are ordinary: an FP8 key's codes are, times
    such a query without the key's scale, beyond FP32."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 300, 2, 128
    c = Call(hip, rng, dtype, n, 0, heads, kvh, d, own=False, slots=ctx)
    kc, vc = c.unit(rng, (ctx, kvh, d)) * np.float32(2.0 ** -up), rng.standard_normal((ctx, kvh, d)).astype(np.float32)
    q = c.unit(rng, (n, heads, d)) * np.float32(d * 2.0 ** up)
    c.fill(0, kc, vc)
    for x in c.dev + [c.out]:
        x.free()
    c.set(0, kc, vc, q, kc[:n], vc[:n])
    c.check(pos0=ctx - n)
    c.check(pos0=ctx - n, softcap=5.0, window=90)
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8"])
@pytest.mark.parametrize("n,heads", [(1, 8), (6, 8), (70, 8), (26, 64)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(hip, dtype, n, heads):
    """NaN and infinities in cached keys and values outside of the rows' windows, inside of some, and in the call's own
    rows, seen by later rows only."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 120, 2, 128
    c = Call(hip, rng, dtype, n, ctx, heads, kvh, d)
    kc, vc = c.unit(rng, (ctx, kvh, d)), rng.standard_normal((ctx, kvh, d)).astype(np.float32)
    q = c.unit(rng, (n, heads, d)) * d
    k, v = c.unit(rng, (n, kvh, d)), rng.standard_normal((n, kvh, d)).astype(np.float32)
    vc[20, 0, 3], kc[21, 1, 4], vc[22, 1, 9] = np.nan, np.nan, np.inf if dtype != "fp8" else np.nan
    if dtype != "fp8":   # its scale would be infinite, and the whole row NaN
        vc[ctx - 3, 0, 5], vc[ctx - 2, 0, 5], vc[ctx - 2, 0, 6] = np.inf, -np.inf, -np.inf
    if n > 3:
        v[n - 3, 1, 2], v[n - 2, 0, 1], k[n - 2, 1, 0] = np.nan, np.inf, np.nan
    c.fill(0, kc, vc)
    for x in c.dev + [c.out]:
        x.free()
    with np.errstate(all="ignore"):
        c.set(0, kc, vc, q, k, v)
        if dtype == "fp8":
            for x, raw in zip(c.keys, (kc, vc)):
                x[:ctx][~np.isfinite(raw)] = np.nan
    c.check(window=30)                    # row i sees from ctx + i - 29 on
    c.check(first=np.full(n, ctx - 1))    # no cached one that is not finite
    c.check()
    c.free()


@pytest.mark.parametrize("dtype", ["bf16", "none"])
@pytest.mark.parametrize("n,heads", [(1, 8), (6, 8), (70, 8), (26, 64), (40, 64)])
def test_rows_whose_scores_are_all_minus_infinity(hip, dtype, n, heads):
    """Such a row is NaN, as its formula is (only a row that sees nothing is zeros); with one other key it is that key's."""
    rng = np.random.default_rng(n)
    ctx, kvh, d = 0 if dtype == "none" else 700, 2, 128
    c = Call(hip, rng, dtype, n, ctx, heads, kvh, d, slots=ctx + n)
    kc, vc = c.unit(rng, (ctx, kvh, d)), rng.standard_normal((ctx, kvh, d)).astype(np.float32)
    q = c.unit(rng, (n, heads, d)) * d
    k, v = c.unit(rng, (n, kvh, d)), rng.standard_normal((n, kvh, d)).astype(np.float32)
    q[..., 0], kc[..., 0] = 1.0, -np.inf
    if dtype == "none":
        k[0, :, 0] = -np.inf
    else:
        c.fill(0, kc, vc)
    for x in c.dev + [c.out]:
        x.free()
    c.set(0, kc, vc, q, k, v)
    got = c.check()
    if dtype == "none":
        assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()
    else:
        assert np.isfinite(got).all()
        assert np.isnan(c.check(end=np.full(n, ctx))).all()
        assert not c.check(first=np.full(n, ctx), end=np.full(n, ctx)).any()
    c.free()


@pytest.mark.parametrize("dtype", ["nvfp4", "bf16", "fp8"])
@pytest.mark.parametrize("n,heads", [(1, 8), (45, 8), (26, 64)])
def test_positions_that_the_cache_does_not_hold(hip, dtype, n, heads):
    """Rows may see positions that were never written: they see nothing there."""
    c = Call(hip, np.random.default_rng(n), dtype, n, 0, heads, 2, 128, slots=900)
    c.at = 800 + np.arange(n)
    assert not c.check(pos0=800, end=np.full(n, 800)).any()
    c.check(pos0=800)
    c.free()


@pytest.mark.parametrize("n,heads", [(1, 8), (5, 8), (66, 8), (26, 64)])
def test_captured_and_replayed(hip, n, heads):
    """A graph of a write, an attention and a read, replayed with eager work between the replays."""
    rng = np.random.default_rng(n)
    c = Call(hip, rng, "nvfp4", n, 900, heads, 2, 128, slots=1100)
    k2, v2 = hip.array(shape=(n, 2, 128), dtype=np.uint16), hip.array(shape=(n, 2, 128), dtype=np.uint16)
    slopes = np.linspace(0.1, 0.2, heads)
    want = c.check(softcap=10.0, slopes=slopes)
    hip.graph_begin()
    c.hip.attention_ext(c.cache, *c.dev, c.out, n, 900, heads, 2, 128, o.BF16, 0, None, 10.0, c.extra[0])
    c.cache.write(900, n, c.dev[1], c.dev[2], o.BF16)
    c.cache.read(900, n, k2, v2, o.BF16)
    g = hip.graph_end("ext")
    stored = o.stored_pair(*(o.bf16_values(x.numpy()) for x in c.dev[1:]), "nvfp4")
    other = Call(hip, rng, "bf16", 33, 50, 8, 2, 128)
    for _ in range(4):
        c.out.upload(np.full(c.out.shape, 0x7fc1, np.uint16))
        k2.upload(np.zeros(k2.shape, np.uint16))
        hip.graph_launch(g)
        np.testing.assert_array_equal(c.result(), want)
        for a, w in zip((k2, v2), stored):
            np.testing.assert_array_equal(o.bf16_values(a.numpy()), w.astype(np.float32))
        other.check(softcap=3.0)   # eager work on the same scratch
    hip.graph_destroy(g)
    for x in (k2, v2):
        x.free()
    c.free()
    other.free()


@pytest.mark.parametrize("n,heads", [(1, 8), (20, 8), (45, 64)])
def test_captured_at_a_later_position_than_the_first_call(pkg, n, heads):
    """The first call of a shape sizes the scratch for every position of the cache: a session that was warmed up at its
    beginning captures its steps far into it."""
    b = pkg.HipBackend(0)
    c = Call(b, np.random.default_rng(n), "nvfp4", n, 4000, heads, 2, 128, slots=5000)
    c.queue(pos0=3)
    b.finish()
    b.graph_begin()
    c.queue()
    g = b.graph_end("late")
    for _ in range(3):
        c.out.upload(np.full(c.out.shape, 0x7fc1, np.uint16))
        b.graph_launch(g)
        got = c.result()
        np.testing.assert_array_equal(c.check(), got)
    b.graph_destroy(g)
    c.free()
    b.close()


@pytest.mark.parametrize("n,heads", [(1, 8), (20, 8), (45, 64)])
def test_the_last_positions(hip, n, heads):
    """Rows up to position 2^31 - 2, over a ring and over their own keys alone."""
    rng, pos0, ring = np.random.default_rng(n), 2 ** 31 - 1 - n, 96
    c = Call(hip, rng, "nvfp4", n, 0, heads, 2, 128, ring)
    kc, vc = Call.unit(rng, (ring, 2, 128)), rng.standard_normal((ring, 2, 128)).astype(np.float32)
    c.fill(pos0 - ring, kc, vc)
    own = c.keys
    c.keys = [np.concatenate([a, b]) for a, b in zip(o.stored_pair(kc, vc, "nvfp4"), own)]
    c.ctx, c.at = pos0, pos0 - ring + np.arange(ring + n)
    c.check(window=90)
    c.check(end=np.full(n, 2 ** 31 - 1), softcap=5.0)
    c.cache.destroy()
    c.cache, c.keys, c.at = None, own, pos0 + np.arange(n)
    c.check()
    c.free()


def test_a_chunk_of_many_blocks(hip):
    """More blocks of rows than the second axis of a grid has (65535): the rows' keys repeat, so that each full window
    gives what a short call gives."""
    n, heads, d, w = 131100, 64, 64, 7
    rng = np.random.default_rng(1)
    k, v = (np.tile(rng.standard_normal((w, 1, d)).astype(np.float32), (n // w + 1, 1, 1))[:n] for _ in range(2))
    q = Call.unit(rng, (1, heads, d)) * np.float32(d)
    dev = [hip.array(o.rows(x, o.BF16)[0]) for x in (np.repeat(q, n, 0), k, v)]
    out = hip.array(shape=(n, heads, d), dtype=np.uint16)
    hip.attention_ext(None, *dev, out, n, 0, heads, 1, d, o.BF16, w)
    got = out.numpy()
    ref, size, most = o.attend(o.bf16(q), o.bf16(k[:w]), o.bf16(v[:w]), np.arange(w), w - 1, d ** -0.5, w)
    tol = o.tolerance(ref, size, most, d, 8, o.BF16)
    for at in range(w - 1, n, 8192):
        rows = o.bf16_values(got[at:at + 8192])
        assert (np.abs(rows - ref) <= tol).all(), at
    for x in dev + [out]:
        x.free()


def test_the_same_call_twice_is_the_same(hip):
    for n, ctx, kw in ((1, 3000, {}), (33, 2000, dict(softcap=8.0)), (200, 1000, {}), (700, 900, dict(window=100))):
        c = Call(hip, np.random.default_rng(n), "nvfp4", n, ctx, 16, 4, 128)
        a = c.run(**kw)
        for _ in range(3):
            np.testing.assert_array_equal(c.run(**kw), a)
        c.free()


def test_two_backends_at_once(hip, pkg):
    """Two handles' calls queued one behind the other do not share workspaces."""
    b = pkg.HipBackend(0)
    calls = [Call(x, np.random.default_rng(i), "nvfp4", 9, 1500, 8, 2, 128) for i, x in enumerate((hip, b))]
    want = [c.check(softcap=6.0) for c in calls]
    for _ in range(5):
        for c in calls:
            c.queue(softcap=6.0)
    for c, w in zip(calls, want):
        np.testing.assert_array_equal(c.result(), w)
        c.free()
    b.close()


def test_decode_loop_as_it_is_used(hip):
    """A prompt in chunks, then tokens one by one: each call attends and then writes its rows (a ring beside a linear
    cache), against 64 bits over what the caches hold."""
    rng = np.random.default_rng(11)
    heads, kvh, d, total, ring, window = 8, 2, 128, 180, 96, 32
    k, v = Call.unit(rng, (total, kvh, d)), rng.standard_normal((total, kvh, d)).astype(np.float32)
    q = Call.unit(rng, (total, heads, d)) * d
    caches = [hip.kv_cache(kvh, d, total, 0, 2), hip.kv_cache(kvh, d, 0, ring, 2)]
    sk, sv = o.stored_pair(o.bf16(k), o.bf16(v), "nvfp4")
    p = 0
    while p < total:
        n = 50 if p < 150 else 1
        dev = [hip.array(o.bf16_bits(x[p:p + n])) for x in (q, k, v)]
        out = hip.array(shape=(n, heads, d), dtype=np.uint16)
        for cache, w in zip(caches, (0, window)):
            hip.attention_ext(cache, *dev, out, n, p, heads, kvh, d, o.BF16, w, softcap=7.0)
            cache.write(p, n, dev[1], dev[2], o.BF16)
            keys = [np.concatenate([s[:p], o.bf16(x[p:p + n])]) for s, x in ((sk, k), (sv, v))]
            ref, size, most = o.attend(o.bf16(q[p:p + n]), *keys, np.arange(p + n), p, d ** -0.5, w, 7.0)
            off = np.abs(o.bf16_values(out.numpy()) - ref)
            assert (off <= o.tolerance(ref, size, most, d, 8, o.BF16)).all()
        for x in dev + [out]:
            x.free()
        p += n
    for x in caches:
        x.destroy()


def test_refusals(hip, pkg):
    cache = hip.kv_cache(2, 128, 64, 0, 2)
    a = hip.array(shape=(4, 8, 128))
    good = dict(cache=cache, q=a, k=a, v=a, out=hip.array(shape=(4, 8, 128)), n_q=2, pos0=3, heads=8, kv_heads=2,
                head_dim=128)
    hip.attention_ext(**good)
    for change, what in [(dict(n_q=0), "rows at"), (dict(pos0=-1), "rows at"), (dict(pos0=2 ** 31 - 2), "rows at"),
                         (dict(head_dim=96), "head_dim"), (dict(kv_heads=3), "heads over"), (dict(kv_heads=0), "heads over"),
                         (dict(heads=0), "heads over"), (dict(x_dtype=2), "row type"), (dict(scale=float("inf")), "scale"),
                         (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(softcap=1025.0), "softcap"), (dict(q=None), "NULL"),
                         (dict(out=None), "NULL"), (dict(k=None), "both, or neither"), (dict(v=None), "both, or neither"),
                         (dict(cache=None, k=None, v=None), "neither"), (dict(kv_heads=4), "cache of"),
                         (dict(head_dim=64), "cache of"), (dict(q=a.ptr + 8), "16-byte"), (dict(out=a.ptr + 4), "16-byte"),
                         (dict(first=a.ptr + 2), "4-byte"), (dict(n_q=2 ** 27 + 1), "rows of")]:
        with pytest.raises(pkg.XtgError, match=what):
            hip.attention_ext(**dict(good, **change))
    other = hip.kv_cache(2, 128, 64, 0, 2)
    other.destroy()
    hip.finish()
    cache.destroy()


def test_a_destroyed_cache_is_not_no_cache(hip, pkg):
    cache, a, out = hip.kv_cache(2, 128, 64, 0, 2), hip.array(shape=(1, 8, 128)), hip.array(shape=(1, 8, 128))
    hip.attention_ext(cache, a, a, a, out, 1, 3, 8, 2, 128)
    hip.finish()
    cache.destroy()
    with pytest.raises(pkg.XtgError, match="destroyed"):
        hip.attention_ext(cache, a, a, a, out, 1, 3, 8, 2, 128)
    for x in (a, out):
        x.free()
