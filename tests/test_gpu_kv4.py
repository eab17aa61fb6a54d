"""The NVFP4 cache: rows written (FP32 and BF16) and read back, against the format in 64 bits, equal bit for bit."""
import ctypes

import numpy as np
import pytest

import kv4_oracle as o

gpu = pytest.mark.gpu


def write(hip, cache, pos, k, v, x_dtype=o.F32):
    a = [hip.array(o.rows(x, x_dtype)[0]) for x in (k, v)]
    cache.write(pos, k.shape[0], a[0], a[1], x_dtype)
    hip.finish()
    for x in a:
        x.free()


def read(hip, cache, pos, n, x_dtype=o.F32):
    shape = (n, cache.kv_heads, cache.head_dim)
    a = [hip.array(np.full(shape, 0x7fc1 if x_dtype else np.nan, np.uint16 if x_dtype else np.float32)) for _ in "kv"]
    cache.read(pos, n, a[0], a[1], x_dtype)
    got = [x.numpy() for x in a]
    for x in a:
        x.free()
    return [o.bf16_values(g) if x_dtype else g for g in got]


def some_rows(rng, n, kvh, d):
    """Rows whose blocks' magnitudes spread over the whole range of the scales and beyond it."""
    x = rng.standard_normal((n, kvh, d // 16, 16)) * 2.0 ** rng.uniform(-14, 13, (n, kvh, d // 16, 1))
    x[rng.random((n, kvh, d // 16)) < 0.05] = 0.0
    x[rng.random(x.shape) < 0.05] = 0.0
    return x.reshape(n, kvh, d).astype(np.float32)


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("x_dtype", [o.F32, o.BF16])
@pytest.mark.parametrize("n,pos,ring", [(1, 0, 0), (1, 77, 0), (33, 5, 0), (200, 31, 0), (1, 1000, 40), (40, 133, 40),
                                        (37, 91, 40), (100, 7, 40), (97, 1000, 96)])
def test_rows_written_and_read_back(hip, d, x_dtype, n, pos, ring):
    rng = np.random.default_rng(d + n + pos + x_dtype)
    kvh = 3
    k, v = some_rows(rng, n, kvh, d), some_rows(rng, n, kvh, d)
    cache = hip.kv_cache(kvh, d, pos + n + 3, ring, 2)
    write(hip, cache, pos, k, v, x_dtype)
    want = [o.stored_nvfp4(o.rows(x, x_dtype)[1]) for x in (k, v)]
    kept = min(n, ring) if ring else n
    for w in want:
        w[:n - kept] = 0.0   # a ring keeps its last rows; the others read as zeros
    for x in (o.F32, o.BF16):
        for g, w in zip(read(hip, cache, pos, n, x), want):
            np.testing.assert_array_equal(g, w.astype(np.float32))
    # the host's load of a head, of the rows that are held
    hk, hv = cache.load(1, pos + n - kept, pos + n)
    np.testing.assert_array_equal(hk, want[0][n - kept:, 1].astype(np.float32))
    np.testing.assert_array_equal(hv, want[1][n - kept:, 1].astype(np.float32))
    cache.destroy()


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_one_at_a_time_leave_the_others(hip, d):
    """Tokens appended one by one and in threes, over the wrap of a ring that is no multiple of a tile: the codes of
    neighbouring slots share words."""
    rng = np.random.default_rng(d)
    kvh, ring, n = 2, 43, 100
    k, v = some_rows(rng, n, kvh, d), some_rows(rng, n, kvh, d)
    cache = hip.kv_cache(kvh, d, 0, ring, 2)
    p = 0
    while p < n:
        m = min(n - p, 3 if p % 7 == 0 else 1)
        write(hip, cache, p, k[p:p + m], v[p:p + m])
        p += m
    for g, x in zip(read(hip, cache, 0, n), (k, v)):
        want = o.stored_nvfp4(x)
        want[:n - ring] = 0.0
        np.testing.assert_array_equal(g, want.astype(np.float32))
    cache.destroy()


@gpu
def test_midpoints_and_their_neighbours(hip):
    """Values at, one step above and one step below every midpoint of the codes, and block maxima at, above and below
    every midpoint of the scales."""
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    codes = np.arange(127)
    e, m = codes >> 3, codes & 7
    scales = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m * 2.0 ** -9)
    d, blocks = 128, []
    for s in scales[1:]:
        for c in (np.float32(mids * s), np.float32(-mids * s)):
            b = np.concatenate([c, np.nextafter(c, np.float32(np.inf)), [np.float32(6 * s), 0]])
            b2 = np.concatenate([c, np.nextafter(c, np.float32(-np.inf)), [np.float32(-6 * s), 0]])
            blocks += [b, b2]
    top = np.float32((scales[1:] + scales[:-1]) / 2 * 6)
    for t in (top, np.nextafter(top, np.float32(0)), np.nextafter(top, np.float32(np.inf))):
        for x in t:
            blocks.append(np.concatenate([[x], np.float32(np.linspace(-1, 1, 15)) * x]))
    blocks = np.array(blocks, np.float32)
    blocks = np.concatenate([blocks, np.zeros((-len(blocks) % 8, 16), np.float32)]).reshape(-1, 1, d)
    n = len(blocks)
    cache = hip.kv_cache(1, d, n, 0, 2)
    write(hip, cache, 0, blocks, blocks[::-1])
    k, v = read(hip, cache, 0, n)
    np.testing.assert_array_equal(k, o.stored_nvfp4(blocks).astype(np.float32))
    np.testing.assert_array_equal(v, o.stored_nvfp4(blocks[::-1]).astype(np.float32))
    cache.destroy()


@gpu
def test_globals(hip, pkg):
    rng = np.random.default_rng(5)
    n, kvh, d = 50, 2, 64
    k, v = some_rows(rng, n, kvh, d) * np.float32(1e6), some_rows(rng, n, kvh, d) * np.float32(1e-4)
    cache = hip.kv_cache(kvh, d, n, 0, 2)
    cache.globals(2.0 ** 20, 2.0 ** -13)
    write(hip, cache, 0, k, v)
    got = read(hip, cache, 0, n)
    np.testing.assert_array_equal(got[0], o.stored_nvfp4(k, 2.0 ** 20).astype(np.float32))
    np.testing.assert_array_equal(got[1], o.stored_nvfp4(v, 2.0 ** -13).astype(np.float32))
    hk, hv = cache.load(1, 0, n)
    np.testing.assert_array_equal(hk, got[0][:, 1])
    np.testing.assert_array_equal(hv, got[1][:, 1])
    with pytest.raises(pkg.XtgError, match="has been written"):
        cache.globals(1.0, 1.0)
    blob = cache.save()
    other = hip.kv_cache(kvh, d, n, 0, 2)
    with pytest.raises(pkg.XtgError, match="globals"):
        other.restore(blob)
    with pytest.raises(pkg.XtgError, match="globals"):
        cache.copy_to(other)
    other.globals(2.0 ** 20, 2.0 ** -13)
    other.restore(blob)
    for a, b in zip(read(hip, other, 0, n), got):
        np.testing.assert_array_equal(a, b)
    cache.release()
    cache.globals(1.0, 1.0)   # empty again
    assert not read(hip, cache, 0, n)[0].any()
    for c in (cache, other):
        c.destroy()


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_are_not_finite(hip, d):
    """An infinity or a NaN of a head's K or V makes that (position, head) NaN, and leaves its neighbours."""
    rng = np.random.default_rng(d + 9)
    n, kvh = 70, 3
    k, v = some_rows(rng, n, kvh, d), some_rows(rng, n, kvh, d)
    k[3, 0, 5], k[34, 2, d - 1], v[35, 1, 0], v[69, 2, d - 3] = np.inf, np.nan, -np.inf, np.nan
    k[40, 1, 7], v[40, 1, 9] = np.nan, np.inf
    cache = hip.kv_cache(kvh, d, n, 0, 2)
    write(hip, cache, 0, k, v)
    for g, w in zip(read(hip, cache, 0, n), o.stored_pair(k, v, "nvfp4")):
        np.testing.assert_array_equal(g, w.astype(np.float32))
    write(hip, cache, 3, k[:1], v[:1])   # overwritten: finite again
    for g, w in zip(read(hip, cache, 3, 1), (k, v)):
        np.testing.assert_array_equal(g, o.stored_nvfp4(w[:1]).astype(np.float32))
    cache.destroy()


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("x_dtype", [o.F32, o.BF16])
@pytest.mark.parametrize("glob", [2.0 ** -60, 0.5, 1.0])
def test_values_beyond_what_a_global_holds_saturate(hip, d, x_dtype, glob):
    """Finite values up to FP32's largest, whose quotients by the global and by a scale pass FP32, among ordinary ones:
    the largest scale and codes of 6, as the format says, and blocks beside them as ever."""
    rng = np.random.default_rng(d + x_dtype)
    n, kvh = 40, 2
    k, v = some_rows(rng, n, kvh, d) * np.float32(glob), some_rows(rng, n, kvh, d) * np.float32(glob)
    for x in (k, v):
        big = np.float32(10.0 ** rng.uniform(20, 38.5, x.shape)) * np.where(rng.random(x.shape) < 0.5, -1, 1)
        x[...] = np.where(rng.random(x.shape) < 0.1, big, x)
        x[5, 0, :16], x[37, 1, -1] = np.float32(3.38e38), np.float32(-3.38e38)
        x[7] = big[7]
    cache = hip.kv_cache(kvh, d, n, 0, 2)
    cache.globals(glob, glob)
    write(hip, cache, 0, k, v, x_dtype)
    for g, x in zip(read(hip, cache, 0, n), (k, v)):
        np.testing.assert_array_equal(g, o.stored_nvfp4(o.rows(x, x_dtype)[1], glob).astype(np.float32))
    cache.destroy()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_other_caches_write_bf16_rows_and_read_back(hip, dtype, d):
    rng = np.random.default_rng(d + 1)
    n, kvh, ring, pos = 90, 3, 70, 55
    k, v = (rng.standard_normal((n, kvh, d)).astype(np.float32) for _ in "kv")
    for x_dtype in (o.BF16, o.F32):
        cache = hip.kv_cache(kvh, d, 0, ring, o.KV[dtype])
        write(hip, cache, pos, k, v, x_dtype)
        want = [w.astype(np.float32) for w in o.stored_pair(*(o.rows(x, x_dtype)[1] for x in (k, v)), dtype)]
        for w in want:
            w[:n - ring] = 0.0
        for g, w in zip(read(hip, cache, pos, n), want):
            np.testing.assert_array_equal(g, w)
        for g, w in zip(read(hip, cache, pos, n, o.BF16), want):
            np.testing.assert_array_equal(g, o.bf16(w))
        for h in range(kvh):
            for g, w in zip(cache.load(h, pos + n - ring, pos + n), want):
                np.testing.assert_array_equal(g, w[n - ring:, h])
        cache.destroy()


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_fp8_rows_with_infinities_read_back_as_they_load(hip, d):
    """A row with an infinity has an infinite scale: its codes of zero are NaN, in K and V, on the device as on the host;
    a NaN is one by itself."""
    rng = np.random.default_rng(d)
    n, kvh = 40, 2
    k, v = (rng.standard_normal((n, kvh, d)).astype(np.float32) for _ in "kv")
    k[3, 0, 5], v[3, 1, 7], v[36, 0, 2], k[20, 1, 1], v[20, 1, 1] = np.inf, -np.inf, np.inf, np.nan, np.nan
    cache = hip.kv_cache(kvh, d, n + 5, 0, o.KV["fp8"])
    write(hip, cache, 0, k, v)
    got = read(hip, cache, 0, n + 5)
    for h in range(kvh):
        for g, w in zip(got, cache.load(h, 0, n)):
            np.testing.assert_array_equal(g[:n, h], w)
    assert np.isnan(got[1][3, 1]).all() and np.isnan(got[1][20, 1, 1]) and np.isfinite(got[1][20, 1, 2:]).all()
    assert not any(g[n:].any() for g in got)
    cache.destroy()


@gpu
def test_save_restore_copy_release(hip):
    rng = np.random.default_rng(2)
    kvh, d, ring, n = 2, 128, 45, 60
    k, v = some_rows(rng, n, kvh, d), some_rows(rng, n, kvh, d)
    a, b = hip.kv_cache(kvh, d, 0, ring, 2), hip.kv_cache(kvh, d, 0, ring, 2)
    write(hip, a, 0, k, v)
    want = read(hip, a, 15, ring)
    b.restore(a.save())
    c = hip.kv_cache(kvh, d, 0, ring, 2)
    a.copy_to(c)
    for x in (b, c):
        for g, w in zip(read(hip, x, 15, ring), want):
            np.testing.assert_array_equal(g, w)
    b.release()
    assert not any(x.any() for x in read(hip, b, 15, ring))
    assert a.nbytes() == 2 * kvh * 64 * (d // 2 + d // 16) + 64 * 4 + 8   # slots padded to 64, positions, globals
    for x in (a, b, c):
        x.destroy()


@gpu
def test_far_slots(hip):
    """Offsets beyond 32 bits: one head of 256 dims, 2^25 + 70 slots of 144 bytes a side."""
    slots = (1 << 25) + 70
    cache = hip.kv_cache(1, 256, slots, 0, 2)
    rng = np.random.default_rng(4)
    k, v = some_rows(rng, 65, 1, 256), some_rows(rng, 65, 1, 256)
    write(hip, cache, slots - 65, k, v)
    write(hip, cache, 0, k[:1], v[:1])
    for g, x in zip(read(hip, cache, slots - 65, 65), (k, v)):
        np.testing.assert_array_equal(g, o.stored_nvfp4(x).astype(np.float32))
    for g, x in zip(read(hip, cache, 0, 2), (k, v)):
        np.testing.assert_array_equal(g[0], o.stored_nvfp4(x)[0].astype(np.float32))
        assert not g[1].any()
    cache.destroy()


@gpu
def test_refusals(hip, pkg):
    cache = hip.kv_cache(2, 64, 40, 0, 2)
    a = hip.array(shape=(8, 2, 64))
    for call, what in [(lambda: cache.write(39, 2, a, a), "KV cache full"), (lambda: cache.read(39, 2, a, a), "KV cache full"),
                       (lambda: cache.write(-1, 2, a, a), "rows at"), (lambda: cache.write(0, -2, a, a), "rows at"),
                       (lambda: cache.write(0, 2, a, a, 2), "row type"), (lambda: cache.read(0, 2, a, a, 7), "row type"),
                       (lambda: cache.write(0, 2, None, a), "NULL"), (lambda: cache.read(0, 2, a, None), "NULL"),
                       (lambda: cache.write(0, 2, a.ptr + 4, a), "aligned"), (lambda: cache.read(0, 2, a, a.ptr + 8), "aligned"),
                       (lambda: cache.globals(3.0, 1.0), "power of two"), (lambda: cache.globals(1.0, 0.0), "power of two"),
                       (lambda: cache.globals(1.0, -2.0), "power of two"), (lambda: cache.globals(2.0 ** 61, 1.0), "power of two"),
                       (lambda: cache.globals(float("nan"), 1.0), "power of two"),
                       (lambda: hip.kv_cache(2, 64, 40, 0, 3), "unknown KV dtype"),
                       (lambda: hip.kv_cache(2, 64, 40, 0, 0).globals(1.0, 1.0), "not an NVFP4"),
                       (lambda: hip.attention(cache, a, a, a, a, 1, 0, 2), "NVFP4"),
                       (lambda: hip.attention_noalloc(cache, a, a, a, a, 1, 0, 2), "NVFP4")]:
        with pytest.raises(pkg.XtgError, match=what):
            call()
    cache.write(0, 0, None, None)   # no rows: nothing to do
    cache.read(0, 0, None, None)
    assert not read(hip, cache, 0, 40)[0].any()
    a.free()
    cache.destroy()


@gpu
@pytest.mark.parametrize("pos", [2 ** 31 - 1, 2 ** 40, 2 ** 63 - 2, 2 ** 63 - 1])
def test_positions_whose_end_passes_64_bits_are_refused(hip, pkg, wl, pos):
    """The end of the rows, pos + n, is never formed: it would be negative, and below every limit."""
    a = hip.array(shape=(8, 8, 64))
    caches = [hip.kv_cache(2, 64, 40, ring, dtype) for ring in (0, 40) for dtype in (0, 1, 2)]
    for c in caches:
        calls = [lambda: c.store(pos, 2, a, a), lambda: c.write(pos, 2, a, a), lambda: c.read(pos, 2, a, a),
                 lambda: hip.attention_ext(c, a, a, a, a, 2, pos, 4, 2, 64), lambda: hip.attention(c, a, a, a, a, 2, pos, 4),
                 lambda: hip.attention_noalloc(c, a, a, a, a, 2, pos, 4)]
        for call in calls:
            with pytest.raises(pkg.XtgError, match="full|positions|rows at|NVFP4"):
                call()
        assert not read(hip, c, 0, 40)[0].any()
    w = wl.DoryWeights(wl.DORY_TINY, seed=3, context=256)
    d = hip.dory(w)
    x, y = hip.array(shape=(2, w.cfg["hidden"])), hip.array(shape=(2, w.cfg["vocab"]))
    for call in (lambda: d.forward(x, 2, pos, y), lambda: d.prefill(x, 2, pos, pkg.LOGITS_NONE)):
        with pytest.raises(pkg.XtgError, match="context full"):
            call()
    d.destroy()
    for c in caches:
        c.destroy()
    for b in (a, x, y):
        b.free()


class Rows:
    """What the bindings ask of a torch tensor."""

    def __init__(self, dtype="torch.float32", device=0, n=512, whole=True, at=4096):
        self.dtype, self.a = dtype, (device, n, whole, at)

    def get_device(self):
        return self.a[0]

    def numel(self):
        return self.a[1]

    def is_contiguous(self):
        return self.a[2]

    def data_ptr(self):
        return self.a[3]


def test_arrays_that_are_not_the_rows_of_the_call(pkg):
    """Without a GPU: an array of another dtype than the row type (BF16 rows at the default, FP32), in host memory or on
    another device, strided, too short or freed is refused before its address goes anywhere."""
    class Backend:
        device = 0

    freed = pkg.DeviceArray.__new__(pkg.DeviceArray)
    freed.b, freed.ptr, freed.nbytes, freed.dtype = Backend, None, 2048, np.dtype(np.float32)
    for a, kind, what in [(Rows("torch.bfloat16"), pkg.X_F32, "row type FP32"), (Rows(), pkg.X_BF16, "row type BF16"),
                          (Rows("torch.float16"), pkg.X_BF16, "row type BF16"), (Rows("torch.int64"), pkg._I32, "int32"),
                          (Rows(), 7, "row type"), (Rows(device=-1), pkg.X_F32, "memory"), (Rows(device=1), pkg.X_F32, "memory"),
                          (Rows(whole=False), pkg.X_F32, "contiguous"), (Rows(n=511), pkg.X_F32, "511 elements"),
                          (np.zeros(512, np.float32), pkg.X_F32, "device memory"), (freed, pkg.X_F32, "freed")]:
        with pytest.raises(pkg.XtgError, match=what):
            pkg._device_ptr(Backend, "q", a, 512, kind)
    for a, kind in [(Rows(), pkg.X_F32), (Rows("torch.bfloat16"), pkg.X_BF16), (Rows("uint16"), pkg.X_BF16), (4096, 7)]:
        assert pkg._device_ptr(Backend, "q", a, 512, kind) == 4096
    assert pkg._device_ptr(Backend, "q", None, 512, 0) is None and pkg._device_ptr(Backend, "q", Rows(n=0, at=0), 0, 0) == 0


@gpu
def test_arrays_of_another_type_are_refused(hip, pkg):
    """The default row type is FP32: BF16 arrays without x_dtype would be read and written at twice their size."""
    cache = hip.kv_cache(2, 64, 40, 0, 2)
    f, b, out = (hip.array(shape=(4, 4, 64), dtype=t) for t in (np.float32, np.uint16, np.float32))
    i, j, short, host = hip.array(shape=(4,), dtype=np.int64), hip.array(shape=(3,), dtype=np.int32), hip.array(shape=(511,)), np.zeros((4, 4, 64))
    good = dict(cache=cache, q=f, k=f, v=f, out=out, n_q=4, pos0=3, heads=4, kv_heads=2, head_dim=64)
    hip.attention_ext(**good)
    hip.attention_ext(**dict(good, q=f.ptr, k=f.ptr, out=out.ptr))   # addresses are the caller's
    for change in [dict(q=b), dict(k=b), dict(out=b), dict(q=host), dict(first=i), dict(end=j), dict(slopes=i), dict(v=short),
                   dict(out=short), dict(x_dtype=pkg.X_BF16)]:
        with pytest.raises(pkg.XtgError):
            hip.attention_ext(**dict(good, **change))
    for call in (cache.write, cache.read):
        for k, v, x in [(b, b, pkg.X_F32), (f, b, pkg.X_F32), (f, f, pkg.X_BF16), (host, f, pkg.X_F32), (f, short, pkg.X_F32)]:
            with pytest.raises(pkg.XtgError):
                call(0, 4, k, v, x)
    hip.finish()
    for a in (f, b, out, i, j, short):
        a.free()
    cache.destroy()


def test_null_arguments_are_refused(pkg):
    """Without a GPU: a NULL handle or cache is an error, not a fault."""
    lib, err = pkg.lib(), ctypes.create_string_buffer(200)
    assert lib.xtg_hip_kv_globals(None, None, 1.0, 1.0, err, 200) == -1 and b"NULL" in err.value
    assert lib.xtg_hip_kv_write(None, None, 0, 1, None, None, 0, err, 200) == -1 and b"NULL" in err.value
    assert lib.xtg_hip_kv_read(None, None, 0, 1, None, None, 0, err, 200) == -1 and b"NULL" in err.value
    assert lib.xtg_hip_attention_ext(None, None, err, 200) == -1 and b"NULL" in err.value
    e = pkg.AttnExt   # as the C compiler lays xtg_attn_ext out
    assert [getattr(e, n).offset for n in ("pos0", "heads", "scale", "q", "cache", "out", "x_dtype", "slopes", "end")] == \
        [8, 16, 32, 40, 64, 72, 80, 88, 104]
    assert ctypes.sizeof(e) == 112


def test_format_in_64_bits():
    """The oracle's own format against the definition spelt out value by value."""
    rng = np.random.default_rng(0)
    grid = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
    c = np.arange(127)
    scales = np.where(c >> 3 > 0, (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7.0), (c & 7) * 2.0 ** -9)
    for _ in range(300):
        x = (rng.standard_normal(16) * 2.0 ** rng.uniform(-12, 12)).astype(np.float32)
        amax = np.abs(x.astype(np.float64)).max()
        s = scales[1:][np.abs(scales[1:] - amax / 6).argmin()]
        want = grid[np.abs(np.abs(x.astype(np.float64))[:, None] / s - grid).argmin(1)] * s * np.sign(x)
        np.testing.assert_array_equal(o.stored_nvfp4(x), want)
