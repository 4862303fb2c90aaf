"""GPU: the 8-bit K/V cache. The i8 values are exact (ties away from zero), so
they are compared for equality; a scale is one f32 division (2^-24 relative,
twice for the oracle's own rounding), a value read back one f32 product more."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from prana_amd import _lib
from tests import serving_oracle as SO

pytestmark = pytest.mark.gpu


def rows_of(r, n, width, kind):
    if kind == "normal":
        return (r.standard_normal((n, width)) * np.exp(r.normal(0, 2, (n, 1)))).astype(np.float32)
    if kind == "ties":  # integers over a maximum of 254: many quotients are halves exactly
        x = r.integers(-254, 255, (n, width)).astype(np.float32)
        x[:, ::8] = 254
        return x
    if kind == "tiny":  # subnormal values among others
        return (r.standard_normal((n, width)) * 2.0 ** -140).astype(np.float32)
    x = (r.standard_normal((n, width)) * 1e37).astype(np.float32)  # near the largest
    return np.clip(x, -3.4e38, 3.4e38).astype(np.float32)


@pytest.mark.parametrize("kind", ["normal", "ties", "tiny", "large"])
@pytest.mark.parametrize("heads,w", [(8, 128), (2, 64), (6, 48), (1, 256), (3, 8), (5, 24), (2, 200)])
def test_write_and_read(heads, w, kind):
    r = np.random.default_rng(heads * w + len(kind))
    counts, first, caps = [5, 0, 1, 70, 33], [2, 0, 7, 0, 1], [9, 1, 8, 70, 40]
    caches = [P.KvQ8(n, heads, w) for n in caps]
    k, v = rows_of(r, sum(counts), heads * w, kind), rows_of(r, sum(counts), heads * w, kind)
    k[3, :w] = 0  # a head of zeros
    P.kv_write_q8(caches, k, v, first, counts)
    at = 0
    for c, f, n in zip(caches, first, counts):
        for x, dq, ds in ((k, c.k, c.k_scales), (v, c.v, c.v_scales)):
            q, s = dq.to_host(), ds.to_host()
            want_q, want_s = SO.quantize(x[at:at + n], heads, w)
            assert np.array_equal(q[f:f + n], want_q)
            got_s = s[f:f + n].astype(np.float64)
            assert np.all(np.abs(got_s - want_s) <= 2 ** -23 * want_s + 2.0 ** -149)
            # rows around the written ones keep what they held
            assert not q[:f].any() and not q[f + n:].any() and np.all(s[:f] == 1) and np.all(s[f + n:] == 1)
        at += n
    gk, gv = P.kv_read_q8(caches, first, counts)
    hk, hv = P.kv_read_q8(caches, first, counts, half=True)
    at = 0
    for c, f, n in zip(caches, first, counts):
        for g, h, dq, ds in ((gk, hk, c.k, c.k_scales), (gv, hv, c.v, c.v_scales)):
            q, s = dq.to_host()[f:f + n].reshape(n, heads, w), ds.to_host()[f:f + n]
            want = (q.astype(np.float32) * s[..., None]).reshape(n, heads * w)  # one f32 product: the same bits
            assert np.array_equal(g[at:at + n], want)
            # the product (31 bits, exact in f64) rounded to a half at once, or
            # to f32 first, which can move a value onto a half's tie
            exact = (q.astype(np.float64) * s[..., None]).reshape(n, heads * w)
            with np.errstate(over="ignore"):
                once, twice = exact.astype(np.float16), want.astype(np.float16)
            assert np.all((h[at:at + n] == once) | (h[at:at + n] == twice))
        at += n


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_head_with_a_value_that_is_not_finite_reads_back_as_nan(bad):
    r = np.random.default_rng(3)
    k, v = (r.standard_normal((4, 3 * 16)).astype(np.float32) for _ in "kv")
    k[1, 17] = bad
    v[2, 47] = bad
    c = P.KvQ8(4, 3, 16)
    P.kv_write_q8([c], k, v, [0], [4])
    gk, gv = P.kv_read_q8([c], [0], [4])
    for x, g, row, head in ((k, gk, 1, 1), (v, gv, 2, 2)):
        nan = np.zeros((4, 3), bool)
        nan[row, head] = True
        assert np.array_equal(np.isnan(g).reshape(4, 3, 16).all(-1), nan)
        assert np.array_equal(np.isnan(g).reshape(4, 3, 16).any(-1), nan)
        want, s = SO.quantize(np.where(np.isfinite(x), x, 0), 3, 16)
        fine = ~nan
        assert np.allclose(g.reshape(4, 3, 16)[fine], (want.reshape(4, 3, 16) * s[..., None])[fine], rtol=2 ** -22,
                           atol=0)


def test_strided_rows_many_sequences_and_nothing_outside():
    # k and v side by side in wider rows; more sequences than one launch takes
    r = np.random.default_rng(9)
    heads, w, n = 2, 40, 150
    counts = [int(x) for x in r.integers(0, 4, n)]
    total, ld = sum(counts), 2 * heads * w + 8
    src = r.standard_normal((total, ld)).astype(np.float32)
    caches = [P.KvQ8(6, heads, w) for _ in range(n)]
    first = [int(x) for x in r.integers(0, 3, n)]
    d = P.DeviceArray.from_host(src)
    lib = _lib.load()
    f, c = (C.c_size_t * n)(*first), (C.c_size_t * n)(*counts)
    kv = (P.PranaKv * n)(*[x.struct() for x in caches])
    P.check(lib.prana_kv_write_q8(d.ptr, C.c_void_p(d.ptr.value + 4 * heads * w), ld, kv, f, c, n, heads, w, None))
    out = P.DeviceArray.from_host(np.full((total + 1, ld), 7, np.float32))
    P.check(lib.prana_kv_read_q8(kv, f, c, n, heads, w, P.F32, out.ptr, C.c_void_p(out.ptr.value + 4 * heads * w), ld,
                                 None))
    got = out.to_host()
    for x, a in ((src[:, :heads * w], 0), (src[:, heads * w:2 * heads * w], heads * w)):
        q, s = SO.quantize(x, heads, w)
        want = (q.reshape(-1, heads, w) * s[..., None]).reshape(total, -1)
        assert np.allclose(got[:total, a:a + heads * w], want, rtol=2 ** -22, atol=0)
    assert np.all(got[:total, 2 * heads * w:] == 7) and np.all(got[total] == 7)


def test_offsets_past_32_bits():
    # rows that lie 4 GiB behind the cache's first
    heads, w, rows = 8, 256, (1 << 21) + 40
    c = P.KvQ8.__new__(P.KvQ8)
    c.rows, c.n_kv_heads, c.head_dim, c.width = rows, heads, w, heads * w
    c.k, c.v = (P.DeviceArray((rows, heads * w), np.int8) for _ in "kv")
    c.k_scales, c.v_scales = (P.DeviceArray((rows, heads), np.float32) for _ in "kv")
    r = np.random.default_rng(0)
    k, v = (r.standard_normal((50, heads * w)).astype(np.float32) for _ in "kv")
    P.kv_write_q8([c, c], k, v, [rows - 40, 3], [40, 10])
    for got, x in zip(P.kv_read_q8([c, c], [rows - 40, 3], [40, 10]), (k, v)):
        q, s = SO.quantize(x, heads, w)
        want = (q.reshape(50, heads, w) * s[..., None]).reshape(50, heads * w)
        assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -22).all()


def test_empty_calls():
    lib = _lib.load()
    P.init()
    assert lib.prana_kv_write_q8(None, None, 0, None, None, None, 0, 2, 64, None) == 0
    z = (C.c_size_t * 2)(0, 0)
    kv = (P.PranaKv * 2)()
    assert lib.prana_kv_read_q8(kv, z, z, 2, 2, 64, P.F32, None, None, 0, None) == 0
