"""GPU: attention of drafted tokens over f16 and 8-bit caches against the
64-bit form, within the bounds that serving_oracle.py derives."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from prana_amd import _lib
from tests import serving_oracle as SO

pytestmark = pytest.mark.gpu

KINDS = ["f16", "q8"]


def make(seed, kind, past, tokens, heads, kv_heads, w, spare=3, sigma=1.5):
    """(q, caches, the caches' values per sequence)."""
    r = np.random.default_rng(seed)
    q = (r.standard_normal((sum(tokens), heads * w)) * sigma).astype(np.float32)
    caches, ks, vs = [], [], []
    for n, m in zip(past, tokens):
        k, v = (r.standard_normal((n + m + spare, kv_heads * w)) for _ in "kv")
        if kind == "f16":
            k, v = k.astype(np.float16), v.astype(np.float16)
            caches.append(P.KvF16(k, v))
        else:
            c = P.KvQ8(len(k), kv_heads, w)
            scale = lambda: np.exp(r.normal(-4, 1, (len(k), kv_heads))).astype(np.float32)  # noqa: E731
            vals = []
            for a, b in ((c.k, c.k_scales), (c.v, c.v_scales)):
                i8, s = r.integers(-127, 128, a.shape).astype(np.int8), scale()
                lib = _lib.load()
                P.check(lib.prana_memcpy_h2d(a.ptr, C.c_void_p(i8.ctypes.data), i8.nbytes))
                P.check(lib.prana_memcpy_h2d(b.ptr, C.c_void_p(s.ctypes.data), s.nbytes))
                vals.append((i8.astype(np.float64).reshape(len(k), kv_heads, w) * s[..., None]).reshape(len(k), -1))
            k, v = vals
            caches.append(c)
        ks.append(np.asarray(k, np.float64))
        vs.append(np.asarray(v, np.float64))
    return q, caches, ks, vs


def trees(seed, tokens):
    r = np.random.default_rng(seed)
    return np.concatenate([P.tree_mask([int(r.integers(-1, i)) if i else -1 for i in range(m)]) for m in tokens]
                          + [np.zeros(0, np.uint64)])


def check(kind, past, tokens, heads, kv_heads, w, mask="tree", seed=0, **more):
    q, caches, ks, vs = make(seed + sum(past) + w, kind, past, tokens, heads, kv_heads, w, **more)
    m = trees(seed, tokens) if isinstance(mask, str) else mask
    got = P.attention_tree(q, caches, past, tokens, heads, kv_heads, w, m)
    want, bound = SO.tree(q, ks, vs, past, tokens, m, heads, kv_heads, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,tokens", [([0], [1]), ([1], [1]), ([511], [1]), ([3, 0, 40, 31, 32, 33],
                                                                              [5, 64, 1, 0, 17, 16]),
                                         ([700, 127], [13, 40])])
@pytest.mark.parametrize("heads,kv_heads,w", [(6, 6, 48), (14, 2, 64), (8, 2, 128), (4, 1, 256), (3, 3, 80),
                                              (6, 2, 96), (2, 1, 8), (5, 1, 40), (2, 2, 160), (3, 1, 200)])
def test_shapes(kind, past, tokens, heads, kv_heads, w):
    check(kind, past, tokens, heads, kv_heads, w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,tokens,heads,kv_heads,w", [
    ([9000], [1], 4, 1, 128), ([5000, 3, 2500], [7, 2, 30], 4, 2, 64), ([20000], [2], 2, 1, 48),
    ([3000, 3001], [64, 64], 8, 2, 128), ([2000], [33], 32, 1, 32)])
def test_long_caches(kind, past, tokens, heads, kv_heads, w):
    check(kind, past, tokens, heads, kv_heads, w)


@pytest.mark.parametrize("kind", KINDS)
def test_many_sequences(kind):
    # more sequences than one launch takes
    r = np.random.default_rng(1)
    past, tokens = [int(x) for x in r.integers(0, 200, 150)], [int(x) for x in r.integers(0, 4, 150)]
    check(kind, past, tokens, 4, 2, 64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 8, 64])
def test_a_chain_without_a_mask(kind, tokens):
    check(kind, [77], [tokens], 8, 2, 64, mask=None)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing_get_zeros_and_bits_past_the_tree_count_for_nothing(kind):
    heads, kv_heads, w, past, tokens = 4, 2, 64, [0, 0], [5, 3]
    q, caches, ks, vs = make(5, kind, past, tokens, heads, kv_heads, w, spare=70)
    mask = np.array([0, 0b00010, 0, 0b11111, (1 << 64) - (1 << 5), (1 << 64) - 1, 0, 1 << 63], np.uint64)
    got = P.attention_tree(q, caches, past, tokens, heads, kv_heads, w, mask)
    own = mask.copy()
    own[:5] &= np.uint64(0b11111)
    own[5:] &= np.uint64(0b111)
    want, bound = SO.tree(q, ks, vs, past, tokens, own, heads, kv_heads, w)
    assert SO.within(got, want, bound)[0]
    for i in (0, 2, 4, 6, 7):
        assert not got[i].any()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("past", [37, 3000])
def test_f16_values_that_are_not_finite_stay_where_they_are_seen(bad, past):
    # drafted token 2 is seen by tokens 2 and 3 only; rows past the tree by none
    heads, kv_heads, w, tokens = 4, 2, 64, [5]
    mask = P.tree_mask([-1, 0, 0, 2, 1])
    q, caches, ks, vs = make(8, "f16", [past], tokens, heads, kv_heads, w)
    clean = P.attention_tree(q, caches, [past], tokens, heads, kv_heads, w, mask)
    k, v = (c.to_host().view(np.float16) for c in (caches[0].k, caches[0].v))
    k[past + 5:], v[past + 5:] = bad, bad
    v[past + 2, 64 + 3] = bad  # in KV head 1: query heads 2 and 3
    got = P.attention_tree(q, [P.KvF16(k, v)], [past], tokens, heads, kv_heads, w, mask)
    hit = np.zeros(got.shape, bool)
    hit[2:4, 2 * 64 + 3::64] = True
    assert np.array_equal(got[~hit], clean[~hit])
    assert np.isnan(got[hit]).all() if np.isnan(bad) else (got[hit] == bad).all()
    k[past + 2, 70] = np.nan
    got = P.attention_tree(q, [P.KvF16(k, v)], [past], tokens, heads, kv_heads, w, mask)
    hit[2:4, 128:] = True
    assert np.isnan(got[2:4, 128:]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("past", [37, 3000])
def test_q8_scales_that_are_nan_stay_where_they_are_seen(past):
    heads, kv_heads, w, tokens = 4, 2, 64, [5]
    mask = P.tree_mask([-1, 0, 0, 2, 1])
    r = np.random.default_rng(6)
    q = r.standard_normal((5, heads * w)).astype(np.float32)
    k, v = (r.standard_normal((past + 8, kv_heads * w)).astype(np.float32) for _ in "kv")

    def run(k, v):
        c = P.KvQ8(past + 8, kv_heads, w)
        P.kv_write_q8([c], k, v, [0], [past + 8])
        return P.attention_tree(q, [c], [past], tokens, heads, kv_heads, w, mask)

    clean = run(k, v)
    for which in "kv":
        k2, v2 = k.copy(), v.copy()
        k2[past + 5:], v2[past + 5:] = np.nan, np.inf
        (k2 if which == "k" else v2)[past + 2, 64 + 3] = np.inf
        got = run(k2, v2)
        hit = np.zeros(got.shape, bool)
        hit[2:4, 128:] = True  # the whole head is NaN
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("spread", [1e-6, 1e6])
def test_q8_value_scales_far_apart(spread):
    # V rows whose scales differ by six orders of magnitude: the bound is
    # relative to the weighted sum, which the large rows make
    heads, kv_heads, w, past = 2, 1, 64, 600
    q, caches, ks, vs = make(31, "q8", [past], [3], heads, kv_heads, w)
    s = caches[0].v_scales.to_host()
    f = np.where(np.arange(len(s)) % 7 == 0, np.float32(spread), np.float32(1))[:, None]
    s2 = (s * f).astype(np.float32)
    P.check(_lib.load().prana_memcpy_h2d(caches[0].v_scales.ptr, C.c_void_p(s2.ctypes.data), s2.nbytes))
    vs[0] = vs[0] / s.astype(np.float64) * s2
    got = P.attention_tree(q, caches, [past], [3], heads, kv_heads, w)
    want, bound = SO.tree(q, ks, vs, [past], [3], None, heads, kv_heads, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sigma", [0.0, 30.0])
def test_flat_and_sharp_scores(kind, sigma):
    check(kind, [900], [6], 4, 2, 64, sigma=sigma)


@pytest.mark.parametrize("kind", KINDS)
def test_matches_split_decode_and_the_same_call_twice(kind):
    # one token per sequence is the split-K decode; a call repeats bit for bit
    past = [1500, 40]
    q, caches, ks, vs = make(2, kind, past, [1, 1], 8, 2, 128)
    a = P.attention_tree(q, caches, past, [1, 1], 8, 2, 128)
    b = P.attention_tree(q, caches, past, [1, 1], 8, 2, 128)
    assert np.array_equal(a, b)
    if kind == "f16":
        s = P.attention_decode_splitk(q, [c.k for c in caches], [c.v for c in caches], past, 8, 2, 128)
        want, bound = SO.tree(q, ks, vs, past, [1, 1], None, 8, 2, 128)
        assert np.all(np.abs(s - a) <= bound + 1e-4 * np.abs(want) + 2e-6)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,tokens,group", [(37, 5, 2), (6000, 5, 2), (6000, 12, 2), (6000, 40, 4)])
def test_a_query_that_is_not_a_number_spoils_its_row_alone(kind, past, tokens, group):
    # (the longer caches in parts, each without a maximum for that row)
    w = 64
    q, caches, _, _ = make(3, kind, [past], [tokens], 2 * group, 2, w)
    clean = P.attention_tree(q, caches, [past], [tokens], 2 * group, 2, w)
    q[3, w + 5] = np.nan
    got = P.attention_tree(q, caches, [past], [tokens], 2 * group, 2, w)
    assert np.isnan(got[3, w:2 * w]).all()
    got[3, w:2 * w] = clean[3, w:2 * w]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("past,tokens", [(600, 3), (3000, 40)])
def test_q8_value_scales_beyond_a_floats_square(past, tokens):
    # V scales from 2^-66 to 2^80, the small ones first: what is summed before
    # the large ones come stays in the sum that divides
    w = 64
    q, caches, ks, vs = make(32, "q8", [past], [tokens], 4, 1, w)
    s = caches[0].v_scales.to_host()
    f = np.where(np.arange(len(s)) < past // 2, np.float32(2.0 ** -62), np.float32(2.0 ** 84))[:, None]
    s2 = (s * f).astype(np.float32)
    P.check(_lib.load().prana_memcpy_h2d(caches[0].v_scales.ptr, C.c_void_p(s2.ctypes.data), s2.nbytes))
    vs[0] = vs[0] * f.astype(np.float64)  # (a power of two: exact)
    got = P.attention_tree(q, caches, [past], [tokens], 4, 1, w)
    want, bound = SO.tree(q, ks, vs, [past], [tokens], None, 4, 1, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


def test_one_call_of_all_widths():
    # single tokens, small trees and large ones over short and long caches in one call
    check("f16", [5000, 0, 77, 4000, 300, 2], [1, 64, 9, 30, 3, 1], 8, 2, 128)
    check("q8", [5000, 0, 77, 4000, 300, 2], [1, 64, 9, 30, 3, 1], 8, 2, 128)


def test_offsets_past_32_bits():
    # a cache whose last rows lie 4 GiB behind its first; K and V share it
    kv_heads, w, rows, past = 8, 256, (1 << 20) + 300, (1 << 20) + 290
    q = np.zeros((2, kv_heads * w), np.float32)
    c = P.DeviceArray.from_host(np.zeros((rows, kv_heads * w), np.uint16))
    lib = _lib.load()
    r = np.random.default_rng(0)
    some = {t: r.standard_normal(kv_heads * w).astype(np.float16) for t in (5, past - 3, past + 1)}
    for t, x in some.items():
        P.check(lib.prana_memcpy_h2d(C.c_void_p(c.ptr.value + t * kv_heads * w * 2), C.c_void_p(x.ctypes.data), x.nbytes))
    # scores of 20 there and 0 elsewhere
    for i, t in ((0, past - 3), (1, past + 1)):
        for h in range(kv_heads):
            x = some[t][h * w:(h + 1) * w].astype(np.float64)
            q[i, h * w:(h + 1) * w] = 20 * np.sqrt(w) * x / (x @ x)
    got = P.attention_tree(q, [P.KvF16(c, c)], [past], [2], kv_heads, kv_heads, w)
    for i in range(2):
        for h in range(kv_heads):
            a = slice(h * w, (h + 1) * w)
            t = [t for t in some if t <= past + i]
            k = np.stack([some[x][a].astype(np.float64) for x in t])
            s = k @ q[i, a].astype(np.float64) / np.sqrt(w)
            p = np.exp(s)
            den = p.sum() + (past + 1 + i - len(t))  # the rows of zeros
            want = p @ k / den
            # as derived in serving_oracle.py, with n rows of which only these have values
            ds = ((w + 8) * SO.U * (np.abs(k) @ np.abs(q[i, a].astype(np.float64))) / np.sqrt(w) + 4 * SO.U * np.abs(s)).max()
            bound = (p @ np.abs(k) / den) * (2 * ds + 8 * SO.U + 2 * past * SO.U) + 2.0 ** -31 * len(t) * np.abs(k).max()
            assert (np.abs(got[i, a] - want) <= bound).all()


def test_empty_calls():
    lib = _lib.load()
    P.init()
    z = (C.c_size_t * 2)(0, 0)
    kv = (P.PranaKv * 2)()
    assert lib.prana_attention_tree(None, P.KV_F16, kv, z, z, 2, None, 8, 2, 64, None, None, 0, None) == 0
    assert lib.prana_attention_tree(None, P.KV_Q8, None, None, None, 0, None, 8, 2, 64, None, None, 0, None) == 0
