"""GPU: V scales of 8-bit caches in tree attention. A row's result is made of
the scales that it sees and of how much weight they have there, whatever the
other rows of the cache hold."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from prana_amd import _lib
from tests import serving_bounds as SB
from tests import serving_oracle as SO

pytestmark = pytest.mark.gpu


class Caches:
    """Random 8-bit caches, one per sequence, and what they hold in f64."""

    def __init__(self, seed, rows, kv_heads, w):
        r = np.random.default_rng(seed)
        self.kv_heads, self.w = kv_heads, w
        self.caches, self.k, self.vi, self.vs = [], [], [], []
        for n in rows:
            c = P.KvQ8(n, kv_heads, w)
            ki, vi = (r.integers(-127, 128, (n, kv_heads, w)).astype(np.int8) for _ in "kv")
            ks, vs = (np.exp(r.normal(-4, 0.5, (n, kv_heads))).astype(np.float32) for _ in "kv")
            for a, x in ((c.k, ki), (c.v, vi), (c.k_scales, ks), (c.v_scales, vs)):
                put(a, x)
            self.caches.append(c)
            self.k.append((ki * ks[..., None].astype(np.float64)).reshape(n, -1))
            self.vi.append(vi)
            self.vs.append(vs)

    def scale(self, s, f):
        """V scales of sequence s times f [rows, kv_heads] (powers of two: exact)."""
        self.vs[s] = (self.vs[s] * f).astype(np.float32)
        put(self.caches[s].v_scales, self.vs[s])

    def values(self):
        return [(i * s[..., None].astype(np.float64)).reshape(len(i), -1) for i, s in zip(self.vi, self.vs)]

    def tops(self):
        return [127 * np.abs(s.astype(np.float64)) for s in self.vs]


def put(d, a):
    a = np.ascontiguousarray(a)
    P.check(_lib.load().prana_memcpy_h2d(d.ptr, C.c_void_p(a.ctypes.data), a.nbytes))


def check(c, q, past, tokens, mask, heads, got=None):
    if got is None:
        got = P.attention_tree(q, c.caches, past, tokens, heads, c.kv_heads, c.w, mask)
    want, bound = SB.tree(q, c.k, c.values(), past, tokens, mask, heads, c.kv_heads, c.w, c.tops())
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


# One block of narrow rows, two of them, and the wide kernel, at its tile sizes.
SHAPES = [(5, 4, 2, 64), (1, 6, 2, 128), (5, 2, 2, 200), (12, 4, 2, 96), (40, 8, 2, 64), (40, 4, 1, 128),
          (20, 3, 1, 256)]


@pytest.mark.parametrize("power", [10, 30, 57])
@pytest.mark.parametrize("past", [0, 20, 3000])
@pytest.mark.parametrize("tokens,heads,kv_heads,w", [s for s in SHAPES if s[0] > 1])
def test_scales_of_rows_that_a_row_does_not_see(tokens, heads, kv_heads, w, past, power):
    # drafted token 2 is seen by itself and token 3, rows past the tree by none
    parents = [-1, 0, 0, 2] + [1] * (tokens - 4)
    mask = P.tree_mask(parents)
    q = (np.random.default_rng(1).standard_normal((tokens, heads * w)) * 1.5).astype(np.float32)
    c = Caches(2, [past + tokens + 5], kv_heads, w)
    clean = P.attention_tree(q, c.caches, [past], [tokens], heads, kv_heads, w, mask)
    f = np.ones((past + tokens + 5, kv_heads))
    f[past + 2] = f[past + tokens:] = 2.0 ** power
    c.scale(0, f)
    got = P.attention_tree(q, c.caches, [past], [tokens], heads, kv_heads, w, mask)
    others = [i for i in range(tokens) if i not in (2, 3)]
    assert np.array_equal(got[others], clean[others])
    check(c, q, [past], [tokens], mask, heads, got)


@pytest.mark.parametrize("power", [8, 16, 40])
@pytest.mark.parametrize("tokens,heads,kv_heads,w", SHAPES)
def test_a_large_scale_of_little_weight(tokens, heads, kv_heads, w, power):
    # a past row whose score is far below the others' in every head and token:
    # what it adds is small beside the rest, which keeps its bits
    past = 300
    r = np.random.default_rng(3)
    base = np.abs(r.standard_normal(w)) + 0.5
    q = (np.tile(base, (tokens, heads)) + 0.1 * r.standard_normal((tokens, heads * w))).astype(np.float32)
    c = Caches(4, [past + tokens], kv_heads, w)
    row = np.zeros((past + tokens, kv_heads, w), np.int8)
    row[:] = (c.k[0].reshape(row.shape) > 0) * 2 - 1
    row[37] = -127  # against every q
    put(c.caches[0].k, row.reshape(len(row), -1))
    # scores of -40 (in powers of e) there, and within +-1 elsewhere
    ks = np.full((past + tokens, kv_heads), 40 / (127 * base.sum() / np.sqrt(w)), np.float32)
    put(c.caches[0].k_scales, ks)
    c.k[0] = (row * ks[..., None].astype(np.float64)).reshape(len(row), -1)
    f = np.ones((past + tokens, kv_heads))
    f[37] = 2.0 ** power
    c.scale(0, f)
    check(c, q, [past], [tokens], None, heads)


@pytest.mark.parametrize("past", [40, 3000])
@pytest.mark.parametrize("tokens,heads,kv_heads,w", SHAPES)
def test_scales_that_rise_and_fall_along_the_cache(tokens, heads, kv_heads, w, past):
    r = np.random.default_rng(5)
    q = (r.standard_normal((tokens, heads * w)) * 1.5).astype(np.float32)
    c = Caches(6, [past + tokens], kv_heads, w)
    at = np.arange(past + tokens)[:, None] + 17 * np.arange(kv_heads)[None, :]
    c.scale(0, 2.0 ** np.round(20 * np.sin(at / 23.0)))
    check(c, q, [past], [tokens], None, heads)


@pytest.mark.parametrize("size", [1e7, 1e9, 1e30])
@pytest.mark.parametrize("tokens,heads,kv_heads,w", SHAPES)
def test_scores_too_large_to_add_a_scales_exponent_to(tokens, heads, kv_heads, w, size):
    # scores whose neighbours lie further apart than the scales' exponents: 64 bits
    # would pick other keys, but a result is a mean of values all the same
    past = 500
    r = np.random.default_rng(7)
    q = (r.standard_normal((tokens, heads * w)) * size).astype(np.float32)
    c = Caches(8, [past + tokens], kv_heads, w)
    row = np.repeat(r.integers(-127, 128, (9, kv_heads, w)), 100, 0)[:past + tokens].astype(np.int8)  # (equal scores)
    put(c.caches[0].k, row.reshape(len(row), -1))
    put(c.caches[0].k_scales, np.full((past + tokens, kv_heads), 0.01, np.float32))
    c.scale(0, 2.0 ** r.integers(-60, 30, (past + tokens, kv_heads)))
    got = P.attention_tree(q, c.caches, [past], [tokens], heads, kv_heads, w)
    assert np.isfinite(got).all() and np.abs(got).max() <= 1.001 * c.tops()[0].max()
    assert got.any(1).all()


@pytest.mark.parametrize("powers", [(-70,), (-90,), (-100,), (-100, -60), (-100, 57), (57,)])
@pytest.mark.parametrize("past", [20, 3000])
@pytest.mark.parametrize("tokens,heads,kv_heads,w", SHAPES)
def test_scales_at_the_ends_of_their_range(tokens, heads, kv_heads, w, past, powers):
    # (the scales lie around 2^-6; alternating ones, and the first half of the rows small)
    r = np.random.default_rng(9)
    q = (r.standard_normal((tokens, heads * w)) * 1.5).astype(np.float32)
    for split in (False, True):
        c = Caches(10, [past + tokens], kv_heads, w)
        at = np.arange(past + tokens)
        which = (at > len(at) // 2) if split else at % 2
        c.scale(0, 2.0 ** np.array(powers)[np.minimum(which, len(powers) - 1)][:, None])
        check(c, q, [past], [tokens], None, heads)


@pytest.mark.parametrize("past", [40, 3000])
@pytest.mark.parametrize("tokens,heads,kv_heads,w", SHAPES)
def test_scales_of_either_sign_and_none(tokens, heads, kv_heads, w, past):
    # a value is its i8 times its scale, whatever made it
    r = np.random.default_rng(11)
    q = (r.standard_normal((tokens, heads * w)) * 1.5).astype(np.float32)
    c = Caches(12, [past + tokens], kv_heads, w)
    c.scale(0, r.choice([-1.0, 0.0, 1.0], (past + tokens, kv_heads)))
    check(c, q, [past], [tokens], None, heads)
    c.scale(0, np.zeros((past + tokens, kv_heads)))
    assert not P.attention_tree(q, c.caches, [past], [tokens], heads, kv_heads, w).any()
