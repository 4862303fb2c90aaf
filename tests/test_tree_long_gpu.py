"""GPU: tree attention over long caches, key by key: a bound that a lost key
passes (serving_bounds.py), weights that can be read from the result, and
queries that see one key among thousands."""
import numpy as np
import pytest

import prana_amd as P
from tests import serving_bounds as SB
from tests import serving_oracle as SO
from tests.test_tree_attention_gpu import KINDS, make, trees

pytestmark = pytest.mark.gpu

# Parts and joins of each kernel: narrow rows in one block, in two (8-bit), wide ones; narrow with four waves.
LONG = [([9000], [1], 4, 1, 128), ([5000, 3, 2500], [7, 2, 30], 4, 2, 64), ([20000], [2], 2, 1, 48),
        ([3000, 3001], [64, 64], 8, 2, 128), ([2000], [33], 32, 1, 32), ([4000, 130], [12, 11], 4, 2, 96),
        ([6000], [3], 4, 1, 256), ([4100], [40], 4, 2, 200), ([700, 4000], [64, 20], 6, 2, 80)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,tokens,heads,kv_heads,w", LONG)
def test_within_what_errors_leave(kind, past, tokens, heads, kv_heads, w):
    q, caches, ks, vs = make(7, kind, past, tokens, heads, kv_heads, w)
    mask = trees(8, tokens)
    got = P.attention_tree(q, caches, past, tokens, heads, kv_heads, w, mask)
    want, bound = SB.tree(q, ks, vs, past, tokens, mask, heads, kv_heads, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


def marked(kind, n, kv_heads, w, every, columns):
    """A cache whose V rows hold 1 in one column (times 127, 8-bit), and the columns [n]."""
    v = np.zeros((n, kv_heads, w))
    v[np.arange(n), :, columns] = every
    k = np.random.default_rng(0).standard_normal((n, kv_heads * w))
    v = v.reshape(n, -1)
    if kind == "f16":
        return P.KvF16(k.astype(np.float16), v.astype(np.float16))
    c = P.KvQ8(n, kv_heads, w)
    P.kv_write_q8([c], k.astype(np.float32), v.astype(np.float32), [0], [n])
    return c


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,tokens,heads,kv_heads,w", [
    (9000, 1, 4, 1, 128), (2500, 5, 4, 2, 64), (20000, 2, 2, 1, 48), (3001, 64, 8, 2, 128), (4000, 12, 4, 2, 96),
    (6000, 3, 4, 1, 256), (4100, 40, 4, 2, 200), (31, 1, 2, 1, 64), (511, 4, 4, 2, 64), (513, 20, 2, 2, 128)])
def test_equal_weights_count_every_key(kind, past, tokens, heads, kv_heads, w):
    # scores of 0: column d of a row is the share of the keys that it sees whose mark is there
    n = past + tokens
    columns = np.random.default_rng(past).integers(0, w, n)
    c = marked(kind, n, kv_heads, w, 1.0, columns)
    got = P.attention_tree(np.zeros((tokens, heads * w), np.float32), [c], [past], [tokens], heads, kv_heads, w)
    got = got.reshape(tokens, heads, w).astype(np.float64)
    for i in range(tokens):
        count = np.bincount(columns[:past + i + 1], minlength=w)
        # sums of equal weights and the division: 2^-20 in all, a lost or doubled key is 1 of at most n
        assert (np.abs(got[i] * (past + i + 1) - count) <= 2.0 ** -20 * count + 1e-9 * n).all()


def one_key(kind, seed, past, targets, heads, kv_heads, w, tokens):
    """Queries [tokens * heads] that give nearly all weight to one key each (targets, of the past rows)."""
    q, caches, ks, vs = make(seed, kind, [past], [tokens], heads, kv_heads, w)
    group = heads // kv_heads
    q = q.reshape(tokens, heads, w)
    for i in range(tokens):
        for h in range(heads):
            k = ks[0][targets[(i * heads + h) % len(targets)], (h // group) * w:][:w]
            q[i, h] = 40 * np.sqrt(w) * k / (k @ k)
    return q.reshape(tokens, -1), caches, ks, vs


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,tokens,heads,kv_heads,w,step", [
    (9000, 64, 8, 2, 64, 32), (3003, 40, 8, 2, 128, 32), (3000, 64, 6, 1, 96, 32), (5000, 48, 4, 1, 256, 64),
    (9001, 2, 8, 1, 128, 256), (2777, 3, 4, 1, 64, 256), (5000, 12, 4, 2, 64, 256), (4000, 4, 2, 1, 200, 128)])
def test_the_first_and_last_keys_of_tiles_rounds_and_parts(kind, past, tokens, heads, kv_heads, w, step):
    # (a part is a whole number of tiles, so its ends are some tile's)
    ends = np.array(sorted({t for a in range(0, past, step) for t in (a - 1, a, a + 1) if 0 <= t < past} | {past - 1}))
    for first in range(0, len(ends), tokens * heads):
        targets = ends[first:first + tokens * heads]
        q, caches, ks, vs = one_key(kind, 5, past, targets, heads, kv_heads, w, tokens)
        got = P.attention_tree(q, caches, [past], [tokens], heads, kv_heads, w)
        want, bound = SB.tree(q, ks, vs, [past], [tokens], None, heads, kv_heads, w)
        ok, worst = SO.within(got, want, bound)
        assert ok, (first, worst)


def test_a_bound_is_passed_by_a_cache_without_one_row():
    # the same call over a cache that lacks one row of 9001: 64 bits would not take the result
    heads, kv_heads, w, past = 4, 1, 64, 9001
    q, caches, ks, vs = make(3, "f16", [past], [1], heads, kv_heads, w)
    k, v = (c.to_host() for c in (caches[0].k, caches[0].v))
    lost = np.delete(np.arange(len(k)), 4567)
    got = P.attention_tree(q, [P.KvF16(k[lost], v[lost])], [past - 1], [1], heads, kv_heads, w)
    want, bound = SB.tree(q, ks, vs, [past], [1], None, heads, kv_heads, w)
    assert not SO.within(got, want, bound)[0]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("w,past", [(64, 6000), (64, 30000), (256, 2000), (256, 9000)])
def test_single_tokens_beside_a_tree_on_one_kernel_and_on_two(kind, w, past):
    # few cache rows go along on the wide kernel, more on their own
    heads, kv_heads, lens, tokens = 4, 4, [500, past // 2, past, 7], [40, 1, 1, 2]
    q, caches, ks, vs = make(11, kind, lens, tokens, heads, kv_heads, w)
    got = P.attention_tree(q, caches, lens, tokens, heads, kv_heads, w)
    want, bound = SB.tree(q, ks, vs, lens, tokens, None, heads, kv_heads, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst
