"""GPU: infinities and NaN in K, V and their scales, and rows that see nothing, on
every attention kernel: narrow rows in one block and in two, wide ones, prompts
of 32-row and 16-row waves, at every width class."""
import numpy as np
import pytest

import prana_amd as P
from tests import serving_oracle as SO
from tests.test_packed_attention_gpu import inputs
from tests.test_tree_attention_gpu import KINDS, make

pytestmark = pytest.mark.gpu

TREES = [(5, 2), (12, 2), (40, 4), (64, 4)]  # tokens, query heads per KV head: 10, 24, 160 and 256 rows
WIDTHS = [64, 96, 128, 200, 256]
BAD = [np.inf, -np.inf, np.nan]
KV = 2


def tree_of(tokens):
    """Token 2 is seen by itself and token 3 alone, the last one by itself."""
    return P.tree_mask([-1, 0, 0, 2] + [int(x) for x in np.random.default_rng(tokens).choice([0, 1], tokens - 4)])


def hits(tokens, group, w, rows, kv_head, column=None):
    """Results of `rows` in the heads of a KV head, one column of it or all."""
    hit = np.zeros((tokens, KV, group, w), bool)
    hit[rows, kv_head, :, slice(None) if column is None else column] = True
    return hit.reshape(tokens, -1)


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("past", [0, 37, 3000])
@pytest.mark.parametrize("w", WIDTHS)
@pytest.mark.parametrize("tokens,group", TREES)
def test_f16_trees(tokens, group, w, past, bad):
    heads, mask, n = KV * group, tree_of(tokens), past + tokens
    q, caches, _, _ = make(8, "f16", [past], [tokens], heads, KV, w)
    run = lambda k, v: P.attention_tree(q, [P.KvF16(k, v)], [past], [tokens], heads, KV, w, mask)  # noqa: E731
    clean = P.attention_tree(q, caches, [past], [tokens], heads, KV, w, mask)
    k, v = (c.to_host().view(np.float16) for c in (caches[0].k, caches[0].v))
    k[n:], v[n:] = bad, bad  # behind the tree
    # a sibling's value, and all of another token's rows, which itself alone sees
    v[past + 2, w + 3] = bad
    k[n - 1], v[n - 1] = bad, bad
    got = run(k, v)
    hit = hits(tokens, group, w, [2, 3], 1, 3)
    own = np.zeros_like(hit)
    own[tokens - 1] = True
    rest = ~hit & ~own
    assert np.array_equal(got[rest], clean[rest])
    assert np.isnan(got[hit]).all() if np.isnan(bad) else (got[hit] == bad).all()
    assert not np.isfinite(got[own]).any()
    k[past + 2, 5] = np.nan  # a score of KV head 0
    got = run(k, v)
    hit2 = hits(tokens, group, w, [2, 3], 0)
    rest = ~hit & ~hit2 & ~own
    assert np.isnan(got[hit2]).all() and np.array_equal(got[rest], clean[rest])
    if past:  # a value that every row sees, in a tile with and without masks
        k, v = (c.to_host().view(np.float16) for c in (caches[0].k, caches[0].v))
        for row in {0, past // 2, past - 1}:
            v2 = v.copy()
            v2[row, 9] = bad
            got = run(k, v2)
            hit = hits(tokens, group, w, list(range(tokens)), 0, 9)
            assert not np.isfinite(got[hit]).any() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("past", [0, 37, 3000])
@pytest.mark.parametrize("w", WIDTHS)
@pytest.mark.parametrize("tokens,group", TREES)
def test_q8_trees(tokens, group, w, past):
    heads, mask, n = KV * group, tree_of(tokens), past + tokens
    r = np.random.default_rng(6)
    q = r.standard_normal((tokens, heads * w)).astype(np.float32)
    k, v = (r.standard_normal((n + 3, KV * w)).astype(np.float32) for _ in "kv")

    def run(k, v):
        c = P.KvQ8(n + 3, KV, w)
        P.kv_write_q8([c], k, v, [0], [n + 3])
        return P.attention_tree(q, [c], [past], [tokens], heads, KV, w, mask)

    clean = run(k, v)
    for which in "kv":
        k2, v2 = k.copy(), v.copy()
        k2[n:], v2[n:] = np.nan, np.inf
        bad = k2 if which == "k" else v2
        bad[past + 2, w + 3] = np.inf
        bad[n - 1] = np.nan
        got = run(k2, v2)
        hit = hits(tokens, group, w, [2, 3], 1)
        hit[tokens - 1] = True
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
        if past:
            k2, v2 = k.copy(), v.copy()
            (k2 if which == "k" else v2)[past // 2, 7] = np.nan
            got = run(k2, v2)
            hit = hits(tokens, group, w, list(range(tokens)), 0)
            assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("w", WIDTHS)
@pytest.mark.parametrize("tokens,group", TREES)
def test_rows_that_see_nothing(tokens, group, w, kind):
    # a tree over no past with empty masks, beside one that is long enough for parts
    heads, past, tree = KV * group, [0, 3000], [tokens, tokens]
    q, caches, ks, vs = make(5, kind, past, tree, heads, KV, w)
    mask = np.concatenate([tree_of(tokens)] * 2)
    empty = [0, tokens // 2, tokens - 1]
    mask[empty] = 0
    if tokens < 64:
        mask[1] = ((1 << 64) - 1) >> tokens << tokens  # bits past the tree
        empty.append(1)
    mask[tokens] = 0  # (sees the past rows)
    got = P.attention_tree(q, caches, past, tree, heads, KV, w, mask)
    assert not got[empty].any()
    own = mask & np.uint64((1 << tokens) - 1)
    want, bound = SO.tree(q, ks, vs, past, tree, own, heads, KV, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("w", [48, 64, 96, 128, 160, 200, 256])
@pytest.mark.parametrize("heads,lens", [(2, [100, 60]), (6, [300, 129, 5]), (16, [70, 700])])
def test_prompts(heads, lens, w, half, bad):
    total, row = sum(lens), lens[0] - 30
    group = heads // KV
    q, k, v = inputs(12, total, heads, KV, w, half)
    clean = P.attention_packed(q, k, v, lens, heads, KV, w)
    first = np.arange(total) < lens[0]
    after = (first & (np.arange(total) >= row))[:, None, None, None]
    v2 = v.copy()
    v2[row, w + 5] = bad  # KV head 1
    got = P.attention_packed(q, k, v2, lens, heads, KV, w)
    hit = np.zeros((total, KV, group, w), bool)
    hit[:, 1, :, 5] = True
    hit = (hit & after).reshape(total, -1)
    # (an infinity times a weight's smaller half, which may be 0, is a NaN)
    assert np.array_equal(got[~hit], clean[~hit]) and not np.isfinite(got[hit]).any()
    assert np.isnan(got[hit]).all() or not np.isnan(bad)
    k2 = k.copy()
    k2[row, 3] = np.nan
    got = P.attention_packed(q, k2, v, lens, heads, KV, w)
    hit = np.zeros((total, KV, group, w), bool)
    hit[:, 0] = True
    hit = (hit & after).reshape(total, -1)
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
    q2 = q.copy()
    q2[row, 2] = bad  # one row of head 0
    got = P.attention_packed(q2, k, v, lens, heads, KV, w)
    hit = np.zeros(got.shape, bool)
    hit[row, :w] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])
