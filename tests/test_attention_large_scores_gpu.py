"""GPU: scores of 2^22 and more, where neighbouring floats lie further apart than
the probabilities' headroom. A result is a mean of values all the same."""
import numpy as np
import pytest

import prana_amd as P
from tests.test_tree_attention_gpu import make

pytestmark = pytest.mark.gpu

LOG2E = 1.4426950408889634


def neighbours(rows, at, w, size):
    """q [rows, w] and k [rows, w]: a score of `size` (log2 units) against the keys before `at`, one float more
    against those from there on."""
    q, k = np.zeros((rows, w), np.float32), np.zeros((rows, w), np.float16)
    q[:, 0] = np.float32(size * np.sqrt(w) / LOG2E)
    q[:, 1] = np.spacing(np.float32(size)) * np.sqrt(w) / LOG2E
    k[:, 0], k[at:, 1] = 1, 1
    return q, k


# (floats are 0.5, 1, 2, 4, 8, 16 and 64 apart there)
SIZES = [5e6, 1e7, 2e7, 4e7, 1e8, 2e8, 1e9, 1e12]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("w", [64, 96, 128, 200])
@pytest.mark.parametrize("n", [130, 700])
def test_prompts_f32(n, w, size):
    # tiles of 64 and 32 keys, one group of waves and several
    for at in (64, n // 2):
        q, k = neighbours(n, at, w, size)
        v = np.random.default_rng(0).standard_normal((n, w)).astype(np.float16)
        got = P.attention_packed(q, k, v, [n], 1, 1, w)
        assert np.isfinite(got).all() and np.abs(got).max() <= 1.001 * np.abs(v).max()
        assert got.any(1).all()


@pytest.mark.parametrize("w", [64, 96, 128, 200])
@pytest.mark.parametrize("n", [130, 700])
@pytest.mark.parametrize("size", [3e3, 2e4, 6e4])
def test_prompts_f16(n, w, size):
    # products of halves near the end of their range: scores up to 2^36
    r = np.random.default_rng(1)
    q, k = (np.clip(size * (1 + 2.0 ** -8 * r.standard_normal((n, w))), 0, 65504).astype(np.float16) for _ in "qk")
    v = r.standard_normal((n, w)).astype(np.float16)
    got = P.attention_packed(q, k, v, [n], 1, 1, w).astype(np.float32)
    assert np.isfinite(got).all() and np.abs(got).max() <= 1.001 * np.abs(v).max()
    assert got.any(1).all()


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("tokens,heads,w", [(1, 2, 64), (5, 2, 128), (12, 2, 200), (40, 4, 64), (40, 4, 128), (64, 2, 256)])
@pytest.mark.parametrize("past", [480, 3000])
def test_trees_f16(past, tokens, heads, w, size):
    for at in (64, 300, past - 100):
        q, k = neighbours(past + tokens, at, w, size)
        v = np.random.default_rng(2).standard_normal((past + tokens, w)).astype(np.float16)
        got = P.attention_tree(np.tile(q[:tokens], (1, heads)), [P.KvF16(k, v)], [past], [tokens], heads, 1, w)
        assert np.isfinite(got).all() and np.abs(got).max() <= 1.001 * np.abs(v).max()
        assert got.any(1).all()


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("tokens,heads,w", [(5, 2, 64), (12, 2, 96), (40, 4, 128), (64, 2, 256)])
@pytest.mark.parametrize("size", [1e6, 1e8, 1e20])
def test_trees_of_large_queries(kind, tokens, heads, w, size):
    past = 900
    q, caches, _, vs = make(3, kind, [past], [tokens], heads, 1, w, sigma=size)
    got = P.attention_tree(q, caches, [past], [tokens], heads, 1, w)
    assert np.isfinite(got).all() and np.abs(got).max() <= 1.001 * np.abs(vs[0]).max()
    assert got.any(1).all()
