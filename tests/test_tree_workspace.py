"""CPU: the workspace of a tree call never shrinks as its sizes grow, so that one
allocated for the largest sizes serves every smaller call."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from tests.test_tree_attention_gpu import make


def sizes(values):
    return (C.c_size_t * len(values))(*values)


SHAPES = [(32, 8, 128), (14, 2, 64), (6, 6, 48), (8, 1, 256), (12, 4, 96), (64, 1, 8), (3, 1, 200)]


@pytest.mark.parametrize("heads,kv_heads,w", SHAPES)
def test_more_of_anything_needs_no_less(heads, kv_heads, w):
    r = np.random.default_rng(heads * w)
    need = lambda past, tree: P.attention_tree_workspace(past, tree, heads, kv_heads, w)  # noqa: E731
    for _ in range(300):
        n = int(r.integers(1, 12))
        past = [int(x) for x in np.exp(r.uniform(0, 13, n))]
        drafted = [int(x) for x in r.integers(0, 65, n)]
        large = need(past, drafted)
        small_past = [int(x) for x in np.array(past) * r.uniform(0, 1, n) ** 0.3]
        small_tree = [int(x) for x in np.array(drafted) * r.uniform(0, 1, n) ** 0.3]
        some = int(r.integers(0, n + 1))
        assert need(small_past, drafted) <= large
        assert need(past, small_tree) <= large
        assert need(small_past[:some], small_tree[:some]) <= large


@pytest.mark.parametrize("tokens", [1, 4, 64])
def test_along_a_cache_that_grows(tokens):
    last = 0
    for past in range(0, 40000, 37):
        b = P.attention_tree_workspace([past], [tokens], 32, 8, 128)
        assert b >= last
        last = b


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_one_workspace_for_every_length(kind):
    heads, kv_heads, w, tokens = 8, 2, 128, 64
    longest = [9000, 5000]
    q, kv, _, _ = make(1, kind, longest, [tokens] * 2, heads, kv_heads, w)
    need = P.attention_tree_workspace(longest, [tokens] * 2, heads, kv_heads, w)
    work, out, dq = P.DeviceArray((need,), np.uint8), P.DeviceArray(q.shape, np.float32), P.DeviceArray.from_host(q)
    for past, tree in (([9000, 5000], [64, 64]), ([4032, 4100], [64, 1]), ([130, 8000 - 3001], [40, 3]), ([7000], [9]),
                       ([0, 2000], [64, 64])):
        n = sum(tree)
        want = P.attention_tree(q[:n], kv[:len(past)], past, tree, heads, kv_heads, w)
        P.check(P.load().prana_attention_tree(dq.ptr, kv[0].kind, P._kv_structs(kv), sizes(past), sizes(tree), len(past),
                                              None, heads, kv_heads, w, out.ptr, work.ptr, need, None))
        assert np.array_equal(out.to_host()[:n], want)
