"""CPU: the bound of serving_bounds.py is one that the kernels' arithmetic keeps
with a share that can be seen, and that a lost key or lost lower halves pass."""
import numpy as np
import pytest

from tests import serving_bounds as SB


def halves(x):
    hi = x.astype(np.float16)
    return hi.astype(np.float32), (x - hi.astype(np.float32)).astype(np.float16).astype(np.float32)


def arithmetic(q, k, v, lower=True, without=()):
    """The kernels' arithmetic for one row: operands in two halves, products summed in f32 (tiles of 32 keys, one
    after another), the maximum of all keys kept."""
    w = len(q)
    seen = np.ones(len(k), bool)
    seen[list(without)] = False
    k, v = k[seen].astype(np.float32), v[seen].astype(np.float32)
    f = np.float32(2.0 ** (9 - np.floor(np.log2(max(np.abs(q).max(), 2.0 ** -40)))))
    hi, lo = halves(q.astype(np.float32) * f * np.float32(1.4426950408889634 / np.sqrt(w)))
    s = k @ hi + (k @ lo if lower else np.float32(0))
    s = s / f
    p = np.exp2(s - s.max() + np.float32(7))
    hi, lo = halves(p)
    o, l = np.zeros(v.shape[1], np.float32), np.float32(0)
    for t in range(0, len(k), 32):
        a = slice(t, t + 32)
        o = o + hi[a] @ v[a]
        if lower:
            o = o + lo[a] @ v[a]
        l = l + p[a].sum(dtype=np.float32)
    return o / l


def inputs(n, w, sigma, seed=0):
    r = np.random.default_rng(seed)
    q = (r.standard_normal(w) * sigma).astype(np.float32)
    return q, *(r.standard_normal((n, w)).astype(np.float16).astype(np.float64) for _ in "kv")


def share(q, k, v, got):
    want, bound = SB.attend(q[None].astype(np.float64), k, v, np.ones((1, len(k)), bool), np.abs(v).max(1))
    return (np.abs(got - want[0]) / bound[0]).max()


LENGTHS = [64, 511, 3064, 9001, 20002]


@pytest.mark.parametrize("sigma", [0.0, 1.5])
@pytest.mark.parametrize("w", [64, 128])
@pytest.mark.parametrize("n", LENGTHS)
def test_what_the_bound_takes_and_refuses(n, w, sigma):
    q, k, v = inputs(n, w, sigma)
    right = share(q, k, v, arithmetic(q, k, v))
    assert 1e-3 < right < 0.5, right
    if sigma:
        assert share(q, k, v, arithmetic(q, k, v, lower=False)) > 2
    # a key of middling weight, the first, the last; 32 in a row
    p = SB.weights(q.astype(np.float64), k)[0]
    for t in {int(np.argsort(p)[n // 2]), *((0, n - 1) if sigma == 0 else ())}:
        assert share(q, k, v, arithmetic(q, k, v, without=[t])) > 2, t
    assert share(q, k, v, arithmetic(q, k, v, without=range(n // 2, n // 2 + 32))) > 2
