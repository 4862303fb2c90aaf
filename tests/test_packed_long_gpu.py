"""GPU: packed prompts, key by key: a bound that a lost key passes
(serving_bounds.py), and weights that can be read from the result."""
import numpy as np
import pytest

import prana_amd as P
from tests import serving_bounds as SB
from tests import serving_oracle as SO
from tests.test_packed_attention_gpu import inputs

pytestmark = pytest.mark.gpu

# Whole and divided workgroups, tiles of 64 and 32 keys, 16-row waves.
SHAPES = [(2, 1, 64), (14, 2, 64), (6, 6, 48), (3, 1, 96), (2, 1, 128), (32, 8, 128), (2, 2, 160), (4, 1, 256)]


@pytest.mark.parametrize("heads,kv_heads,w", SHAPES)
@pytest.mark.parametrize("lens", [[1500, 77], [300, 1, 513, 0, 260]])
def test_f32_within_what_errors_leave(heads, kv_heads, w, lens):
    q, k, v = inputs(3, sum(lens), heads, kv_heads, w, False)
    got = P.attention_packed(q, k, v, lens, heads, kv_heads, w)
    kd, vd, at = k.astype(np.float64), v.astype(np.float64), 0
    r = np.random.default_rng(0)
    for n in lens:
        rows = sorted({*r.integers(0, n, 60).tolist(), 0, n - 1}) if n else []
        for h in {0, heads // 2, heads - 1}:
            a, b = h * w, h // (heads // kv_heads) * w
            seen = np.tril(np.ones((n, n), bool))[rows]
            top = np.abs(vd[at:at + n, b:b + w]).max(1, initial=0)
            want, bound = SB.attend(q[at:at + n, a:a + w].astype(np.float64)[rows], kd[at:at + n, b:b + w],
                                    vd[at:at + n, b:b + w], seen, top)
            ok, worst = SO.within(got[at:at + n, a:a + w][rows], want, bound)
            assert ok, worst
        at += n


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kv_heads,w", SHAPES)
@pytest.mark.parametrize("lens", [[1500, 77], [300, 1, 513, 0, 260]])
def test_equal_weights_count_every_key(heads, kv_heads, w, lens, half):
    # scores of 0: column d of a row is the share of the keys before it whose mark is there. Weights of one are
    # halves exactly; an f16 result rounds once (2^-11), which a key of 1500 passes in columns of few marks.
    total = sum(lens)
    columns = np.random.default_rng(1).integers(0, w, total)
    q = np.zeros((total, heads * w), np.float16 if half else np.float32)
    v = np.zeros((total, kv_heads, w), np.float16)
    v[np.arange(total), :, columns] = 1
    k = np.random.default_rng(2).standard_normal((total, kv_heads * w)).astype(np.float16)
    got = P.attention_packed(q, k, v.reshape(total, -1), lens, heads, kv_heads, w).astype(np.float64)
    got, at = got.reshape(total, heads, w), 0
    for n in lens:
        marks = np.zeros((n, w))
        marks[np.arange(n), columns[at:at + n]] = 1
        count = marks.cumsum(0)[:, None, :]
        off = np.abs(got[at:at + n] * np.arange(1, n + 1)[:, None, None] - count)
        assert (off <= (2.0 ** -11 + 2.0 ** -20 if half else 2.0 ** -20) * count + 1e-9 * n).all()
        at += n
