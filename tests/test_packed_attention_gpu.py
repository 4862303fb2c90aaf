"""GPU: causal attention of packed prompts against the 64-bit form, within the
bounds that serving_oracle.py derives."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from prana_amd import _lib
from tests import serving_oracle as SO

pytestmark = pytest.mark.gpu


def inputs(seed, rows, heads, kv_heads, w, half, sigma=1.5):
    r = np.random.default_rng(seed)
    q = (r.standard_normal((rows, heads * w)) * sigma).astype(np.float16 if half else np.float32)
    k, v = (r.standard_normal((rows, kv_heads * w)).astype(np.float16) for _ in "kv")
    return q, k, v


def check(q, k, v, lens, heads, kv_heads, w):
    got = P.attention_packed(q, k, v, lens, heads, kv_heads, w)
    want, bound = SO.packed(q, k, v, lens, heads, kv_heads, w)
    ok, worst = SO.within(got, want, bound)
    assert ok, worst


LENS = [[1], [2, 1, 3], [17, 0, 64, 65, 1, 129], [300, 127, 128]]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,kv_heads,w", [(6, 6, 48), (14, 2, 64), (8, 2, 128), (4, 1, 256), (3, 3, 80),
                                              (6, 2, 96), (2, 1, 8), (5, 1, 40), (2, 2, 160), (3, 1, 200),
                                              (2, 1, 224)])
def test_shapes(heads, kv_heads, w, lens, half):
    q, k, v = inputs(heads * w + sum(lens), sum(lens), heads, kv_heads, w, half)
    check(q, k, v, lens, heads, kv_heads, w)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kv_heads,w,n", [(2, 1, 128, 1500), (7, 1, 64, 1111), (1, 1, 256, 700),
                                                (24, 1, 32, 333)])
def test_longer_prompts(heads, kv_heads, w, n, half):
    q, k, v = inputs(n, n + 5, heads, kv_heads, w, half)
    check(q, k, v, [n, 5], heads, kv_heads, w)


@pytest.mark.parametrize("half", [False, True])
def test_many_sequences(half):
    # more sequences than one launch takes, of lengths 0 to 40
    r = np.random.default_rng(4)
    lens = [int(x) for x in r.integers(0, 41, 300)]
    q, k, v = inputs(5, sum(lens), 4, 2, 64, half)
    check(q, k, v, lens, 4, 2, 64)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kv_heads,w", [(4, 2, 64), (3, 1, 72)])
def test_row_strides(heads, kv_heads, w, half):
    # q | k | v fused in one f16 buffer (f16), or q in wider rows (f32); the
    # result in wider rows too, whose other columns and rows stay as they were
    lens = [33, 90]
    rows, qw, kw = sum(lens), heads * w, kv_heads * w
    q, k, v = inputs(8, rows, heads, kv_heads, w, half)
    want, bound = SO.packed(q, k, v, lens, heads, kv_heads, w)
    ld_kv = qw + 2 * kw + 16
    kv = np.zeros((rows, ld_kv), np.float16)
    kv[:, qw:qw + kw], kv[:, qw + kw:qw + 2 * kw] = k, v
    if half:
        kv[:, :qw] = q
    d = P.DeviceArray.from_host(kv)
    dq = d if half else P.DeviceArray.from_host(np.concatenate([q, np.full((rows, 4), 9, np.float32)], 1))
    ld_q, ld_out = ld_kv if half else qw + 4, qw + 24
    t = np.float16 if half else np.float32
    do = P.DeviceArray.from_host(np.full((rows + 1, ld_out), 5, t))
    lib = _lib.load()
    P.check(lib.prana_attention_packed(dq.ptr, C.c_void_p(d.ptr.value + 2 * qw), C.c_void_p(d.ptr.value + 2 * (qw + kw)),
                                       P.F16 if half else P.F32, (C.c_size_t * 2)(*lens), 2, heads, kv_heads, w, ld_q,
                                       ld_kv, ld_out, do.ptr, None))
    got = do.to_host()
    ok, worst = SO.within(got[:rows, :qw], want, bound)
    assert ok, worst
    assert np.all(got[:rows, qw:] == 5) and np.all(got[rows] == 5)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite_stay_where_they_are_seen(half, bad):
    # row 70 of the first sequence: earlier rows and the other sequence never
    # see it, in K or in V
    lens, heads, kv_heads, w = [100, 60], 2, 1, 64
    q, k, v = inputs(12, 160, heads, kv_heads, w, half)
    clean = P.attention_packed(q, k, v, lens, heads, kv_heads, w)
    v2 = v.copy()
    v2[70, 5] = bad
    got = P.attention_packed(q, k, v2, lens, heads, kv_heads, w)
    hit = np.zeros(got.shape, bool)
    hit[70:100, 5::64] = True
    assert np.array_equal(got[~hit], clean[~hit])
    if np.isnan(bad):
        assert np.isnan(got[hit]).all()
    else:
        assert (got[hit] == bad).all()
    k2 = k.copy()
    k2[70, 3] = np.nan
    got = P.attention_packed(q, k2, v, lens, heads, kv_heads, w)
    assert np.isnan(got[70:100]).all()
    assert np.array_equal(got[:70], clean[:70]) and np.array_equal(got[100:], clean[100:])
    q2 = q.copy()
    q2[30, 64 + 2] = bad  # one row of one head
    got = P.attention_packed(q2, k, v, lens, heads, kv_heads, w)
    hit = np.zeros(got.shape, bool)
    hit[30, 64:] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("sigma", [0.0, 1e-3, 30.0])
def test_flat_and_sharp_scores(half, sigma):
    # equal scores, and scores hundreds apart: rising ones move the maximum at
    # every tile
    n, w = 400, 64
    q, k, v = inputs(21, n, 2, 1, w, half, sigma=sigma)
    k = np.sort(k, 0)  # the largest last
    q = np.abs(q)
    check(q, k, v, [n], 2, 1, w)


@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_f32_queries_beyond_halves(size):
    # values of q that no f16 holds; K scaled the other way where it can be
    n, w = 90, 64
    r = np.random.default_rng(2)
    q = (r.standard_normal((n, w)) * size).astype(np.float32)
    q[::3] = (r.standard_normal((30, w)) * 2).astype(np.float32)  # ordinary rows among them
    q[1::3] *= np.float32(1e-30) if size > 1 else np.float32(1)
    k, v = (r.standard_normal((n, w)).astype(np.float16) for _ in "kv")
    got = P.attention_packed(q, k, v, [n], 1, 1, w)
    want, bound = SO.packed(q, k, v, [n], 1, 1, w)
    rows = np.ones(n, bool)
    if size > 1:  # scores of 1e30: all weight on one row, which 64 bits and 32 agree on unless they tie
        rows[2::3] = False
        assert np.isfinite(got[2::3]).all()
    ok, worst = SO.within(got[rows], want[rows], bound[rows])
    assert ok, worst


@pytest.mark.parametrize("w", [64, 256])
def test_f16_results_at_the_end_of_their_range(w):
    # means of +-65504 and of it alone: no rounding of a weight carries one past it
    n = 150
    q, k, v = inputs(5, n, 2, 1, w, True)
    v[:] = np.float16(65504)
    v[:, 1::2] = np.float16(-65504)
    got = P.attention_packed(q, k, v, [n], 2, 1, w).reshape(n, 2, w)
    # off by the weights' roundings (2^-11) and the result's own, and never past the end
    assert np.isfinite(got).all() and (np.abs(got.astype(np.float64)) >= 65504 * (1 - 2.0 ** -10)).all()
    assert (got[..., 0::2] > 0).all() and (got[..., 1::2] < 0).all()
    v[7, 3] = np.inf  # but an infinity that a row sees is one
    got = P.attention_packed(q, k, v, [n], 2, 1, w).reshape(n, 2, w)
    assert not np.isfinite(got[7:, :, 3]).any() and np.isfinite(got[:7]).all()
    assert np.isfinite(np.delete(got, 3, 2)).all()


@pytest.mark.parametrize("w", [8, 136])
def test_many_small_probabilities_of_an_f16_call_are_not_lost(w):
    # the first key outweighs each other one by 2^25: 20000 of those are 6e-4 of
    # the result. A probability is off by at most 2^-32 of the largest, the rest
    # are the roundings of a probability and of the result (2^-11 each, 2^-25).
    n = 20000
    q, k, v = np.zeros((n, w), np.float16), np.zeros((n, w), np.float16), np.zeros((n, w), np.float16)
    s0 = 25 * np.log(2)
    q[:, 0] = 4
    k[0, 0] = s0 * np.sqrt(w) / 4
    v[1:] = 1
    got = P.attention_packed(q, k, v, [n], 1, 1, w).astype(np.float64)
    p = np.exp(-float(k[0, 0]) * 4 / np.sqrt(w))
    i = np.arange(n)[:, None]
    want = i * p / (1 + i * p)
    assert (np.abs(got - want) <= want * 2.0 ** -10 + 2.0 ** -25 + i * 2.0 ** -32 + want * n * 2.0 ** -23).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("w", [64, 256])
def test_a_query_that_is_not_a_number_spoils_its_row_alone(half, w):
    q, k, v = inputs(9, 200, 4, 2, w, half)
    clean = P.attention_packed(q, k, v, [200], 4, 2, w)
    q[70, w + 5] = np.nan
    got = P.attention_packed(q, k, v, [200], 4, 2, w)
    assert np.isnan(got[70, w:2 * w]).all()
    got[70, w:2 * w] = clean[70, w:2 * w]
    assert np.array_equal(got, clean)


def test_offsets_past_32_bits():
    # f16 rows of a fused buffer 2^24 values apart: q, k and v beside one another,
    # the second prompt 4 GiB behind the first
    heads, w, ld, lens = 1, 8, 1 << 24, [130, 7]
    n = sum(lens)
    q, k, v = inputs(4, n, heads, heads, w, True)
    lib = _lib.load()
    buf = P.DeviceArray((n * ld,), np.uint16)
    host = np.ascontiguousarray(np.concatenate([q, k, v], 1))
    for i in range(n):
        P.check(lib.prana_memcpy_h2d(C.c_void_p(buf.ptr.value + i * ld * 2), C.c_void_p(host[i].ctypes.data), 48))
    out = P.DeviceArray((n, w), np.float16)
    at = [C.c_void_p(buf.ptr.value + 16 * i) for i in range(3)]
    P.check(lib.prana_attention_packed(at[0], at[1], at[2], P.F16, (C.c_size_t * 2)(*lens), 2, heads, heads, w, ld, ld,
                                       w, out.ptr, None))
    want, bound = SO.packed(q, k, v, lens, heads, heads, w)
    ok, worst = SO.within(out.to_host(), want, bound)
    assert ok, worst


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kv_heads,w", [(2, 2, 48), (6, 2, 64), (3, 1, 80), (5, 1, 96), (7, 1, 128), (2, 2, 104)])
def test_few_rows_over_long_prompts(heads, kv_heads, w, half):
    # the keys of a workgroup divided among groups of waves, some of which see
    # nothing: prompts that end in the first group's tile, at and past a round's end
    lens = [700, 3, 0, 257, 64, 65, 129, 1]
    n = sum(lens)
    q, k, v = inputs(13, n, heads, kv_heads, w, half)
    check(q, k, v, lens, heads, kv_heads, w)
    # values that are not finite stay with the rows that see them: row 600 of the first prompt
    clean = P.attention_packed(q, k, v, lens, heads, kv_heads, w)
    v[600, 5], k[690, 7] = np.inf, np.nan  # (KV head 0)
    q[650, 3] = np.nan  # (head 0)
    got = P.attention_packed(q, k, v, lens, heads, kv_heads, w)
    group = heads // kv_heads
    hit = np.zeros(got.shape, bool)
    for h in range(group):
        hit[600:700, h * w + 5] = True
        hit[690:700, h * w:(h + 1) * w] = True
    hit[650, :w] = True
    assert not np.isfinite(got[hit]).any() and np.array_equal(got[~hit], clean[~hit])


def test_empty_calls():
    lib = _lib.load()
    P.init()
    z = (C.c_size_t * 3)(0, 0, 0)
    assert lib.prana_attention_packed(None, None, None, P.F32, z, 3, 8, 2, 64, 0, 0, 0, None, None) == 0
    assert lib.prana_attention_packed(None, None, None, P.F16, None, 0, 8, 2, 64, 0, 0, 0, None, None) == 0
