"""CPU: what the serving entry points refuse. Every check runs before the
device is touched, so none of these calls needs a GPU, and no pointer here is
ever followed."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from prana_amd import _lib

INVALID = -1
AT = 1 << 20  # an address on 16 bytes that nothing reads


def sizes(*v):
    return (C.c_size_t * max(len(v), 1))(*v)


def packed(q=AT, k=AT, v=AT, kind=P.F32, lens=(5, 7), heads=8, kv_heads=2, hd=64, ld_q=512, ld_kv=128, ld_out=512,
           out=AT, lens_ptr=True):
    return _lib.load().prana_attention_packed(q, k, v, kind, sizes(*lens) if lens_ptr else None, len(lens), heads,
                                              kv_heads, hd, ld_q, ld_kv, ld_out, out, None)


def message():
    return _lib.load().prana_last_error().decode()


@pytest.mark.parametrize("change,says", [
    (dict(kind=P.Q8_0), "PRANA_F32 or PRANA_F16"),
    (dict(heads=7), "multiple of n_kv_heads"),
    (dict(kv_heads=0), "multiple of n_kv_heads"),
    (dict(heads=0), "multiple of n_kv_heads"),
    (dict(heads=1 << 17, ld_q=1 << 24, ld_out=1 << 24), "65535 heads"),
    (dict(hd=0), "multiple of 8 up to 256"),
    (dict(hd=36), "multiple of 8 up to 256"),
    (dict(hd=264, ld_q=2112, ld_kv=528, ld_out=2112), "multiple of 8 up to 256"),
    (dict(lens_ptr=False), "null seq_lens"),
    (dict(lens=(1 << 31,)), "sequence 0 is too long"),
    (dict(lens=(3, 1 << 29)), "sequence 1 is too long"),  # 2^29 rows of a group of 4: 2^31
    (dict(q=None), "null buffer"),
    (dict(k=None), "null buffer"),
    (dict(v=None), "null buffer"),
    (dict(out=None), "null buffer"),
    (dict(q=AT + 4), "16-byte aligned"),
    (dict(k=AT + 2), "16-byte aligned"),
    (dict(v=AT + 8), "16-byte aligned"),
    (dict(out=AT + 8), "16-byte aligned"),
    (dict(ld_q=514), "multiples of 16 bytes"),
    (dict(kind=P.F16, ld_q=516), "multiples of 16 bytes"),
    (dict(ld_kv=132), "multiples of 16 bytes"),
    (dict(ld_out=513), "multiples of 16 bytes"),
    (dict(ld_q=508), "shorter than its row"),
    (dict(ld_kv=120), "shorter than its row"),
    (dict(ld_out=508), "shorter than its row"),
    (dict(ld_q=1 << 40), "too long"),
])
def test_packed_refuses(change, says):
    assert packed(**change) == INVALID
    assert says in message() and message().startswith("attention_packed")


def caches(n=2, rows=64, k=AT, v=AT, ks=AT, vs=AT):
    return (P.PranaKv * n)(*[P.PranaKv(k, v, ks, vs, rows) for _ in range(n)])


KV_CHANGES = [
    (dict(kv=None), "null argument"),
    (dict(first=None), "null argument"),
    (dict(rows=None), "null argument"),
    (dict(kv_heads=0), "multiple of n_kv_heads"),
    (dict(hd=20), "multiple of 8 up to 256"),
    (dict(rows=(65, 1)), "sequence 0: rows past the end"),
    (dict(first=(0, 62)), "sequence 1: rows past the end"),
    (dict(first=((1 << 64) - 1, 0)), "sequence 0: rows past the end"),
    (dict(rows=(1, (1 << 64) - 1)), "sequence 1: rows past the end"),
    (dict(kv=caches(k=None)), "sequence 0: null cache pointer"),
    (dict(kv=caches(v=None)), "null cache pointer"),
    (dict(kv=caches(ks=None)), "null cache pointer"),
    (dict(kv=caches(vs=None)), "null cache pointer"),
    (dict(kv=caches(k=AT + 8)), "caches must be 16-byte aligned"),
    (dict(kv=caches(vs=AT + 2)), "scales must be 4-byte aligned"),
    (dict(kv=caches(rows=(1 << 30) + 1)), "more than 2^30 rows"),
    (dict(k=None), "null buffer"),
    (dict(v=None), "null buffer"),
    (dict(k=AT + 4), "buffers must be 16-byte aligned"),
    (dict(ld=258), "multiple of 16 bytes"),
    (dict(ld=248), "shorter than a row"),
    (dict(ld=1 << 62), "too long"),
]


def kv_call(write, kv=caches(), first=(0, 5), rows=(3, 4), kv_heads=4, hd=64, k=AT, v=AT, ld=256, kind=P.F32, n=2):
    lib = _lib.load()
    f, r = (None if x is None else sizes(*x) for x in (first, rows))
    if write:
        return lib.prana_kv_write_q8(k, v, ld, kv, f, r, n, kv_heads, hd, None)
    return lib.prana_kv_read_q8(kv, f, r, n, kv_heads, hd, kind, k, v, ld, None)


@pytest.mark.parametrize("write", [True, False])
@pytest.mark.parametrize("change,says", KV_CHANGES)
def test_kv_refuses(write, change, says):
    assert kv_call(write, **change) == INVALID
    assert says in message() and message().startswith("kv_write_q8" if write else "kv_read_q8")


def test_kv_read_refuses_other_types():
    assert kv_call(False, kind=P.Q8_0) == INVALID and "PRANA_F32 or PRANA_F16" in message()
    assert kv_call(False, kind=P.F16, ld=260) == INVALID and "multiple of 16 bytes" in message()


def tree(q=AT, kind=P.KV_Q8, kv=caches(), past=(10, 20), tokens=(3, 4), mask=AT, heads=8, kv_heads=2, hd=64, out=AT,
         work=AT, nbytes=1 << 40, n=2):
    p, t = (None if x is None else sizes(*x) for x in (past, tokens))
    return _lib.load().prana_attention_tree(q, kind, kv, p, t, n, mask, heads, kv_heads, hd, out, work, nbytes, None)


@pytest.mark.parametrize("change,says", [
    (dict(kind=0), "PRANA_KV_F16 or PRANA_KV_Q8"),
    (dict(heads=9), "multiple of n_kv_heads"),
    (dict(hd=12), "multiple of 8 up to 256"),
    (dict(past=None), "null sizes"),
    (dict(tokens=None), "null sizes"),
    (dict(kv=None), "null caches"),
    (dict(tokens=(3, 65)), "sequence 1: more than 64 drafted tokens"),
    (dict(past=(1 << 30, 0)), "sequence 0 is too long"),
    (dict(past=(62, 0)), "sequence 0: rows past the end"),
    (dict(past=(0, 64)), "sequence 1: rows past the end"),
    (dict(kv=caches(k=None)), "null cache pointer"),
    (dict(kv=caches(v=None)), "null cache pointer"),
    (dict(kv=caches(v=AT + 4)), "caches must be 16-byte aligned"),
    (dict(kv=caches(ks=None)), "null scales"),
    (dict(kv=caches(ks=AT + 1)), "scales must be 4-byte aligned"),
    (dict(kv=caches(rows=1 << 31)), "more than 2^30 rows"),
    (dict(q=None), "null buffer"),
    (dict(out=None), "null buffer"),
    (dict(q=AT + 4), "16-byte aligned"),
    (dict(out=AT + 4), "16-byte aligned"),
    (dict(mask=AT + 4), "mask must be 8-byte aligned"),
    (dict(work=AT + 4), "workspace must be 16-byte aligned"),
])
def test_tree_refuses(change, says):
    assert tree(**change) == INVALID
    assert says in message() and message().startswith("attention_tree")


def test_tree_refuses_a_small_workspace():
    past, tokens = (1 << 20, 1 << 20), (64, 64)
    need = P.attention_tree_workspace(past, tokens, 8, 2, 64)
    kv = caches(rows=1 << 21)
    if need:  # long caches are split over their rows, and the parts joined
        assert tree(kv=kv, past=past, tokens=tokens, nbytes=need - 1) == INVALID and str(need) in message()
        assert tree(kv=kv, past=past, tokens=tokens, work=None) == INVALID and "null workspace" in message()


def test_workspace_sizes():
    # nothing drafted: nothing needed
    assert P.attention_tree_workspace([100, 5], [0, 0], 8, 2, 64) == 0
    assert P.attention_tree_workspace([], [], 8, 2, 64) == 0
    n = C.c_size_t()
    lib = _lib.load()
    assert lib.prana_attention_tree_workspace(sizes(1), sizes(65), 1, 8, 2, 64, C.byref(n)) == INVALID
    assert lib.prana_attention_tree_workspace(sizes(1), sizes(5), 1, 8, 2, 64, None) == INVALID
    # bounded by the rows: at most one partial state per 32 rows, head and token
    for past in (0, 1, 31, 511, 5000, 1 << 20):
        for t in (1, 3, 64):
            b = P.attention_tree_workspace([past], [t], 32, 8, 128)
            assert 0 <= b <= 4 * t * 32 * (128 + 2) * (past + t + 31) // 32 + 64


def test_tree_mask():
    m = P.tree_mask([-1, 0, 0, 2, -1])
    assert [int(x) for x in m] == [0b1, 0b11, 0b101, 0b1101, 0b10000]
    for bad in ([0], [-1, 1], [-1, -2]):
        with pytest.raises(ValueError):
            P.tree_mask(bad)


class Cache:
    """A cache that is never touched: the shapes are refused first."""

    def __init__(self, kind=P.KV_Q8, n_kv_heads=2, head_dim=8, rows=9):
        self.kind, self.n_kv_heads, self.head_dim, self.rows = kind, n_kv_heads, head_dim, rows
        self.width = n_kv_heads * head_dim


def rows(n, width, dtype=np.float32):
    return np.zeros((n, width), dtype)


@pytest.mark.parametrize("call,says", [
    (lambda: P.attention_packed(rows(5, 32), rows(5, 16, np.float16), rows(5, 16, np.float16), [2, 2], 4, 2, 8), "q holds"),
    (lambda: P.attention_packed(rows(4, 32), rows(4, 16, np.float16), rows(3, 16, np.float16), [4], 4, 2, 8), "k and v hold"),
    (lambda: P.attention_packed(rows(4, 32), rows(4, 16), rows(4, 16), [4], 4, 2, 8), "halves"),
    (lambda: P.attention_packed(rows(4, 32, np.float64), *[rows(4, 16, np.float16)] * 2, [4], 4, 2, 8), "f32 or f16"),
    (lambda: P.attention_packed(rows(4, 32), *[rows(4, 16, np.float16)] * 2, [5, -1], 4, 2, 8), "negative"),
    (lambda: P.kv_write_q8([Cache()], rows(4, 16), rows(4, 16), [0], [3]), "k and v hold"),
    (lambda: P.kv_write_q8([Cache()], rows(3, 8), rows(3, 8), [0], [3]), "k and v hold"),
    (lambda: P.kv_write_q8([Cache()] * 2, rows(3, 16), rows(3, 16), [0], [3]), "one size"),
    (lambda: P.kv_write_q8([Cache(P.KV_F16)], rows(3, 16), rows(3, 16), [0], [3]), "another kind"),
    (lambda: P.kv_write_q8([Cache(), Cache(n_kv_heads=1, head_dim=16)], rows(3, 16), rows(3, 16), [0, 0], [1, 2]),
     "other heads"),
    (lambda: P.kv_read_q8([], [], []), "no cache"),
    (lambda: P.kv_read_q8([Cache()], [0, 1], [3]), "one size"),
    (lambda: P.kv_read_q8([Cache(), Cache(head_dim=16)], [0, 1], [3, 3]), "not 16 values"),
    (lambda: P.attention_tree(rows(3, 32), [Cache(), Cache(P.KV_F16)], [2, 2], [1, 2], 4, 2, 8), "another kind"),
    (lambda: P.attention_tree(rows(3, 32), [Cache(head_dim=16)], [2], [3], 4, 2, 8), "not 16 values"),
    (lambda: P.attention_tree(rows(3, 32), [Cache(n_kv_heads=1, head_dim=16)], [2], [3], 4, 2, 8), "other heads"),
    (lambda: P.attention_tree(rows(3, 32), [Cache()], [2], [2], 4, 2, 8), "q holds"),
    (lambda: P.attention_tree(rows(3, 32), [Cache()], [2, 2], [3], 4, 2, 8), "one size"),
    (lambda: P.attention_tree(rows(3, 32), [Cache()], [2], [3], 4, 2, 8, mask=[1, 3]), "one mask word"),
    (lambda: P.attention_tree_workspace([1, 2], [1], 4, 2, 8), "one size"),
])
def test_shapes_that_do_not_belong_together(call, says):
    with pytest.raises(ValueError, match=says):
        call()


def test_a_sequence_of_more_than_2_to_30_rows_and_heads():
    assert packed(lens=((1 << 27) + 1,)) == INVALID and "sequence 0 is too long" in message()
    assert packed(lens=(1 << 27,), q=None) == INVALID and "null buffer" in message()  # (its length is taken)
