"""CPU: sizes of the serving calls that are refused before the device is touched:
those that come in small integer types, whose sums numpy would wrap, where the
shapes fit the wrapped sum, and those past what one launch can hold."""
import numpy as np
import pytest

import prana_amd as P
from tests.test_serving_refusals import INVALID, Cache, message, packed, rows

SMALL = np.array([200, 100], np.uint8)  # 300 rows; 44 in 8 bits
HALVES = [rows(44, 16, np.float16)] * 2


def test_prompts_whose_launch_would_pass_2_to_32_lanes():
    # heads wider than 128: 512 lanes for 64 rows (of a KV head's group); 4 query heads each
    wide = dict(hd=256, ld_q=2048, ld_kv=512, ld_out=2048)
    assert packed(lens=((1 << 26) - 16,), q=None, **wide) == INVALID and "null buffer" in message()  # (length taken)
    assert packed(lens=(5, 1 << 26), q=None, **wide) == INVALID and "sequence 1 is too long" in message()
    assert packed(lens=(1 << 27,), q=None) == INVALID and "null buffer" in message()


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("call,says", [
    (lambda: P.attention_packed(rows(44, 32), *HALVES, SMALL, 4, 2, 8), "q holds"),
    (lambda: P.attention_packed(rows(300, 32), *HALVES, SMALL, 4, 2, 8), "k and v hold"),
    (lambda: P.kv_write_q8([Cache(rows=300)] * 2, rows(44, 16), rows(44, 16), [0, 0], SMALL), "k and v hold"),
    (lambda: P.attention_tree(rows(4, 32), [Cache(rows=300)] * 5, [0] * 5, np.full(5, 52, np.uint8), 4, 2, 8),
     "q holds"),
    (lambda: P.attention_tree(rows(260, 32), [Cache(rows=300)] * 5, [0] * 5, np.full(5, 52, np.uint8), 4, 2, 8,
                              mask=np.zeros(4, np.uint64)), "one mask word"),
    # 8 heads x 40: 320 values; 64 in 8 bits
    (lambda: P.attention_packed(rows(4, 64), *[rows(4, 40, np.float16)] * 2, [4], np.uint8(8), 1, np.uint8(40)), "q holds"),
    (lambda: P.attention_tree(rows(1, 64), [Cache(n_kv_heads=1, head_dim=40)], [0], [1], np.uint8(8), 1, np.uint8(40)),
     "q holds"),
    (lambda: P.attention_packed(rows(5, 32), *[rows(5, 16, np.float16)] * 2, [2.5, 2.5], 4, 2, 8), "q holds"),
])
def test_sizes_in_small_types(call, says):
    with pytest.raises(ValueError, match=says):
        call()


@pytest.mark.gpu
def test_reads_of_sizes_in_small_types():
    c = P.KvQ8(300, 2, 8)
    r = np.random.default_rng(0)
    k, v = (r.integers(-127, 128, (300, 16)).astype(np.float32) for _ in "kv")
    k[:, ::8], v[:, ::8] = 127, 127  # (scales of 1)
    P.kv_write_q8([c], k, v, [0], [300])
    got = P.kv_read_q8([c, c], np.array([0, 200], np.uint8), SMALL)
    assert np.array_equal(got[0], k) and np.array_equal(got[1], v)
