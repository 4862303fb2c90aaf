"""GPU: the serving operators as a server uses them: prompts are attended to
and their rows quantized into 8-bit caches, drafted trees are verified over
those, the accepted path stays; on a caller's stream, captured into graphs, and
without touching anything beside their outputs."""
import ctypes as C

import numpy as np
import pytest

import prana_amd as P
from prana_amd import _lib
from tests import serving_oracle as SO

pytestmark = pytest.mark.gpu

H, G, W = 8, 2, 64  # heads, KV heads, head width
# A scale is rounded in the library and here: 2^-24 of a value each way at most,
# one more beside the bound's (w + 8) 2^-24 of a score and 8 2^-24 of the sum.
SCALES = 9 / 8


def runtime():
    """The HIP runtime that the library has loaded."""
    P.init()
    _lib.load()
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    return C.CDLL(path)


def ok(rc):
    assert rc == 0, rc


class Stream:
    def __init__(self, hip):
        self.hip, self.s = hip, C.c_void_p()
        ok(hip.hipStreamCreate(C.byref(self.s)))

    def wait(self):
        ok(self.hip.hipStreamSynchronize(self.s))

    def capture(self, calls):
        graph, run = C.c_void_p(), C.c_void_p()
        ok(self.hip.hipStreamBeginCapture(self.s, 0))
        calls()
        ok(self.hip.hipStreamEndCapture(self.s, C.byref(graph)))
        ok(self.hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
        return run

    def replay(self, run):
        ok(self.hip.hipGraphLaunch(run, self.s))


def upload(d, a):
    a = np.ascontiguousarray(a)
    P.check(_lib.load().prana_memcpy_h2d(d.ptr, C.c_void_p(a.ctypes.data), a.nbytes))


def sizes(v):
    return (C.c_size_t * max(len(v), 1))(*v)


def values(x, kv_heads=G, w=W):
    """What the 8-bit cache holds for rows x, in f64."""
    q, s = SO.quantize(x, kv_heads, w)
    s = s.astype(np.float32).astype(np.float64)
    return (q.reshape(len(x), kv_heads, w) * s[..., None]).reshape(len(x), kv_heads * w)


def rows(r, n, width):
    return r.standard_normal((n, width)).astype(np.float32)


def test_prompts_a_drafted_tree_and_the_accepted_path():
    r = np.random.default_rng(3)
    lens, n = [300, 0, 17, 1], 4
    q, k, v = rows(r, sum(lens), H * W), rows(r, sum(lens), G * W), rows(r, sum(lens), G * W)
    got = P.attention_packed(q, k.astype(np.float16), v.astype(np.float16), lens, H, G, W)
    want, bound = SO.packed(q, k.astype(np.float16), v.astype(np.float16), lens, H, G, W)
    assert SO.within(got, want, bound)[0]

    caches = [P.KvQ8(m + 100, G, W) for m in lens]
    P.kv_write_q8(caches, k, v, [0] * n, lens)
    at = np.cumsum([0] + lens)
    held = [[values(x[at[i]:at[i + 1]]) for x in (k, v)] for i in range(n)]  # per sequence (k, v)
    past = list(lens)
    for step, tree in enumerate(([5, 1, 64, 12], [1, 1, 1, 1], [7, 0, 3, 30])):
        q, k, v = (rows(r, sum(tree), x * W) for x in (H, G, G))
        parents = [[int(r.integers(-1, i)) if i else -1 for i in range(m)] for m in tree]
        mask = np.concatenate([P.tree_mask(p) for p in parents])
        P.kv_write_q8(caches, k, v, past, tree)
        got = P.attention_tree(q, caches, past, tree, H, G, W, mask)
        at = np.cumsum([0] + tree)
        drafted = [[values(x[at[i]:at[i + 1]]) for x in (k, v)] for i in range(n)]
        ks, vs = ([np.concatenate([held[i][c], drafted[i][c]]) for i in range(n)] for c in (0, 1))
        want, bound = SO.tree(q, ks, vs, past, tree, mask, H, G, W)
        worst = SO.within(got, want, bound * SCALES)
        assert worst[0], (step, worst)
        # the longest path is accepted: its rows move up behind the past ones
        moved_k, moved_v, kept = [], [], []
        for i in range(n):
            path, t = [], tree[i] - 1
            while t >= 0:
                path.insert(0, t)
                t = parents[i][t]
            kept.append(len(path))
            moved_k.append(k[at[i]:at[i + 1]][path])
            moved_v.append(v[at[i]:at[i + 1]][path])
            for c in (0, 1):
                held[i][c] = np.concatenate([held[i][c], drafted[i][c][path]])
        P.kv_write_q8(caches, np.concatenate(moved_k), np.concatenate(moved_v), past, kept)
        past = [p + m for p, m in zip(past, kept)]
    back = P.kv_read_q8(caches, [0] * n, past)
    for c in (0, 1):
        all_rows = np.concatenate([held[i][c] for i in range(n)])
        # a scale's division rounds once (2^-24) and the oracle's once more, the product once
        assert (np.abs(back[c] - all_rows) <= 3 * 2.0 ** -24 * np.abs(all_rows)).all()


class Step:
    """A verify step with its buffers on the device: the drafted rows go into
    the caches, attention follows."""

    def __init__(self, seed, past, tree, w=W):
        self.r, self.past, self.tree, self.w = np.random.default_rng(seed), past, tree, w
        n = sum(tree)
        self.caches = [P.KvQ8(p + t, G, w) for p, t in zip(past, tree)]
        P.kv_write_q8(self.caches, rows(self.r, sum(past), G * w), rows(self.r, sum(past), G * w), [0] * len(past), past)
        self.q, self.k, self.v = (P.DeviceArray((n, x * w), np.float32) for x in (H, G, G))
        self.mask = P.DeviceArray((n,), np.uint64)
        self.out = P.DeviceArray.from_host(np.full((n + 2, H * w), 7, np.float32))  # (two rows behind the last)
        self.bytes = P.attention_tree_workspace(past, tree, H, G, w)
        self.work = P.DeviceArray.from_host(np.full(self.bytes + 256, 0xA5, np.uint8))
        self.inputs()

    def inputs(self):
        for d in (self.q, self.k, self.v):
            upload(d, rows(self.r, *d.shape))
        upload(self.mask, np.concatenate(
            [P.tree_mask([int(self.r.integers(-1, i)) if i else -1 for i in range(m)]) for m in self.tree]))

    def run(self, stream):
        lib, kv, n = _lib.load(), P._kv_structs(self.caches), len(self.past)
        P.check(lib.prana_kv_write_q8(self.k.ptr, self.v.ptr, G * self.w, kv, sizes(self.past), sizes(self.tree), n, G,
                                      self.w, stream))
        P.check(lib.prana_attention_tree(self.q.ptr, P.KV_Q8, kv, sizes(self.past), sizes(self.tree), n, self.mask.ptr,
                                         H, G, self.w, self.out.ptr, self.work.ptr, self.bytes, stream))

    def result(self):
        out = self.out.to_host()
        assert (out[-2:] == 7).all()
        assert (self.work.to_host()[self.bytes:] == 0xA5).all()
        return out[:-2]

    def clear(self):
        upload(self.out, np.concatenate([np.zeros((self.out.shape[0] - 2, H * self.w), np.float32),
                                         np.full((2, H * self.w), 7, np.float32)]))


@pytest.mark.parametrize("w", [64, 128, 256])
def test_on_a_stream_of_the_caller_nothing_beside_the_outputs_changes(w):
    s, a = Stream(runtime()), Step(1, [5000, 40, 3000], [1, 30, 9], w=w)
    assert a.bytes > 0  # (the long caches go in parts)
    a.run(None)
    P.check(_lib.load().prana_synchronize())
    want = a.result()
    a.clear()
    a.run(s.s)
    s.wait()
    assert np.array_equal(a.result(), want)


def test_two_calls_at_once_with_workspaces_of_their_own():
    hip = runtime()
    steps = [Step(i, [6000, 7], [4, 50]) for i in (1, 2)]
    want = []
    for a in steps:
        a.run(None)
        P.check(_lib.load().prana_synchronize())
        want.append(a.result())
        a.clear()
    streams = [Stream(hip) for _ in steps]
    for _ in range(5):
        for a, s in zip(steps, streams):
            a.run(s.s)
    for a, s, x in zip(steps, streams, want):
        s.wait()
        assert np.array_equal(a.result(), x)


def test_captured_steps_replay_with_new_inputs_and_eager_calls_between():
    s = Stream(runtime())
    # two graphs, one with parts to join and one without, and an eager step
    steps = [Step(5, [7000, 64, 900], [1, 64, 12]), Step(6, [3, 200], [20, 1])]
    other = Step(7, [4000], [16])
    other.run(None)
    P.check(_lib.load().prana_synchronize())
    other_want = other.result()
    graphs = [s.capture(lambda a=a: a.run(s.s)) for a in steps]
    for turn in range(4):
        for a, g in zip(steps, graphs):
            a.inputs()
            a.run(None)
            P.check(_lib.load().prana_synchronize())
            want = a.result()
            a.clear()
            other.clear()
            s.replay(g)
            other.run(s.s)  # behind the replay
            s.wait()
            assert np.array_equal(a.result(), want), turn
            assert np.array_equal(other.result(), other_want), turn


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_captured_prompts_and_reads(kind):
    s, lib = Stream(runtime()), _lib.load()
    r, lens = np.random.default_rng(8), [90, 0, 700, 5]
    n, t = sum(lens), P.F32 if kind == np.float32 else P.F16
    q, out = P.DeviceArray((n, H * W), kind), P.DeviceArray.from_host(np.full((n + 1, H * W), 7, kind))
    k, v = (P.DeviceArray((n, G * W), np.float32) for _ in "kv")
    k16, v16 = (P.DeviceArray.from_host(np.full((n + 1, G * W), 7, np.float16)) for _ in "kv")
    caches = [P.KvQ8(m, G, W) for m in lens]
    first = [0] * 4

    def run(stream):  # the rows that later steps will read from the 8-bit caches
        kv = P._kv_structs(caches)
        P.check(lib.prana_kv_write_q8(k.ptr, v.ptr, G * W, kv, sizes(first), sizes(lens), 4, G, W, stream))
        P.check(lib.prana_kv_read_q8(kv, sizes(first), sizes(lens), 4, G, W, P.F16, k16.ptr, v16.ptr, G * W, stream))
        P.check(lib.prana_attention_packed(q.ptr, k16.ptr, v16.ptr, t, sizes(lens), 4, H, G, W, H * W, G * W, H * W,
                                           out.ptr, stream))

    graph = s.capture(lambda: run(s.s))
    for turn in range(4):
        qh = r.standard_normal((n, H * W)).astype(kind)
        upload(q, qh)
        upload(k, rows(r, n, G * W))
        upload(v, rows(r, n, G * W))
        run(None)
        P.check(lib.prana_synchronize())
        want = out.to_host()
        assert (want[-1] == 7).all() and all((x.to_host()[-1] == 7).all() for x in (k16, v16))
        upload(out, np.full((n + 1, H * W), 7, kind))
        s.replay(graph)
        s.wait()
        assert np.array_equal(out.to_host(), want), turn
        if turn == 0:
            plain, bound = SO.packed(qh, k16.to_host()[:n], v16.to_host()[:n], lens, H, G, W)
            assert SO.within(want[:n], plain, bound)[0]


def test_the_same_cache_for_two_sequences_and_a_prefix_they_share():
    # reading is free to share: two drafts over one cache, and a shorter past of it
    r = np.random.default_rng(2)
    c = P.KvQ8(900, G, W)
    k, v = rows(r, 900, G * W), rows(r, 900, G * W)
    P.kv_write_q8([c], k, v, [0], [900])
    past, tree = [850, 850, 20, 0], [3, 50, 4, 1]
    q = rows(r, sum(tree), H * W)
    got = P.attention_tree(q, [c] * 4, past, tree, H, G, W)
    ks, vs = [values(k)] * 4, [values(v)] * 4
    want, bound = SO.tree(q, ks, vs, past, tree, None, H, G, W)
    worst = SO.within(got, want, bound * SCALES)
    assert worst[0], worst
