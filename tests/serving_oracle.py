"""Plain 64-bit forms of the serving operators and the error their kernels may
show, for the GPU tests.

Error of an f32 result. A score is a dot product of w terms whose q operand is
kept to 22 bits (two halves) and whose sum runs in f32, times a constant:
  ds <= (w + 8) 2^-24 sum_i |q_i k_i| / sqrt(w) + |s| 2^-22.
Its probability is off by ds on its own side and by the largest ds in the sum
that divides it, and each rounds a few times (2^-21 together); the weighted sum
of n terms runs in f32 in some order: n 2^-24 of S_d = sum_t p_t |v_td|, twice
for numerator and denominator. So per element
  |got - want| <= S_d (2 ds + 2^-21 + 2 n 2^-24) + 2^-31 sum_t max_d |v|.
The last term: a probability (times its V row's scale) is kept as two halves
of which the smaller has steps of 2^-24, with the largest at 2^7 or more, so
each is off by up to 2^-25 / 2^7 = 2^-32 of the largest, whatever its own size;
an 8-bit row's scale is taken relative to the largest scale, up to a factor of
2. (A row may see one key only but for probabilities of 1e-50, and that key's
value may be 0: the result is then 1e-50 in 64 bits and 0 in f32.)
A half result rounds its probabilities once (2^-11 S_d; those under 2^-14 of
the largest to 2^-25 absolute: 2^-25 sum_t |v_td|) and the result once
(2^-11 |want|, at least 2^-25)."""
import numpy as np

U = 2.0 ** -24


def attend(q, k, v, seen, half=False):
    """One head: q [m, w], k / v [n, w] in f64, seen [m, n] -> (result, bound)."""
    m, w = q.shape
    out, bound = np.zeros((m, v.shape[1])), np.zeros((m, v.shape[1]))
    if k.shape[0] == 0:
        return out, bound
    for i in range(m):
        t = np.nonzero(seen[i])[0]
        if not len(t):
            continue
        s = k[t] @ q[i] / np.sqrt(w)
        ds = ((w + 8) * U * (np.abs(k[t]) @ np.abs(q[i])) / np.sqrt(w) + 4 * U * np.abs(s)).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = p @ v[t]
        sd = p @ np.abs(v[t])
        bound[i] = sd * (2 * ds + 8 * U + 2 * len(t) * U) + 2.0 ** -31 * len(t) * np.abs(v[t]).max()
        if half:
            bound[i] += 2.0 ** -11 * sd + 2.0 ** -25 * np.abs(v[t]).sum(0) + 2.0 ** -11 * np.abs(out[i]) + 2.0 ** -25
    return out, bound


def packed(q, k, v, lens, heads, kv_heads, w):
    """Causal attention of packed prompts: (result, bound) [rows, heads*w]."""
    half = q.dtype == np.float16
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    out, bound, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for n in lens:
        seen = np.tril(np.ones((n, n), bool))
        for h in range(heads):
            c = h // (heads // kv_heads)
            a, b = slice(at, at + n), slice(h * w, (h + 1) * w)
            out[a, b], bound[a, b] = attend(q[a, b], k[a, c * w:(c + 1) * w], v[a, c * w:(c + 1) * w], seen, half)
        at += n
    return out, bound


def tree(q, ks, vs, past, tokens, masks, heads, kv_heads, w):
    """ks / vs: per sequence the cache rows' values in f64; masks: words or None (a chain)."""
    q = q.astype(np.float64)
    out, bound, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for s, (n, m) in enumerate(zip(past, tokens)):
        seen = np.zeros((m, n + m), bool)
        seen[:, :n] = True
        for i in range(m):
            word = (2 << i) - 1 if masks is None else int(masks[at + i])
            for j in range(m):
                seen[i, n + j] = word >> j & 1
        for h in range(heads):
            c = h // (heads // kv_heads)
            a, b = slice(at, at + m), slice(h * w, (h + 1) * w)
            out[a, b], bound[a, b] = attend(q[a, b], ks[s][:n + m, c * w:(c + 1) * w],
                                            vs[s][:n + m, c * w:(c + 1) * w], seen)
        at += m
    return out, bound


def quantize(x, heads, w):
    """(i8 values, scales in f64) of rows x [n, heads*w]: exact integer arithmetic where it decides."""
    x = x.astype(np.float64).reshape(len(x), heads, w)
    amax = np.abs(x).max(-1)
    t = np.abs(x) * 127 / np.where(amax > 0, amax, 1)[..., None]
    q = np.floor(t + 0.5) * np.sign(x)
    return q.reshape(len(x), heads * w).astype(np.int64), np.where(amax > 0, amax / 127, 1.0)


def within(got, want, bound):
    got = np.asarray(got, np.float64)
    off = np.abs(got - want)
    ok = off <= bound
    return bool(np.all(ok)), (float(np.max(off / np.maximum(bound, 1e-300))) if off.size else 0.0)
