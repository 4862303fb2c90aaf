"""A 64-bit form of attention over a cache with a bound that follows how errors
add up, for the GPU tests (serving_oracle.py's counts every one at its worst,
which over a long cache is far more than a lost key).

The weights. q is kept to 22 bits (two halves, 2^-22 relative), a score's sum
of 2 w products runs in f32 (each addition off by up to 2^-23 of what is summed
so far, also where it truncates), the exponential and the products around it
round a few times (2^-21 together). With R = sqrt(sum_i (q_i k_i)^2), what
independent roundings leave of a sum of w terms, and r = R / sqrt(w):
  eps_t = 2^-22 r + 2^-23 sqrt(2 w) (r + |s_t|) + 2^-22 |s_t| + 2^-21.
The sum. Key t moves the result by p_t (v_t - out) for a relative change of its
weight; the roundings of n keys are independent, and each is at most its eps:
  E1 = sqrt(sum_t (p_t (|v_t| + |out|) eps_t)^2).
Both halves' products run through a sum of 2 n terms whose part sums stay near
sqrt(sum_t (p_t v_t)^2) + |out|, 2^-23 each:
  E2 = 2^-23 sqrt(2 n) (sqrt(sum_t (p_t v_t)^2) + |out|).
A weight (times its V scale, 8-bit) has halves down to 2^-25 with the largest
of the row at 2^6 or more, so none is better than 2^-31 of that:
  E3 = 2^-31 sqrt(n) max_t (p_t top_t), top_t the largest |v_t| (8-bit: 127 scales).
Uniform roundings have a deviation of 0.58 of their largest, so
  bound = 8 (E1 + E2 + E3) + 2^-22 |out|
is about 14 deviations. A lost key moves the result by p_t (v_t - out), which is
eps_t^-1 / sqrt(n) times as much as E1 allows for: over 2^17 at n = 64, over
2^10 at 2^20 rows."""
import numpy as np


def weights(q, k):
    """(p, eps) of one row q over the keys k, f64."""
    w = len(q)
    s = k @ q / np.sqrt(w)
    r = np.sqrt((k * k) @ (q * q)) / np.sqrt(w)
    p = np.exp(s - s.max())
    p /= p.sum()
    eps = 2.0 ** -22 * r + 2.0 ** -23 * np.sqrt(2 * w) * (r + np.abs(s)) + 2.0 ** -22 * np.abs(s) + 2.0 ** -21
    return p, eps


def attend(q, k, v, seen, top):
    """One head: q [m, w], k / v [n, w] in f64, seen [m, n], top [n] -> (result, bound)."""
    out, bound = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    for i in range(len(q)):
        t = np.nonzero(seen[i])[0]
        if not len(t):
            continue
        p, eps = weights(q[i], k[t])
        out[i] = p @ v[t]
        a, o = np.abs(v[t]), np.abs(out[i])
        e1 = np.sqrt((((p * eps)[:, None] * (a + o)) ** 2).sum(0))
        e2 = 2.0 ** -23 * np.sqrt(2 * len(t)) * (np.sqrt(((p[:, None] * a) ** 2).sum(0)) + o)
        e3 = 2.0 ** -31 * np.sqrt(len(t)) * (p * top[t]).max()
        bound[i] = 8 * (e1 + e2 + e3) + 2.0 ** -22 * o
    return out, bound


def seen_by(past, tokens, words):
    """Which of past + tokens rows each drafted token sees; words: its masks, None = a chain."""
    seen = np.zeros((tokens, past + tokens), bool)
    seen[:, :past] = True
    for i in range(tokens):
        word = (2 << i) - 1 if words is None else int(words[i])
        for j in range(tokens):
            seen[i, past + j] = word >> j & 1
    return seen


def tree(q, ks, vs, past, tokens, masks, heads, kv_heads, w, tops=None):
    """ks / vs: per sequence the cache rows' values in f64, tops [rows, kv_heads] the bound of a head's values
    (None: its largest); masks: words of all tokens or None (a chain)."""
    q = q.astype(np.float64)
    out, bound, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for s, (n, m) in enumerate(zip(past, tokens)):
        seen = seen_by(n, m, None if masks is None else masks[at:at + m])
        for h in range(heads):
            c = h // (heads // kv_heads)
            a, b, kv = slice(at, at + m), slice(h * w, (h + 1) * w), slice(c * w, (c + 1) * w)
            k, v = ks[s][:n + m, kv], vs[s][:n + m, kv]
            top = np.abs(v).max(1) if tops is None else tops[s][:n + m, c]
            out[a, b], bound[a, b] = attend(q[a, b], k, v, seen, top)
        at += m
    return out, bound
