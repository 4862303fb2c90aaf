"""Serving operators around a K/V cache, as measurable cases.

The calls go through the C entry points on device buffers, the way an engine
that binds the library makes them. Inputs are made on the GPU from the seed.

  prompt : causal attention of whole prompts of different lengths packed
           behind one another (prana_attention_packed): f16 K/V rows, q and
           the result in f32 or f16; the f16 form reads q, K and V in place
           from one buffer of fused projections
  kv     : rows of K and V into the 8-bit caches of several sequences
           (prana_kv_write_q8), and back out (prana_kv_read_q8); "write" does
           both, "read" only the second
  tree   : attention of drafted tokens, a tree per sequence, over the
           sequences' caches (prana_attention_tree): f16 or 8-bit ("q8")
           caches, split over the cache rows; a tree of one token is a decode
           step
"""
import ctypes as C
import math
import random

import numpy as np
import torch

own = False

# (query heads, KV heads, head width) of the 15M, 0.5B and 7B shapes, and of other widths the entry points take
HEADS = ((6, 6, 48), (14, 2, 64), (32, 8, 128), (8, 1, 256), (16, 16, 80), (12, 4, 96))


def listed():
    return [
        # three short prompts through the 15M shape: latency counts
        {"name": "prompt_short", "op": "prompt", "type": "f32", "seqs": 3, "longest": 37, "heads": 6, "kv_heads": 6,
         "width": 48},
        # a batch of ordinary prompts through the 0.5B shape
        {"name": "prompt_batch", "op": "prompt", "type": "f32", "seqs": 9, "longest": 1501, "heads": 14,
         "kv_heads": 2, "width": 64},
        # documents through the 7B shape, fused projections in f16
        {"name": "prompt_long", "op": "prompt", "type": "f16", "seqs": 2, "longest": 8191, "heads": 32,
         "kv_heads": 8, "width": 128},
        # wide heads sharing one K/V head
        {"name": "prompt_wide", "op": "prompt", "type": "f16", "seqs": 4, "longest": 1025, "heads": 8, "kv_heads": 1,
         "width": 256},
        # one decode step's K/V rows of eight sequences
        {"name": "kv_step", "op": "kv", "mode": "write", "type": "f32", "seqs": 8, "longest": 1, "kv_heads": 8,
         "width": 128},
        # the K/V rows of four prompts
        {"name": "kv_prompt", "op": "kv", "mode": "write", "type": "f32", "seqs": 4, "longest": 8191, "kv_heads": 8,
         "width": 128},
        # a long cache back to f16, for an operator that takes f16 rows
        {"name": "kv_read", "op": "kv", "mode": "read", "type": "f16", "seqs": 1, "longest": 32767, "kv_heads": 8,
         "width": 128},
        # one sequence, one token, a short cache: the smallest decode step
        {"name": "tree_token", "op": "tree", "cache": "f16", "seqs": 1, "longest": 511, "tokens": 1, "heads": 32,
         "kv_heads": 8, "width": 128},
        # a few drafted tokens in each of four chats on the 0.5B shape
        {"name": "tree_draft", "op": "tree", "cache": "f16", "seqs": 4, "longest": 4099, "tokens": 13, "heads": 14,
         "kv_heads": 2, "width": 64},
        # the widest trees over long caches
        {"name": "tree_wide", "op": "tree", "cache": "f16", "seqs": 8, "longest": 16385, "tokens": 64, "heads": 32,
         "kv_heads": 8, "width": 128},
        # a decode step of eight long sequences over 8-bit caches
        {"name": "tree_q8_token", "op": "tree", "cache": "q8", "seqs": 8, "longest": 32767, "tokens": 1, "heads": 32,
         "kv_heads": 8, "width": 128},
        # drafted tokens over 8-bit caches
        {"name": "tree_q8_draft", "op": "tree", "cache": "q8", "seqs": 3, "longest": 9001, "tokens": 25, "heads": 12,
         "kv_heads": 4, "width": 96},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "kv", "tree", "tree", "tree"))
    heads, kv_heads, width = rng.choice(HEADS)
    if op == "prompt":
        seqs = _log(rng, 1, 24)
        most = math.isqrt(2 * 8191 * 8191 * 32 * 128 // (seqs * heads * width))
        return {"op": op, "type": rng.choice(("f32", "f16")), "seqs": seqs,
                "longest": _log(rng, 1, min(8191, most // 2)), "heads": heads, "kv_heads": kv_heads, "width": width}
    if op == "kv":
        seqs = _log(rng, 1, 24)
        most = 4 * 8191 * 1024 // (seqs * kv_heads * width)
        return {"op": op, "mode": rng.choice(("write", "read")), "type": rng.choice(("f32", "f16")), "seqs": seqs,
                "longest": _log(rng, 1, min(32767, most)), "kv_heads": kv_heads, "width": width}
    seqs, tokens = _log(rng, 1, 24), rng.choice((1, 1, rng.randint(2, 16), rng.randint(2, 64)))
    most = min(8 * 32767 * 1024 // (seqs * kv_heads * width),
               8 * 16385 * 64 * 4096 // (seqs * tokens * heads * width))
    return {"op": op, "cache": rng.choice(("f16", "q8")), "seqs": seqs, "longest": _log(rng, 1, min(32767, most)),
            "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "width": width}


def _lengths(case):
    """Lengths of the sequences: the longest, and others between an eighth of it and all of it."""
    rng = random.Random(case["seqs"] * 100003 + case["longest"])
    return [case["longest"]] + [max(1, int(case["longest"] * rng.uniform(0.125, 1.0)))
                                for _ in range(case["seqs"] - 1)]


def _tokens(case):
    """Drafted tokens of the sequences: the widest tree, and others of at least half of it."""
    rng = random.Random(case["seqs"] * 100019 + case["tokens"])
    return [case["tokens"]] + [rng.randint((case["tokens"] + 1) // 2, case["tokens"])
                               for _ in range(case["seqs"] - 1)]


def _ancestors(rng, n):
    """Bit j of word i: drafted token i attends to drafted token j (itself and its ancestors in a random tree)."""
    words = []
    for i in range(n):
        parent = int(rng.integers(-1, i)) if i else -1
        words.append((words[parent] if parent >= 0 else 0) | (1 << i))
    return np.array(words, np.uint64).view(np.int64)


def _sizes(values):
    return (C.c_size_t * len(values))(*values)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, sigma=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * sigma

    n = _lengths(case)
    # the calls go behind what the program's stream makes of their inputs (its default stream is 0, the library's own
    # to these calls: such a program waits for its inputs first)
    s = {"case": case, "lens": n, "sizes": _sizes(n), "stream": torch.cuda.current_stream().cuda_stream or None}
    kvw = case["kv_heads"] * case["width"]
    if case["op"] == "prompt":
        total, qw = sum(n), case["heads"] * case["width"]
        if case["type"] == "f16":  # the fused projections' rows: q | k | v
            rows = torch.cat([normal(total, qw, sigma=1.5), normal(total, 2 * kvw)], 1).half()
            s["q"], s["k"], s["v"] = rows[:, :qw], rows[:, qw:qw + kvw], rows[:, qw + kvw:]
        else:
            s["q"], s["k"], s["v"] = normal(total, qw, sigma=1.5), normal(total, kvw).half(), normal(total, kvw).half()
        s["out"] = torch.empty(total, qw, device="cuda", dtype=s["q"].dtype)
        return s
    draft = _tokens(case) if case["op"] == "tree" else [0] * len(n)
    # one pool of caches, a sequence's rows behind one another in its own part of it
    rows = max(a + b for a, b in zip(n, draft)) + 5
    if case.get("cache") == "f16":
        s["k"], s["v"] = normal(case["seqs"], rows, kvw).half(), normal(case["seqs"], rows, kvw).half()
    else:
        s["k"], s["v"] = (torch.randint(-127, 128, (case["seqs"], rows, kvw), device="cuda", generator=g,
                                        dtype=torch.int8) for _ in "kv")
        s["ks"], s["vs"] = (0.002 + 0.024 * torch.rand(case["seqs"], rows, case["kv_heads"], device="cuda",
                                                      generator=g) for _ in "kv")
    if case["op"] == "tree":
        rng = np.random.default_rng(seed)
        s["draft"], s["drafts"] = draft, _sizes(draft)
        s["q"] = normal(sum(draft), case["heads"] * case["width"], sigma=1.5)
        s["mask"] = torch.from_numpy(np.concatenate([_ancestors(rng, t) for t in draft])).cuda()
        s["out"] = torch.empty_like(s["q"])
        return s
    s["first"] = [0 if case["longest"] > 1 else 3] * len(n)
    s["firsts"] = _sizes(s["first"])
    if case["mode"] == "write":  # the projections' rows: k | v
        s["src"] = normal(sum(n), 2 * kvw) * (0.25 + 4 * torch.rand(sum(n), 1, device="cuda", generator=g))
    t = torch.float32 if case["type"] == "f32" else torch.float16
    s["k_out"], s["v_out"] = (torch.empty(sum(n), kvw, device="cuda", dtype=t) for _ in "kv")
    return s


# ------------------------------------------------------------------ the library's calls
def _caches(P, s):
    """The sequences' caches, and the tree's workspace: what a serving program keeps from step to step."""
    if "caches" not in s:
        kv = (P.PranaKv * s["case"]["seqs"])()
        for i in range(len(kv)):
            kv[i].k, kv[i].v = s["k"][i].data_ptr(), s["v"][i].data_ptr()
            kv[i].rows = s["k"].shape[1]
            if "ks" in s:
                kv[i].k_scales, kv[i].v_scales = s["ks"][i].data_ptr(), s["vs"][i].data_ptr()
        s["caches"] = kv
        if s["case"]["op"] == "tree":
            c, need = s["case"], C.c_size_t()
            P.check(P.load().prana_attention_tree_workspace(s["sizes"], s["drafts"], c["seqs"], c["heads"],
                                                            c["kv_heads"], c["width"], C.byref(need)))
            s["work"] = torch.empty(max(1, need.value), device="cuda", dtype=torch.uint8)
    return s["caches"]


def _own(s):
    import prana_amd as P

    P.init()
    c, lib = s["case"], P.load()
    if c["op"] == "prompt":
        q, k, v, out = s["q"], s["k"], s["v"], s["out"]
        P.check(lib.prana_attention_packed(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                           P.F32 if c["type"] == "f32" else P.F16, s["sizes"], c["seqs"], c["heads"],
                                           c["kv_heads"], c["width"], q.stride(0), k.stride(0), out.stride(0),
                                           out.data_ptr(), s["stream"]))
        return out
    kv = _caches(P, s)
    if c["op"] == "tree":
        P.check(lib.prana_attention_tree(s["q"].data_ptr(), P.KV_F16 if c["cache"] == "f16" else P.KV_Q8, kv,
                                         s["sizes"], s["drafts"], c["seqs"], s["mask"].data_ptr(), c["heads"],
                                         c["kv_heads"], c["width"], s["out"].data_ptr(), s["work"].data_ptr(),
                                         s["work"].numel(), s["stream"]))
        return s["out"]
    if c["mode"] == "write":
        src = s["src"]
        P.check(lib.prana_kv_write_q8(src.data_ptr(), src.data_ptr() + 2 * src.shape[1], src.shape[1], kv,
                                      s["firsts"], s["sizes"], c["seqs"], c["kv_heads"], c["width"], s["stream"]))
    P.check(lib.prana_kv_read_q8(kv, s["firsts"], s["sizes"], c["seqs"], c["kv_heads"], c["width"],
                                 P.F32 if c["type"] == "f32" else P.F16, s["k_out"].data_ptr(),
                                 s["v_out"].data_ptr(), s["k_out"].shape[1], s["stream"]))
    return s["k_out"], s["v_out"]


# ------------------------------------------------------------------ plain forms, in 32 bits
def _rows(lens, starts, device):
    """Index of row i of sequence s, [seqs, longest], and which of them exist."""
    lens, starts = torch.tensor(lens, device=device), torch.tensor(starts, device=device)
    at = torch.arange(int(max(lens.tolist())), device=device)
    there = at[None, :] < lens[:, None]
    return starts[:, None] + torch.minimum(at[None, :], lens[:, None] - 1), there


def _starts(lens):
    return [sum(lens[:i]) for i in range(len(lens))]


def _softmax_rows(scores, allowed):
    scores = scores.masked_fill(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return p / p.sum(-1, keepdim=True)


def _prompt(s):
    c = s["case"]
    h, kv, w = c["heads"], c["kv_heads"], c["width"]
    at, there = _rows(s["lens"], _starts(s["lens"]), s["q"].device)
    n, longest = at.shape
    q = s["q"][at].float().reshape(n, longest, kv, h // kv, w).permute(0, 2, 3, 1, 4)
    k = s["k"][at].float().reshape(n, longest, kv, 1, w).permute(0, 2, 3, 4, 1)
    v = s["v"][at].float().reshape(n, longest, kv, 1, w).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(n, kv, -1, w) @ k.reshape(n, kv, w, longest).contiguous()) / math.sqrt(w)
    i = torch.arange(longest, device=q.device)
    causal = i[None, :] <= i[:, None]
    p = _softmax_rows(scores.reshape(n, kv, h // kv, longest, longest), causal)
    o = p.reshape(n, kv, -1, longest) @ v.reshape(n, kv, longest, w).contiguous()
    o = o.reshape(n, kv, h // kv, longest, w).permute(0, 3, 1, 2, 4).reshape(n, longest, h * w)
    return o[there].to(s["q"].dtype)


def _kv(s):
    c = s["case"]
    heads, w, rows = c["kv_heads"], c["width"], s["k"].shape[1]
    at, there = _rows(s["lens"], [i * rows + f for i, f in enumerate(s["first"])], s["k"].device)
    at = at[there]  # the cache row of every packed row
    out = []
    for i, (values, scales) in enumerate((("k", "ks"), ("v", "vs"))):
        q, scale = s[values].view(-1, heads, w), s[scales].view(-1, heads)
        if c["mode"] == "write":
            x = s["src"][:, i * heads * w:(i + 1) * heads * w].reshape(-1, heads, w)
            amax = x.abs().amax(-1)
            # the quotient decides which way a value rounds: 64 bits
            t = x.double() * 127.0 / torch.where(amax > 0, amax, 1.0).double()[..., None]
            q[at] = (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8)
            scale[at] = torch.where(amax > 0, amax.double() / 127.0, 1.0).float()
        y = q[at].float() * scale[at][..., None]
        out.append(y.reshape(-1, heads * w).to(s[values + "_out"].dtype))
    return tuple(out)


def _tree(s):
    c = s["case"]
    h, kv, w = c["heads"], c["kv_heads"], c["width"]
    at, there = _rows(s["draft"], _starts(s["draft"]), s["q"].device)
    n, tokens = at.shape
    k, v = s["k"].float(), s["v"].float()
    keys = k.shape[1]
    if c["cache"] == "q8":
        k = k.reshape(n, keys, kv, w) * s["ks"][..., None]
        v = v.reshape(n, keys, kv, w) * s["vs"][..., None]
    q = s["q"][at].reshape(n, tokens, kv, h // kv, w).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, w)
    k = k.reshape(n, keys, kv, w).permute(0, 2, 3, 1).contiguous()
    v = v.reshape(n, keys, kv, w).permute(0, 2, 1, 3).contiguous()
    scores = (q @ k) / math.sqrt(w)
    drafted = torch.arange(keys, device=k.device)[None, :] - torch.tensor(s["lens"], device=k.device)[:, None]
    bit = (s["mask"][at][:, :, None] >> drafted[:, None, :].clamp(0, 63)) & 1
    allowed = (drafted[:, None, :] < 0) | ((drafted[:, None, :] < 64) & (bit == 1))
    p = _softmax_rows(scores.reshape(n, kv, h // kv, tokens, keys), allowed[:, None, None])
    o = (p.reshape(n, kv, -1, keys) @ v).reshape(n, kv, h // kv, tokens, w)
    return o.permute(0, 3, 1, 2, 4).reshape(n, tokens, h * w)[there]


def run(state):
    if own:
        return _own(state)
    return {"prompt": _prompt, "kv": _kv, "tree": _tree}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n, kvw = _lengths(case), case["kv_heads"] * case["width"]
    size = 4 if case.get("type") == "f32" else 2
    if case["op"] == "kv":
        rows = sum(n)
        cache = kvw + 4 * case["kv_heads"]
        write = case["mode"] == "write"
        return {"bytes": 2 * rows * ((4 * kvw + cache if write else 0) + cache + size * kvw),
                "flops": 2 * rows * kvw * (3 if write else 1)}
    qw = case["heads"] * case["width"]
    if case["op"] == "prompt":
        return {"bytes": sum(n) * (2 * size * qw + 4 * kvw), "flops": sum(2 * qw * a * (a + 1) for a in n)}
    draft = _tokens(case)
    row = 4 * kvw if case["cache"] == "f16" else 2 * (kvw + 4 * case["kv_heads"])
    # a drafted token sees the cache and its ancestors, about the logarithm of the tree's size
    return {"bytes": sum((a + t) * row + 8 * t * qw for a, t in zip(n, draft)),
            "flops": sum(4 * qw * t * (a + 1 + math.log(t)) for a, t in zip(n, draft))}


# ------------------------------------------------------------------ in 64 bits
def _attend(q, k, v, seen):
    """One head: rows of q over rows of k and v, where `seen` says which row sees which."""
    out = torch.empty(q.shape[0], v.shape[1], device=q.device, dtype=torch.float64)
    for i in range(0, q.shape[0], 2048):
        s = torch.mm(q[i:i + 2048].double(), k.double().t().contiguous()) / math.sqrt(q.shape[1])
        s[~seen(i, min(q.shape[0], i + 2048))] = -math.inf
        out[i:i + 2048] = torch.mm(torch.softmax(s, -1), v.double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kvh, w = case["kv_heads"], case["width"]
    lens = s["lens"]
    if case["op"] == "kv":
        out = []
        for i, (values, scales) in enumerate((("k", "ks"), ("v", "vs"))):
            if case["mode"] == "write":
                x = s["src"].double()[:, i * kvh * w:(i + 1) * kvh * w].reshape(-1, kvh, w)
                step = x.abs().amax(-1, keepdim=True) / 127
                y = torch.sign(x) * torch.floor(x.abs() / step + 0.5) * step
            else:
                y = torch.cat([s[values][j, f:f + n].double().reshape(n, kvh, w) * s[scales][j, f:f + n, :, None]
                               for j, (f, n) in enumerate(zip(s["first"], lens))])
            out.append(y.reshape(-1, kvh * w))
        return tuple(out)
    heads = case["heads"]
    group, out = heads // kvh, torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    at = 0
    for j, n in enumerate(lens):
        m = n if case["op"] == "prompt" else s["draft"][j]
        if case["op"] == "prompt":
            k, v = s["k"][at:at + n], s["v"][at:at + n]

            def seen(a, b, n=n):
                return torch.ones(b - a, n, device="cuda", dtype=torch.bool).tril(a)
        else:
            k, v = s["k"][j, :n + m].double(), s["v"][j, :n + m].double()
            if case["cache"] == "q8":
                k = (k.reshape(-1, kvh, w) * s["ks"][j, :n + m, :, None].double()).reshape(n + m, -1)
                v = (v.reshape(-1, kvh, w) * s["vs"][j, :n + m, :, None].double()).reshape(n + m, -1)
            words = s["mask"][at:at + m].cpu().numpy().view(np.uint64)
            tree = torch.tensor([[bool(int(word) >> b & 1) for b in range(m)] for word in words], device="cuda")
            full = torch.cat([torch.ones(m, n, device="cuda", dtype=torch.bool), tree], 1)

            def seen(a, b, full=full):
                return full[a:b]
        for hd in range(heads):
            c = hd // group
            out[at:at + m, hd * w:(hd + 1) * w] = _attend(s["q"][at:at + m, hd * w:(hd + 1) * w],
                                                          k[:, c * w:(c + 1) * w], v[:, c * w:(c + 1) * w], seen)
        at += m
    return out
