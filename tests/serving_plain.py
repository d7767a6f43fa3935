"""Plain 64-bit forms of the serving operators, written from their contracts
(masks as whole matrices, one softmax per head), and the cases their tests
share."""

import math

import numpy as np

from nkipy_amd.core import dtypes as dt

HALF_STEP = {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 2.0**-24}
NP = {"bf16": dt.bfloat16, "f16": dt.float16, "f32": dt.float32}


def cast(x, t):
    return dt.to_bf16(x) if t == "bf16" else np.asarray(x, np.float32).astype(NP[t])


def up(x):
    return dt.to_float32(x).astype(np.float64)


def masked_attention(q, k, v, seen, scale):
    """(result, mean |v| under the weights, largest scale sum |q k|) of q (n, Hq, D),
    k / v (m, Hkv, D) under the mask seen (n, m); rows that see nothing are 0."""
    n, hq, d = q.shape
    rep = hq // k.shape[1]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    big = 0.0
    if k.shape[0] == 0 or n == 0:
        return out, mag, big
    for h in range(hq):
        kk, vv = k[:, h // rep], v[:, h // rep]
        used = seen.any(0)
        kk, vv = np.where(used[:, None], kk, 0), np.where(used[:, None], vv, 0)
        s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
        top = s.max(1, keepdims=True)
        w = np.exp(s - np.where(np.isfinite(top), top, 0))
        total = w.sum(1, keepdims=True)
        w = w / np.where(total > 0, total, 1)
        out[:, h], mag[:, h] = w @ vv, w @ np.abs(vv)
        big = max(big, float((np.abs(q[:, h]) @ np.abs(kk).T * scale).max()))
    return out, mag, big


def tolerance(o, mag, big, keys, d, t):
    """A result is rounded once (half a step), each weight once where the
    operands have 16 bits, and sums of keys and products lose at most a 32-bit
    half step per term; a subnormal result loses the type's last place."""
    h = HALF_STEP[t]
    tiny = {"bf16": 2.0**-133, "f16": 2.0**-24, "f32": 2.0**-149}[t]
    return h * np.abs(o) + mag * ((h if t != "f32" else 0) + (keys + d + 16) * 2.0**-24 * (1 + big)) + tiny


def see(p, keys, length, window, sinks):
    p, j = np.asarray(p)[:, None], np.asarray(keys)[None, :]
    m = (j <= p) & (p < length) & (j < length)
    if window:
        m &= (p - j < window) | (j < sinks)
    return m


def sequences(tables, lens, starts, n):
    for b in range(len(lens)):
        lo, hi = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        yield b, lo, hi - lo, lens[b]


def paged(q, kc, vc, tables, lens, starts, window, sinks, t, scale=None):
    """(result, tolerance) of paged_attention."""
    n, _, d = q.shape
    pages, page = kc.shape[:2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b, lo, m, length in sequences(tables, lens, starts, n):
        keys = np.arange(min(length, tables.shape[1] * page))
        at = tables[b][keys // page]
        ok = (at >= 0) & (at < pages)
        keys, at = keys[ok], at[ok]
        seen = see(np.arange(length - m, length), keys, length, window, sinks)
        o, mag, big = masked_attention(up(q[lo:lo + m]), up(kc[at, keys % page]), up(vc[at, keys % page]), seen,
                                       1 / math.sqrt(d) if scale is None else scale)
        out[lo:lo + m], tol[lo:lo + m] = o, tolerance(o, mag, big, len(keys), d, t)
    return out, tol


def dense(q, k, v, lengths, positions, window, sinks, t, scale=None):
    """(result, tolerance) of window_attention."""
    (B, S, _, d), T = q.shape, k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        length = T if lengths is None else min(max(lengths[b], 0), T)
        p = np.arange(S) + (T - S if positions is None else positions[b])
        seen = see(p, np.arange(T), length, window, sinks)
        o, mag, big = masked_attention(up(q[b]), up(k[b]), up(v[b]), seen, 1 / math.sqrt(d) if scale is None else scale)
        out[b], tol[b] = o, tolerance(o, mag, big, T, d, t)
    return out, tol


def append(q, k, v, cos, sin, kc, vc, tables, lens, starts, t):
    """Results and tolerances of rotary_append: (q, k cache, v cache), all
    float64; elements nobody writes have tolerance 0."""
    half = cos.shape[1]
    page = kc.shape[1]

    def turn(x, p):
        x = up(x)
        c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
        a, z = x[:, :half], x[:, half:2 * half]
        y = np.concatenate([a * c - z * s, a * s + z * c, x[:, 2 * half:]], 1)
        size = np.concatenate([abs(a * c) + abs(z * s), abs(a * s) + abs(z * c), 0 * x[:, 2 * half:]], 1)
        # two products and their sum in 32 bits, then the storage type (its
        # last place where the result is subnormal)
        h = HALF_STEP[t]
        return y, np.where(size > 0, h * abs(y) + 2.0**-22 * size + {"f16": 2.0**-24}.get(t, 0), 0)

    res, tol = [np.zeros(q.shape), up(kc), up(vc)], [np.zeros(q.shape), np.zeros(kc.shape), np.zeros(vc.shape)]
    for b, lo, m, length in sequences(tables, lens, starts, q.shape[0]):
        for i in range(m):
            p, at = length - m + i, lo + i
            if not 0 <= p < cos.shape[0]:
                continue
            res[0][at], tol[0][at] = turn(q[at], p)
            pg = tables[b, p // page] if p // page < tables.shape[1] else -1
            if 0 <= pg < kc.shape[0]:
                res[1][pg, p % page], tol[1][pg, p % page] = turn(k[at], p)
                res[2][pg, p % page] = up(v[at])
    return res, tol


def kept(x, temperature, top_k, top_p, min_p):
    """(kept tokens in vocabulary order, their weights) of one row of logits."""
    z = np.where(np.isnan(x), -np.inf, x)
    order = sorted(range(len(z)), key=lambda i: (-z[i], i))
    w = np.array([1.0 if z[i] == z[order[0]] else math.exp((z[i] - z[order[0]]) / temperature) if z[i] > -np.inf else 0.0
                  for i in order])
    n = len(w) if not top_k or top_k < 0 else min(top_k, len(w))
    if top_p is not None and top_p < 1:
        run, goal = np.cumsum(w[:n]), top_p * w[:n].sum()
        n = int(np.argmax(run >= goal)) + 1
    ids = [i for i, m in zip(order[:n], w) if m > 0 and m >= (min_p or 0)]
    weight = {i: m for i, m in zip(order, w)}
    ids.sort()
    return np.array(ids), np.array([weight[i] for i in ids])


def batch(rng, lens, new, page, extra=2, width=0):
    """A block table of shuffled pages for sequences of these lengths."""
    need = [-(-max(n, 0) // page) for n in lens]
    width = max(need + [1, width])
    ids = rng.permutation(sum(need) + extra)
    tables, at = np.full((len(lens), width), -1, np.int32), 0
    for b, n in enumerate(need):
        tables[b, :n] = ids[at:at + n]
        at += n
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return tables, np.asarray(lens, np.int32), starts, len(ids)
