"""The attention layer over a paged cache in 64 bits, with a bound on what 32-bit
sums and a storage type's roundings may make of it."""

import numpy as np

import serving_plain as P

U = 2.0**-24


def layer(x, w, qn, kn, eps, hq, hkv, dim, cos, sin, kc, vc, tables, lens, starts, wo, window, sinks, half_step):
    """((result, k cache, v cache), their bounds).  Each stage's error bound is that
    of its input passed on, its sums' roundings (U a term) and its own rounding."""
    x, w, qn, kn, wo, kc, vc = (np.asarray(P.up(a), np.float64) for a in (x, w, qn, kn, wo, kc, vc))
    n, half = len(x), cos.shape[1]
    kc, vc = kc.copy(), vc.copy()
    kt, vt = np.zeros_like(kc), np.zeros_like(vc)
    qkv = x @ w
    e = (x.shape[1] + 1) * U * (np.abs(x) @ np.abs(w)) + half_step * np.abs(qkv)
    cut = [hq * dim, (hq + hkv) * dim]
    parts = [a.reshape(n, -1, dim) for a in np.split(qkv, cut, axis=1)]
    errs = [a.reshape(n, -1, dim) for a in np.split(e, cut, axis=1)]
    page, width = kc.shape[1], tables.shape[1]
    starts = np.arange(len(lens) + 1) if starts is None else starts

    def norm(y, d, g):
        rms = np.sqrt((y * y).mean(-1, keepdims=True) + eps)
        out = y / rms * g
        d = np.abs(g) / rms * (d + np.abs(y) / rms * d.max(-1, keepdims=True))
        return out, d + ((dim + 8) * U + 2 * half_step) * np.abs(out)  # (normalised, then weighed)

    def turn(y, d, p):
        a, b = y[:, :, :half], y[:, :, half:2 * half]
        c, s = cos[p][:, None].astype(np.float64), sin[p][:, None].astype(np.float64)
        out = np.concatenate([a * c - b * s, a * s + b * c], axis=-1)
        d = np.abs(np.concatenate([d[:, :, :half] + d[:, :, half:]] * 2, axis=-1))
        return out, d + 4 * U * np.abs(np.concatenate([y, y], -1)).max(-1, keepdims=True) + half_step * np.abs(out)

    q, qe = norm(parts[0], errs[0], qn)
    k, ke = norm(parts[1], errs[1], kn)
    v, ve = parts[2], errs[2]
    pos = np.zeros(n, int)
    for b in range(len(lens)):
        for i in range(starts[b], starts[b + 1]):
            pos[i] = lens[b] - (starts[b + 1] - starts[b]) + i - starts[b]
    q, qe = turn(q, qe, pos)
    k, ke = turn(k, ke, pos)
    for b in range(len(lens)):
        for i in range(starts[b], starts[b + 1]):
            at = tables[b, pos[i] // page], pos[i] % page
            kc[at], vc[at], kt[at], vt[at] = k[i], v[i], ke[i], ve[i]
    o, oe = np.zeros((n, hq, dim)), np.zeros((n, hq, dim))
    for b in range(len(lens)):
        rows = tables[b, np.arange(width * page) // page], np.arange(width * page) % page
        for i in range(starts[b], starts[b + 1]):
            j = np.arange(pos[i] + 1)
            if window:
                j = j[(pos[i] - j < window) | (j < sinks)]
            at = rows[0][j], rows[1][j]
            for h in range(hq):
                g = h // (hq // hkv)
                keys, vals, kd, vd = kc[at][:, g], vc[at][:, g], kt[at][:, g], vt[at][:, g]
                s = keys @ q[i, h] / np.sqrt(dim)
                ds = (np.abs(keys) @ qe[i, h] + kd @ np.abs(q[i, h]) + (dim + 2) * U * (np.abs(keys) @ np.abs(q[i, h])))
                p = np.exp(s - s.max())
                p /= p.sum()
                o[i, h] = p @ vals
                share = np.expm1(2 * (ds / np.sqrt(dim)).max()) + (len(j) + 12) * U + 2 * half_step
                oe[i, h] = vd.max(0) + share * np.abs(vals).max(0) + half_step * np.abs(o[i, h])
    o, oe = o.reshape(n, -1), oe.reshape(n, -1)
    out = o @ wo
    tol = oe @ np.abs(wo) + (len(wo) + 2) * U * (np.abs(o) @ np.abs(wo)) + half_step * np.abs(out)
    return (out, kc, vc), (tol + half_step * tol, kt, vt)


def case(rng, t, lens, new, hidden, hq, hkv, dim, page, q_weight=1.0):
    """Operands of a call: the cached beginnings of the sequences at random.  A small
    q_weight keeps the scores, and with them the bound on the softmax, small."""
    tables, lens, starts, pages = P.batch(rng, lens, new, page)
    n = int(starts[-1]) if starts is not None else len(lens)
    g = lambda *s, std=1.0: P.cast(rng.standard_normal(s) * std, t)  # noqa: E731
    return dict(x=g(n, hidden), w=g(hidden, (hq + 2 * hkv) * dim, std=hidden**-0.5),
                qn=P.cast(rng.uniform(0.5, 1.0, dim) * q_weight, t), kn=P.cast(rng.uniform(0.5, 1.0, dim), t),
                kc=g(pages, page, hkv, dim), vc=g(pages, page, hkv, dim), tables=tables, lens=lens, starts=starts,
                wo=g(hq * dim, hidden, std=(hq * dim)**-0.5))
