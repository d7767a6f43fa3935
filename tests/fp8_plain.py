"""Plain 64-bit forms of the operators on a paged cache of 8-bit codes, written
from their contracts."""

import math

import numpy as np

from nkipy_amd.core import dtypes as dt

import serving_plain as P

TABLE = dt.E4M3FN_VALUES.astype(np.float64)


def bits(codes):
    return np.ascontiguousarray(codes).view(np.uint8)


def values(codes, exps):
    """codes (..., heads, dim), exps (..., heads); or whole caches, with exps
    (pages, heads)."""
    scale = 2.0 ** np.clip(exps, -120, 120).astype(np.float64)[..., None]
    return TABLE[bits(codes)] * (scale[:, None] if codes.ndim == 4 else scale)


def nearest(y):
    """float64 values in the codes' range rounded to the table's, ties to even."""
    t = TABLE[:127]
    i = np.clip(np.searchsorted(t, np.abs(y)), 1, 126)
    lo, hi = t[i - 1], t[i]
    mid = (lo + hi) / 2
    up = (np.abs(y) > mid) | ((np.abs(y) == mid) & (i % 2 == 0))
    return np.where(np.abs(y) >= t[126], np.sign(y) * t[126], np.sign(y) * np.where(up, hi, lo))


def random_cache(rng, pages, page, hkv, d, lo=-9, hi=-4):
    """Random codes (NaN ones left out) and exponents."""
    codes = rng.integers(0, 127, (pages, page, hkv, d)).astype(np.uint8) | (rng.integers(0, 2, (pages, page, hkv, d)) << 7).astype(np.uint8)
    return codes.view(dt.float8_e4m3fn), rng.integers(lo, hi, (pages, hkv)).astype(np.int32)


def least_exponent(y):
    top = np.abs(y[np.isfinite(y)]).max(initial=0.0)
    e = -120
    while top > 448 * 2.0**e:
        e += 1
    return e


def append(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts, t):
    """(rotated q, its tolerance), then for keys and values (exponents, values,
    tolerances, which of them are written now), values of what is not written
    by this call being those of the codes there under the new exponents."""
    half, page, n = cos.shape[1], kc.shape[1], q.shape[0]

    def turn(x, p):
        x = P.up(x)
        c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
        a, z = x[:, :half], x[:, half:2 * half]
        y = np.concatenate([a * c - z * s, a * s + z * c, x[:, 2 * half:]], 1)
        size = np.concatenate([abs(a * c) + abs(z * s), abs(a * s) + abs(z * c), 0 * x[:, 2 * half:]], 1)
        return y, 2.0**-22 * size  # two products and their sum in 32 bits

    rq, tq = np.zeros(q.shape), np.zeros(q.shape)
    out = [(e.copy().astype(np.int64), values(c, e), np.zeros(c.shape), np.zeros(c.shape, bool)) for c, e in ((kc, ke), (vc, ve))]
    rows = {}
    for b, lo, m, length in P.sequences(tables, lens, starts, n):
        for i in range(m):
            p, at = length - m + i, lo + i
            if not 0 <= p < cos.shape[0]:
                continue
            y, off = turn(q[at], p)
            rq[at], tq[at] = y, P.HALF_STEP[t] * np.abs(y) * (off > 0) + off + ({"f16": 2.0**-24}.get(t, 0) if half else 0)
            pg = tables[b, p // page] if p // page < tables.shape[1] else -1
            if 0 <= pg < kc.shape[0]:
                rows.setdefault(int(pg), []).append((p % page, turn(k[at], p), (P.up(v[at]), 0 * P.up(v[at]))))
    for pg, new in rows.items():
        for which, (codes, exps) in enumerate(((kc, ke), (vc, ve))):
            e_out, val, tol, wrote = out[which]
            x = np.stack([r[1 + which][0] for r in new])
            off = np.stack([r[1 + which][1] for r in new])
            first = new[0][0]
            for h in range(x.shape[1]):
                old = int(np.clip(exps[pg, h], -120, 120))
                e = least_exponent(x[:, h])
                if first:
                    e = max(e, old)
                val[pg, :, h] = TABLE[bits(codes[pg, :, h])] * 2.0**e
                if first:
                    had = TABLE[bits(codes[pg, :first, h])]
                    val[pg, :first, h] = nearest(np.where(np.isnan(had), 0, had) * 2.0 ** (old - e)) * 2.0**e + had * 0
                e_out[pg, h] = e
                for i, r in enumerate(new):
                    y = np.where(np.isfinite(x[i, h]), x[i, h], np.nan)
                    val[pg, r[0], h], wrote[pg, r[0], h] = y, True
                    # half a step of the code: 2^-4 of it, or of the subnormal ones 2^-10
                    tol[pg, r[0], h] = np.maximum(np.abs(y) * 2.0**-4, 2.0 ** (e - 10)) + off[i, h]
    return (rq, tq), out


def paged(q, kc, vc, ke, ve, tables, lens, starts, window, sinks, t, scale=None):
    """(result, tolerance) of paged_attention_fp8."""
    n, _, d = q.shape
    pages, page = kc.shape[:2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b, lo, m, length in P.sequences(tables, lens, starts, n):
        keys = np.arange(min(length, tables.shape[1] * page))
        at = tables[b][keys // page]
        ok = (at >= 0) & (at < pages)
        keys, at = keys[ok], at[ok]
        seen = P.see(np.arange(length - m, length), keys, length, window, sinks)
        o, mag, big = P.masked_attention(P.up(q[lo:lo + m]), values(kc[at, keys % page], ke[at]), values(vc[at, keys % page], ve[at]),
                                         seen, 1 / math.sqrt(d) if scale is None else scale)
        out[lo:lo + m], tol[lo:lo + m] = o, P.tolerance(o, mag, big, len(keys), d, t)
    if t == "f16":
        # 65520 and above round to infinity; what is that within the tolerance may be either
        over = np.abs(out) - tol >= 65520
        tol = np.where(~over & (np.abs(out) + tol >= 65520), np.inf, tol)
        out = np.where(over, np.copysign(np.inf, out), out)
    return out, tol
