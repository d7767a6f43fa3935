"""Operators of a serving step: a paged key / value cache, attention over it
and over plain tensors with a sliding window, and the draw of the next token.

A paged cache is two arrays of shape (pages, page_size, n_kv_heads, head_dim).
Row b of ``block_tables`` (sequences, width) lists the pages of sequence b in
order; an entry outside 0 .. pages-1 is no page (-1 by custom).
``context_lens`` (sequences,) counts the tokens of a sequence, its new ones
included.  The new tokens of all sequences are packed along the first axis of
q / k / v; ``query_starts`` (sequences + 1,), not decreasing, says where each
sequence's begin, and is left out where every sequence has exactly one.  New
token i of n of a sequence of length L sits at position p = L - n + i.

Which keys the query at position p sees (the same in both attentions):

    0 <= j <= p,  j below the sequence's length,  j's page a page of the cache,
    and with a window W also   p - j < W  or  j < sinks

A query that sees no key, or only scores of -inf, gives zeros; so do rows of
the packed batch outside every sequence.  What a query does not see has no
part in its result, NaN and infinities included; a value that is not finite
reaches every query that sees its key with a score above -inf, however small
the weight.

The CPU forms are the definitions, evaluated in float64 and rounded once.  On
the GPU scores and weighted values are 32-bit sums: a row that sees a score past
their range is NaN.  Operands of 16 bits with a head_dim of 64 or 128 have their
weights rounded to the operands' type before the values are summed, which adds
up to half a step of that type to the result's own.
"""

from __future__ import annotations

import math

import numpy as np

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core.ops._registry import Op

MAX_HEAD_DIM = 256
_FLOATS = (dt.bfloat16, dt.float16, dt.float32)


# ---------------------------------------------------------------------------
# Checks shared by the traced and the CPU forms
# ---------------------------------------------------------------------------
def _shape(x, name, ndim):
    shape = getattr(x, "shape", None)
    if shape is None or len(shape) != ndim:
        raise ValueError(f"{name} must be an array of {ndim} dimensions, got "
                         f"{'a ' + type(x).__name__ if shape is None else 'shape ' + str(tuple(shape))}")
    return tuple(int(s) for s in shape)


def _float(x, name, types=_FLOATS):
    d = dt.canonical(x.dtype)
    if d == dt.float64:  # narrowed to 32 bits when traced, as every argument is
        d = dt.float32
    if d not in types:
        raise TypeError(f"{name} must be of {' / '.join(dt.name(t) for t in types)}, got {dt.name(x.dtype)}")
    return d


def _ints(x, name, shape):
    if _shape(x, name, len(shape)) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if not dt.is_int(x.dtype):
        raise TypeError(f"{name} must hold integers, got {dt.name(x.dtype)}")


def _same(named):
    kinds = {n: _float(x, n) for n, x in named.items()}
    if len(set(kinds.values())) != 1:
        raise TypeError("operands must share one type, got " + ", ".join(f"{n} {dt.name(d)}" for n, d in kinds.items()))
    return next(iter(kinds.values()))


def _heads(hq, hkv, dim):
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads are no multiple of {hkv} key / value heads")
    if not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in 1..{MAX_HEAD_DIM}, got {dim}")


def _tables(n, key_cache, value_cache, block_tables, context_lens, query_starts):
    """(pages, page size, kv heads, head dim, sequences) of a paged call of n tokens."""
    pages, page, hkv, dim = _shape(key_cache, "key_cache", 4)
    if _shape(value_cache, "value_cache", 4) != (pages, page, hkv, dim):
        raise ValueError(f"value_cache must have key_cache's shape {(pages, page, hkv, dim)}, got {tuple(value_cache.shape)}")
    if pages < 1 or page < 1:
        raise ValueError("the cache holds no page")
    seqs, width = _shape(block_tables, "block_tables", 2)
    if seqs < 1 or width < 1:
        raise ValueError(f"block_tables of shape {(seqs, width)} name no page")
    _ints(block_tables, "block_tables", (seqs, width))
    _ints(context_lens, "context_lens", (seqs,))
    if query_starts is not None:
        _ints(query_starts, "query_starts", (seqs + 1,))
    elif n != seqs:
        raise ValueError(f"without query_starts every sequence has one new token: got {n} tokens of {seqs} sequences")
    if width * page >= 2**30 or pages * page >= 2**31:
        raise ValueError("block_tables or cache too large: positions and cache rows are 32-bit")
    return pages, page, hkv, dim, seqs


def _window(window, sinks):
    if window is not None:
        if isinstance(window, bool) or not isinstance(window, (int, np.integer)) or window < 1:
            raise ValueError(f"window must be None or a whole number from 1, got {window!r}")
        window = min(int(window), 2**30)
    if isinstance(sinks, bool) or not isinstance(sinks, (int, np.integer)) or sinks < 0:
        raise ValueError(f"sinks must be a whole number from 0, got {sinks!r}")
    if sinks and window is None:
        raise ValueError("sinks stay visible behind a window: give one")
    return window, min(int(sinks), 2**30)


def _scale(scale, dim):
    if scale is None:
        return 1.0 / math.sqrt(dim)
    scale = float(scale)
    if not 2.0**-64 <= scale <= 2.0**64:
        raise ValueError(f"scale must be a positive number, of 2^-64 to 2^64, got {scale}")
    return scale


def _check_append(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts):
    n, hq, dim = _shape(q, "q", 3)
    pages, page, hkv, cdim, seqs = _tables(n, key_cache, value_cache, block_tables, context_lens, query_starts)
    for x, name in ((k, "k"), (v, "v")):
        if _shape(x, name, 3) != (n, hkv, cdim):
            raise ValueError(f"{name} must have shape {(n, hkv, cdim)}, got {tuple(x.shape)}")
    if dim != cdim:
        raise ValueError(f"q has head_dim {dim}, the cache {cdim}")
    _heads(hq, hkv, dim)
    _same({"q": q, "k": k, "v": v, "key_cache": key_cache, "value_cache": value_cache})
    positions, half = _shape(cos, "cos", 2)
    if _shape(sin, "sin", 2) != (positions, half):
        raise ValueError(f"sin must have cos's shape {(positions, half)}, got {tuple(sin.shape)}")
    if not 1 <= half <= dim // 2 or positions < 1:
        raise ValueError(f"cos / sin of shape {(positions, half)} do not fit head_dim {dim}: (positions, up to head_dim / 2)")
    for x, name in ((cos, "cos"), (sin, "sin")):
        _float(x, name, (dt.float32,))


def _check_paged(q, key_cache, value_cache, block_tables, context_lens, query_starts, window, sinks, scale):
    n, hq, dim = _shape(q, "q", 3)
    pages, page, hkv, cdim, seqs = _tables(n, key_cache, value_cache, block_tables, context_lens, query_starts)
    if dim != cdim:
        raise ValueError(f"q has head_dim {dim}, the cache {cdim}")
    _heads(hq, hkv, dim)
    _same({"q": q, "key_cache": key_cache, "value_cache": value_cache})
    return _window(window, sinks) + (_scale(scale, dim),)


def _check_window(q, k, v, lengths, positions, window, sinks, scale):
    b, s, hq, dim = _shape(q, "q", 4)
    kb, t, hkv, kdim = _shape(k, "k", 4)
    if kb != b or kdim != dim:
        raise ValueError(f"k of shape {(kb, t, hkv, kdim)} does not fit q of shape {(b, s, hq, dim)}")
    if _shape(v, "v", 4) != (kb, t, hkv, kdim):
        raise ValueError(f"v must have k's shape {(kb, t, hkv, kdim)}, got {tuple(v.shape)}")
    _heads(hq, hkv, dim)
    _same({"q": q, "k": k, "v": v})
    for x, name in ((lengths, "lengths"), (positions, "positions")):
        if x is not None:
            _ints(x, name, (b,))
    if t >= 2**30 or s >= 2**30:
        raise ValueError("sequences too long: positions are 32-bit")
    return _window(window, sinks) + (_scale(scale, dim),)


def _row_values(x, name, rows, whole=False):
    """A filter of sample: a number, or an array of one value per row."""
    if hasattr(x, "shape") and tuple(x.shape) != ():
        if tuple(x.shape) != (rows,):
            raise ValueError(f"{name} must be a number or an array of shape {(rows,)}, got {tuple(x.shape)}")
        if whole and not dt.is_int(x.dtype):
            raise TypeError(f"{name} must hold integers, got {dt.name(x.dtype)}")
        if not whole:
            _float(x, name, (dt.float32,))
        return x
    if hasattr(x, "backend_tensor"):
        raise ValueError(f"{name} must be a number or an array of shape {(rows,)}, got shape ()")
    x = x.item() if isinstance(x, (np.ndarray, np.generic)) else x
    if isinstance(x, bool) or not isinstance(x, int if whole else (int, float)):
        raise TypeError(f"{name} must be {'a whole number' if whole else 'a number'} or an array, got {x!r}")
    if whole:
        return max(-1, min(int(x), 2**31 - 1))
    x = float(x)
    if math.isnan(x) or x < 0 or (name != "temperature" and x > 1):
        raise ValueError(f"{name} must be {'at least 0' if name == 'temperature' else 'in 0..1'}, got {x}")
    return x


def _check_sample(logits, uniform, temperature, top_k, top_p, min_p):
    rows, vocab = _shape(logits, "logits", 2)
    if not 1 <= vocab < 2**31:
        raise ValueError(f"logits of shape {(rows, vocab)} hold no token to draw")
    if vocab > 2**22:
        raise ValueError(f"a vocabulary of {vocab} is too large: up to {2**22} tokens")
    _float(logits, "logits")
    if _shape(uniform, "uniform", 1) != (rows,):
        raise ValueError(f"uniform must have shape {(rows,)}, got {tuple(uniform.shape)}")
    _float(uniform, "uniform", (dt.float32,))
    return (rows, vocab, _row_values(temperature, "temperature", rows),
            None if top_k is None else _row_values(top_k, "top_k", rows, whole=True),
            None if top_p is None else _row_values(top_p, "top_p", rows),
            None if min_p is None else _row_values(min_p, "min_p", rows))


# ---------------------------------------------------------------------------
# Traced forms: one IR node per result
# ---------------------------------------------------------------------------
def _int_value(x):
    from nkipy_amd.core.ops._helpers import ctx
    from nkipy_amd.core.ops.indexing import _index_value

    return _index_value(ctx(), x)


_LAYOUT_OPS = ("slice", "reshape", "transpose", "broadcast_in_dim")
_WRITE_OPS = ("dynamic_update_slice", "scatter_along_axis", "put_along_axis", "scatter_strided", "paged_write")


def _part_of(v):
    """The argument that ``v`` is a part or another layout of, None for a whole
    argument and for an array that the kernel makes."""
    part = False
    while v.node is not None and v.node.op in _LAYOUT_OPS + _WRITE_OPS:  # (written into: the same argument)
        part = part or v.node.op in _LAYOUT_OPS
        v = v.node.inputs[0]
    return v if part and v.is_parameter else None


rotary_append = Op("rotary_append")


@rotary_append.impl("hip")
def _rotary_append_hip(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts=None):
    from nkipy_amd.core.ops._helpers import ctx, is_traced, val, wrap

    _check_append(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts)
    for c, name in ((key_cache, "key_cache"), (value_cache, "value_cache")):
        if not is_traced(c):
            raise TypeError(f"{name} is written in place: it must be an argument of the kernel or computed from one")
        whole = _part_of(val(c))
        if whole is not None:
            raise ValueError(f"{name} is a part or another layout of the argument {whole.name!r}, which a write into it would not "
                             "reach: pass each cache as an argument of its own")
    if key_cache is value_cache:
        raise ValueError("key_cache and value_cache are the same array")
    cx = ctx()
    where = [_int_value(block_tables), _int_value(context_lens)]
    starts = [] if query_starts is None else [_int_value(query_starts)]
    turn = [val(cos, dt.float32), val(sin, dt.float32)]
    qv, kv, vv, kc, vc = (val(x) for x in (q, k, v, key_cache, value_cache))
    rotated = cx.build_op("rotate_rows", [qv] + turn + where[1:] + starts, qv.shape, qv.dtype, {"starts": bool(starts)})
    for cache, cv, x, extra in ((key_cache, kc, kv, turn), (value_cache, vc, vv, [])):
        out = cx.build_op("paged_write", [cv, x] + extra + where + starts, cv.shape, cv.dtype,
                          {"rotary": bool(extra), "starts": bool(starts), "positions": int(cos.shape[0])})
        cache._is_mutated = True
        cache._rebind(wrap(out))
    return wrap(rotated)


paged_attention = Op("paged_attention")


@paged_attention.impl("hip")
def _paged_attention_hip(q, key_cache, value_cache, block_tables, context_lens, query_starts=None, *, window=None,
                         sinks=0, scale=None):
    from nkipy_amd.core.ops._helpers import ctx, val, wrap

    window, sinks, scale = _check_paged(q, key_cache, value_cache, block_tables, context_lens, query_starts, window,
                                        sinks, scale)
    ops = [val(q), val(key_cache), val(value_cache), _int_value(block_tables), _int_value(context_lens)]
    if query_starts is not None:
        ops.append(_int_value(query_starts))
    return wrap(ctx().build_op("paged_attention", ops, ops[0].shape, ops[0].dtype,
                               {"window": window or 0, "sinks": sinks, "scale": scale,
                                "starts": query_starts is not None}))


window_attention = Op("window_attention")


@window_attention.impl("hip")
def _window_attention_hip(q, k, v, lengths=None, positions=None, *, window=None, sinks=0, scale=None):
    from nkipy_amd.core.ops._helpers import ctx, val, wrap

    window, sinks, scale = _check_window(q, k, v, lengths, positions, window, sinks, scale)
    ops = [val(q), val(k), val(v)] + [_int_value(x) for x in (lengths, positions) if x is not None]
    return wrap(ctx().build_op("window_attention", ops, ops[0].shape, ops[0].dtype,
                               {"window": window or 0, "sinks": sinks, "scale": scale,
                                "lengths": lengths is not None, "positions": positions is not None}))


sample = Op("sample")


@sample.impl("hip")
def _sample_hip(logits, uniform, temperature=1.0, top_k=None, top_p=None, min_p=None):
    from nkipy_amd.core.ops._helpers import ctx, is_traced, val, wrap

    rows, vocab, temperature, top_k, top_p, min_p = _check_sample(logits, uniform, temperature, top_k, top_p, min_p)
    ops, given = [val(logits), val(uniform, dt.float32)], {}
    for name, x in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if x is None:
            continue
        if is_traced(x) or isinstance(x, np.ndarray):
            ops.append(_int_value(x) if name == "top_k" else val(x, dt.float32))
            given[name] = "rows"
        else:
            given[name] = x
    return wrap(ctx().build_op("sample", ops, (rows,), dt.int32, given))


# ---------------------------------------------------------------------------
# CPU forms
# ---------------------------------------------------------------------------
def _to64(x):
    return dt.to_float32(x).astype(np.float64) if np.asarray(x).dtype != np.float64 else np.asarray(x)


def _store(x, dtype):
    """float64 values rounded once to a storage type."""
    if dtype == dt.bfloat16:
        # float32 keeps 16 more bits than bfloat16; rounding it to odd first
        # makes the two steps one rounding
        with np.errstate(over="ignore", invalid="ignore"):
            f = x.astype(np.float32)
            back = f.astype(np.float64)
            u = f.view(np.uint32)
            off = np.isfinite(x) & (back != x)
            away = off & (np.abs(back) > np.abs(x))
            u = np.where(away, u - 1, u)
            u = np.where(off, u | 1, u).astype(np.uint32)
        return dt.to_bf16(u.view(np.float32))
    with np.errstate(over="ignore"):
        return x.astype(dtype)


def _packed(seqs, n, context_lens, query_starts):
    """(sequence, first row, rows, length) of every sequence of a packed batch."""
    for b in range(seqs):
        lo, hi = b, b + 1
        if query_starts is not None:
            lo = min(max(int(query_starts[b]), 0), n)
            hi = min(max(int(query_starts[b + 1]), lo), n)
        yield b, lo, hi - lo, min(max(int(context_lens[b]), 0), 2**30)


@rotary_append.impl("cpu")
def _rotary_append_cpu(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts=None):
    """Rotates q and k by the tables' rows at the tokens' positions and writes
    k and v into the cache; returns the rotated q.

    q (tokens, heads, head_dim), k / v (tokens, kv_heads, head_dim); cos / sin
    (positions, r / 2) float32 turn the pairs (i, i + r / 2) of the first r
    elements of a head, the rest stay as they are.  A token whose position is
    outside the tables is dropped (its row of the result is 0 and nothing is
    written); a token whose page is none is rotated but not written.  Two
    tokens of one call must not share a cache row."""
    _check_append(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts)
    if key_cache is value_cache:
        raise ValueError("key_cache and value_cache are the same array")
    dtype, half = q.dtype, cos.shape[1]
    pages, page = key_cache.shape[:2]
    width, n = block_tables.shape[1], q.shape[0]
    out = _store(np.zeros(q.shape), dtype)
    for b, lo, m, length in _packed(block_tables.shape[0], n, context_lens, query_starts):
        for i in range(m):
            p, t = length - m + i, lo + i
            if not 0 <= p < cos.shape[0]:
                continue
            c, s = (np.asarray(x[p], np.float64) for x in (cos, sin))

            def turn(x):
                x = _to64(x)
                a, z = x[:, :half], x[:, half:2 * half]
                return _store(np.concatenate([a * c - z * s, a * s + z * c, x[:, 2 * half:]], 1), dtype)

            out[t] = turn(q[t])
            at = int(block_tables[b, p // page]) if p // page < width else -1
            if 0 <= at < pages:
                key_cache[at, p % page] = turn(k[t])
                value_cache[at, p % page] = v[t]
    return out


def _attend(q, k, v, seen, scale):
    """q (n, Hq, D), k / v (m, Hkv, D), seen (n, m), all float64."""
    n, hq, dim = q.shape
    rep = hq // k.shape[1]
    out = np.zeros(q.shape)
    with np.errstate(invalid="ignore", over="ignore"):
        for h in range(hq):
            kk, vv = k[:, h // rep], v[:, h // rep]
            for i in range(n):  # a query's own keys only: nothing else enters
                s = (kk[seen[i]] @ q[i, h]) * scale
                if s.size == 0 or s.max() == -np.inf:
                    continue
                e = np.exp(s - s.max())
                e = np.where(s == -np.inf, 0.0, np.maximum(e, 5e-324))  # (no weight of a finite score is 0)
                out[i, h] = (e @ vv[seen[i]]) / e.sum()
    return out


def _seen(p, keys, length, window, sinks):
    p, j = np.asarray(p)[:, None], np.asarray(keys)[None]
    ok = (j <= p) & (j < length) & (p < length)
    return ok & ((p - j < window) | (j < sinks)) if window is not None else ok


@paged_attention.impl("cpu")
def _paged_attention_cpu(q, key_cache, value_cache, block_tables, context_lens, query_starts=None, *, window=None,
                         sinks=0, scale=None):
    """softmax(scale q . k) v of the new tokens q (tokens, heads, head_dim)
    over the cached keys and values of their sequences; the result has q's
    shape.  ``window`` / ``sinks``: see the module; ``scale`` defaults to
    1 / sqrt(head_dim)."""
    window, sinks, scale = _check_paged(q, key_cache, value_cache, block_tables, context_lens, query_starts, window,
                                        sinks, scale)
    pages, page, hkv, dim = key_cache.shape
    out = np.zeros(q.shape)
    for b, lo, m, length in _packed(block_tables.shape[0], q.shape[0], context_lens, query_starts):
        keys = np.arange(min(length, block_tables.shape[1] * page))
        at = np.asarray(block_tables)[b][keys // page].astype(np.int64)
        keys, at = keys[(at >= 0) & (at < pages)], at[(at >= 0) & (at < pages)]
        p = np.arange(length - m, length)
        out[lo:lo + m] = _attend(_to64(q[lo:lo + m]), _to64(key_cache[at, keys % page]),
                                 _to64(value_cache[at, keys % page]), _seen(p, keys, length, window, sinks), scale)
    return _store(out, q.dtype)


@window_attention.impl("cpu")
def _window_attention_cpu(q, k, v, lengths=None, positions=None, *, window=None, sinks=0, scale=None):
    """Causal attention of q (B, S, heads, head_dim) to k / v (B, T, kv_heads,
    head_dim), with a window and sinks as the module says.  Query i of
    sequence b sits at position positions[b] + i (T - S + i by default);
    ``lengths`` counts a sequence's keys (T by default), and queries at or
    past it are padding, whose rows come out 0."""
    window, sinks, scale = _check_window(q, k, v, lengths, positions, window, sinks, scale)
    (B, S), T = q.shape[:2], k.shape[1]
    out = np.zeros(q.shape)
    for b in range(B):
        length = T if lengths is None else min(max(int(lengths[b]), 0), T)
        p = np.arange(S) + (T - S if positions is None else int(positions[b]))
        out[b] = _attend(_to64(q[b]), _to64(k[b]), _to64(v[b]), _seen(p, np.arange(T), length, window, sinks), scale)
    return _store(out, q.dtype)


@sample.impl("cpu")
def _sample_cpu(logits, uniform, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """One token of each row of logits (rows, vocab) -> int32 (rows,), drawn by
    the given numbers ``uniform`` (rows,) in [0, 1).

    Weights are exp((x - max) / temperature).  Kept are, of the tokens in
    descending order of their logit (ties: the lower index first), the first
    ``top_k`` (None, or below 1: all), of these the shortest beginning that
    holds ``top_p`` of their weight, at least one, and of these the ones that
    weigh ``min_p`` of the first.  The draw is the first kept token, in the
    order of the vocabulary, up to and with which the kept weights exceed
    uniform times their sum.  A temperature of 0 takes the largest logit.
    Filters are numbers or one value per row; those of a row outside their
    range count as the nearest end.  NaN and -inf logits are never drawn; a
    row without any other gives -1.

    On the GPU weights are whole steps of 2^-36 of the largest: tokens below
    2^-37 of it (25.6 temperatures under the largest logit) are never drawn and
    add nothing to a sum; a share is taken of those sums, exactly."""
    rows, vocab, temperature, top_k, top_p, min_p = _check_sample(logits, uniform, temperature, top_k, top_p, min_p)
    x = _to64(logits)
    row = lambda v, r: v if not hasattr(v, "shape") else v[r]  # noqa: E731
    out = np.full(rows, -1, np.int32)
    for r in range(rows):
        z = np.where(np.isnan(x[r]), -np.inf, x[r])
        order = np.argsort(-z, kind="stable")
        best = z[order[0]]
        if best == -np.inf:
            continue
        t = float(row(temperature, r))
        if not t > 0:
            out[r] = order[0]
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            d = np.where(z == best, 0.0, (z - best) / t)
        w = np.exp(np.where(np.isnan(d), -np.inf, d))
        n = vocab
        if top_k is not None and int(row(top_k, r)) > 0:
            n = min(n, int(row(top_k, r)))
        if top_p is not None and float(row(top_p, r)) < 1:
            mass = np.cumsum(w[order[:n]])
            n = min(n, 1 + int(np.searchsorted(mass, float(row(top_p, r)) * mass[-1], side="left")))
        kept = order[:n]
        if min_p is not None and float(row(min_p, r)) > 0:
            kept = kept[w[kept] >= min(float(row(min_p, r)), 1.0)]
        kept = np.sort(kept[w[kept] > 0])
        mass = np.cumsum(w[kept])
        i = int(np.searchsorted(mass, max(float(uniform[r]), 0.0) * mass[-1], side="right"))
        out[r] = kept[min(i, len(kept) - 1)]
    return out
