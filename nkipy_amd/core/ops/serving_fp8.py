"""A paged cache of 8-bit keys and values, and attention over it.

A cache is an array of float8_e4m3fn codes of shape (pages, page_size,
n_kv_heads, head_dim) and an int32 array of exponents (pages, n_kv_heads): a
code on page g, head h stands for code * 2^exponent[g, h].  Exponents outside
-120 .. 120 count as the nearest end.  Pages, block tables, lengths, query
starts, what a query sees and what its row holds then are those of
:mod:`nkipy_amd.core.ops.serving`.

The scale is a power of two because e4m3 floats: its four significant bits are
the same under any scale, and a power of two is taken off and put on exactly.

A page's exponent belongs to the rows written so far.  A call that writes a
page's first row sets it afresh, to the least exponent (of at least -120) under
which the largest finite magnitude that the call writes on that page and head
is up to 448; a call that writes behind rows written earlier takes the larger
of that and the exponent there, and where it grows, rounds the codes of the
earlier rows again to the new scale (exact but for codes that get subnormal).
Values that are not finite become NaN.

The CPU forms are evaluated in float64.  On the GPU the two products of a
rotation and their sum are 32-bit roundings, so a code may be the neighbouring
one where a value lies that close to the middle between two.
"""

from __future__ import annotations

import numpy as np

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core.ops._registry import Op
from nkipy_amd.core.ops.serving import (
    _LAYOUT_OPS, _WRITE_OPS, _attend, _float, _heads, _int_value, _packed, _same, _scale, _seen, _shape, _store, _tables,
    _to64, _window,
)

EXP_MIN, EXP_MAX = -120, 120


# ---------------------------------------------------------------------------
# Checks shared by the traced and the CPU forms
# ---------------------------------------------------------------------------
def check_exps(exps, name, pages, hkv):
    if _shape(exps, name, 2) != (pages, hkv):
        raise ValueError(f"{name} must have shape {(pages, hkv)}, got {tuple(exps.shape)}")
    if dt.canonical(exps.dtype) != dt.int32:
        raise TypeError(f"{name} must be of int32, got {dt.name(exps.dtype)}")


def _check_caches(key_cache, value_cache, key_exps, value_exps):
    pages, _, hkv, _ = _shape(key_cache, "key_cache", 4)
    for x, name in ((key_cache, "key_cache"), (value_cache, "value_cache")):
        if dt.canonical(x.dtype) != dt.float8_e4m3fn:
            raise TypeError(f"{name} must be of float8_e4m3fn, got {dt.name(x.dtype)}")
    check_exps(key_exps, "key_exps", pages, hkv)
    check_exps(value_exps, "value_exps", pages, hkv)


def _check_append(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                  query_starts):
    n, hq, dim = _shape(q, "q", 3)
    _, _, hkv, cdim, _ = _tables(n, key_cache, value_cache, block_tables, context_lens, query_starts)
    _check_caches(key_cache, value_cache, key_exps, value_exps)
    for x, name in ((k, "k"), (v, "v")):
        if _shape(x, name, 3) != (n, hkv, cdim):
            raise ValueError(f"{name} must have shape {(n, hkv, cdim)}, got {tuple(x.shape)}")
    if dim != cdim:
        raise ValueError(f"q has head_dim {dim}, the cache {cdim}")
    _heads(hq, hkv, dim)
    _same({"q": q, "k": k, "v": v})
    positions, half = _shape(cos, "cos", 2)
    if _shape(sin, "sin", 2) != (positions, half):
        raise ValueError(f"sin must have cos's shape {(positions, half)}, got {tuple(sin.shape)}")
    if not 1 <= half <= dim // 2 or positions < 1:
        raise ValueError(f"cos / sin of shape {(positions, half)} do not fit head_dim {dim}: (positions, up to head_dim / 2)")
    for x, name in ((cos, "cos"), (sin, "sin")):
        _float(x, name, (dt.float32,))
    distinct(key_cache=key_cache, value_cache=value_cache, key_exps=key_exps, value_exps=value_exps)


def _check_attention(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens, query_starts, window,
                     sinks, scale):
    n, hq, dim = _shape(q, "q", 3)
    _, _, hkv, cdim, _ = _tables(n, key_cache, value_cache, block_tables, context_lens, query_starts)
    _check_caches(key_cache, value_cache, key_exps, value_exps)
    if dim != cdim:
        raise ValueError(f"q has head_dim {dim}, the cache {cdim}")
    _heads(hq, hkv, dim)
    _float(q, "q")
    return _window(window, sinks) + (_scale(scale, dim),)


def distinct(**arrays):
    """Arrays that a call writes: no two of them the same."""
    seen = {}
    for name, x in arrays.items():
        if x is None:
            continue
        if id(x) in seen:
            raise ValueError(f"{seen[id(x)]} and {name} are the same array")
        seen[id(x)] = name


# ---------------------------------------------------------------------------
# Traced forms: a node for each result, all over the same operands
# ---------------------------------------------------------------------------
def updated_argument(x, name):
    """The value of an array that a call writes in place: a whole argument of
    the kernel, possibly written before."""
    from nkipy_amd.core.ops._helpers import is_traced, val

    if not is_traced(x):
        raise TypeError(f"{name} is written in place: it must be an argument of the kernel")
    v = here = val(x)
    part = False
    while v.node is not None and ("target" in v.node.attrs or v.node.op in _LAYOUT_OPS + _WRITE_OPS):
        part = part or v.node.op in _LAYOUT_OPS
        v = v.node.inputs[v.node.attrs.get("target") or 0]
    if not v.is_parameter:
        raise TypeError(f"{name} is written in place: it must be an argument of the kernel, not computed in it")
    if part:
        raise ValueError(f"{name} is a part or another layout of the argument {v.name!r}, which a write into it would not "
                         "reach: pass each array as an argument of its own")
    if x._original_parameter is None:  # (a slice or reshape that changes nothing: the argument's value, not itself)
        raise ValueError(f"{name} is a view of the argument {v.name!r}, which a write into it would not reach: "
                         "pass the argument itself")
    return here


def build_updates(op, operands, results, updates, attrs):
    """Nodes ``op`` over the same operands: one for each result (part, shape,
    dtype), then one for each updated array (part, traced array, its place
    among the operands), which is rebound to its node.  Returns the results."""
    from nkipy_amd.core.ops._helpers import ctx, wrap

    cx = ctx()
    out = [wrap(cx.build_op(op, operands, shape, dtype, {**attrs, "part": part})) for part, shape, dtype in results]
    for part, x, at in updates:
        v = operands[at]
        new = cx.build_op(op, operands, v.shape, v.dtype, {**attrs, "part": part, "target": at})
        x._is_mutated = True
        x._rebind(wrap(new))
    return out


rotary_append_fp8 = Op("rotary_append_fp8")


@rotary_append_fp8.impl("hip")
def _rotary_append_fp8_hip(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                           query_starts=None):
    from nkipy_amd.core.ops._helpers import val

    _check_append(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens, query_starts)
    arrays = {"key_cache": key_cache, "value_cache": value_cache, "key_exps": key_exps, "value_exps": value_exps}
    ops = [val(q), val(k), val(v), val(cos, dt.float32), val(sin, dt.float32)]
    ops += [updated_argument(x, name) for name, x in arrays.items()]
    ops += [_int_value(block_tables), _int_value(context_lens)]
    if query_starts is not None:
        ops.append(_int_value(query_starts))
    return build_updates("append_fp8", ops, [("q", ops[0].shape, ops[0].dtype)],
                         [(name, x, 5 + i) for i, (name, x) in enumerate(arrays.items())],
                         {"starts": query_starts is not None})[0]


paged_attention_fp8 = Op("paged_attention_fp8")


@paged_attention_fp8.impl("hip")
def _paged_attention_fp8_hip(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                             query_starts=None, *, window=None, sinks=0, scale=None):
    from nkipy_amd.core.ops._helpers import ctx, val, wrap

    window, sinks, scale = _check_attention(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                                            query_starts, window, sinks, scale)
    ops = [val(q), val(key_cache), val(value_cache), val(key_exps), val(value_exps), _int_value(block_tables),
           _int_value(context_lens)]
    if query_starts is not None:
        ops.append(_int_value(query_starts))
    return wrap(ctx().build_op("paged_attention_fp8", ops, ops[0].shape, ops[0].dtype,
                               {"window": window or 0, "sinks": sinks, "scale": scale,
                                "starts": query_starts is not None}))


# ---------------------------------------------------------------------------
# CPU forms
# ---------------------------------------------------------------------------
def _codes(x):
    """float64 values of up to 448 in magnitude rounded once to e4m3 (ties to
    even); what is not finite becomes NaN."""
    fine = np.isfinite(x)
    x = np.where(fine, x, 0.0)
    step = np.ldexp(1.0, np.maximum(np.frexp(x)[1] - 4, -9))  # of the last place
    y = np.copysign(np.rint(x / step) * step, x)
    return dt.to_e4m3fn(np.where(fine, y, np.nan).astype(np.float32))


def _exponent(x):
    """The least exponent >= -120 that brings the finite values of x to 448."""
    top = np.abs(x[np.isfinite(x)]).max(initial=0.0)
    if top == 0:
        return EXP_MIN
    m, e = np.frexp(top)  # 448 = 0.875 * 2^9
    return max(int(e) - 9 + int(m > 0.875), EXP_MIN)


def _clip(exps):
    return np.clip(np.asarray(exps).astype(np.int64), EXP_MIN, EXP_MAX)


def _values(codes, exps):
    """float64 values of codes (..., heads, dim) under exponents (..., heads)."""
    return np.ldexp(_to64(codes), _clip(exps)[..., None])


@rotary_append_fp8.impl("cpu")
def _rotary_append_fp8_cpu(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                           query_starts=None):
    """Rotates q and k by the tables' rows at the tokens' positions and writes
    k and v into the cache as codes, updating the pages' exponents; returns the
    rotated q.

    Operands as those of ``rotary_append``, with caches of float8_e4m3fn and
    int32 exponents (pages, kv_heads) for keys and values.  The same tokens are
    dropped.  Two sequences of one call must not write the same page."""
    _check_append(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens, query_starts)
    half, (pages, page) = cos.shape[1], key_cache.shape[:2]
    width, n = block_tables.shape[1], q.shape[0]
    out = _store(np.zeros(q.shape), q.dtype)

    def turn(x, p):
        x = _to64(x)
        c, s = (np.asarray(t[p], np.float64) for t in (cos, sin))
        a, z = x[:, :half], x[:, half:2 * half]
        with np.errstate(invalid="ignore", over="ignore"):
            return np.concatenate([a * c - z * s, a * s + z * c, x[:, 2 * half:]], 1)

    for b, lo, m, length in _packed(block_tables.shape[0], n, context_lens, query_starts):
        at = {}  # page: its new rows, in order, and their tokens
        for i in range(m):
            p, t = length - m + i, lo + i
            if not 0 <= p < cos.shape[0]:
                continue
            out[t] = _store(turn(q[t], p), q.dtype)
            pg = int(block_tables[b, p // page]) if p // page < width else -1
            if 0 <= pg < pages:
                at.setdefault((p // page, pg), []).append((p, t))
        for (_, pg), rows in at.items():
            first = rows[0][0] % page
            for codes, exps, x in ((key_cache, key_exps, [turn(k[t], p) for p, t in rows]),
                                   (value_cache, value_exps, [_to64(v[t]) for _, t in rows])):
                x = np.stack(x)
                for h in range(x.shape[1]):
                    e, old = _exponent(x[:, h]), int(_clip(exps[pg, h]))
                    if first > 0:
                        e = max(e, old)
                        if e > old:
                            codes[pg, :first, h] = _codes(np.ldexp(_to64(codes[pg, :first, h]), old - e))
                    codes[pg, first:first + len(rows), h] = _codes(np.ldexp(x[:, h], -e))
                    exps[pg, h] = e
    return out


@paged_attention_fp8.impl("cpu")
def _paged_attention_fp8_cpu(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                             query_starts=None, *, window=None, sinks=0, scale=None):
    """softmax(scale q . k) v of the new tokens q (tokens, heads, head_dim) of
    bf16, fp16 or fp32 over the cached keys and values of their sequences; the
    result has q's shape and type.  ``window``, ``sinks``, ``scale`` as those of
    ``paged_attention``.

    On the GPU keys and values enter as exactly what they stand for.  Weights
    have 32 bits, but where q has 16 bits and a head dim of 64 or 128: there
    they keep 2^-16 of themselves before the values are summed, and with
    ``query_starts`` and a bfloat16 q are rounded to bfloat16."""
    window, sinks, scale = _check_attention(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                                            query_starts, window, sinks, scale)
    pages, page = key_cache.shape[:2]
    out = np.zeros(q.shape)
    for b, lo, m, length in _packed(block_tables.shape[0], q.shape[0], context_lens, query_starts):
        keys = np.arange(min(length, block_tables.shape[1] * page))
        at = np.asarray(block_tables)[b][keys // page].astype(np.int64)
        keys, at = keys[(at >= 0) & (at < pages)], at[(at >= 0) & (at < pages)]
        p = np.arange(length - m, length)
        out[lo:lo + m] = _attend(_to64(q[lo:lo + m]), _values(key_cache[at, keys % page], key_exps[at]),
                                 _values(value_cache[at, keys % page], value_exps[at]),
                                 _seen(p, keys, length, window, sinks), scale)
    return _store(out, q.dtype)
