"""What a generation loop does around its kernels, on the GPU: block tables and
slots of a step from its lengths, the choice of a beam search's beams, and the
paged caches that follow them.

Rows of ``block_tables`` (rows, width) name pages of a cache as in
:mod:`nkipy_amd.core.ops.serving`.  Rows may share pages: a page that holds
page_size tokens of a row is not written again, so ``beam_reorder`` lets rows
share those and keeps only the page that still fills a row's own.  No list of
free pages is kept: ``assign_pages`` takes every page that no row names among
the pages it holds.
"""

from __future__ import annotations

import numpy as np

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core.ops._registry import Op
from nkipy_amd.core.ops.serving import _FLOATS, _float, _int_value, _ints, _shape, _to64
from nkipy_amd.core.ops.serving_fp8 import build_updates, check_exps, distinct, updated_argument

MAX_BEAMS = 32
MAX_PAGES = 2**20
MAX_VOCAB = 2**22
MAX_CHOICES = 2**23  # beams x vocabulary


# ---------------------------------------------------------------------------
# Checks shared by the traced and the CPU forms
# ---------------------------------------------------------------------------
def _whole(x, name, lo, hi):
    if isinstance(x, bool) or not isinstance(x, (int, np.integer)) or not lo <= x <= hi:
        raise ValueError(f"{name} must be a whole number of {lo} to {hi}, got {x!r}")
    return int(x)


def _check_table(block_tables):
    rows, width = _shape(block_tables, "block_tables", 2)
    if rows < 1 or width < 1:
        raise ValueError(f"block_tables of shape {(rows, width)} name no page")
    if dt.canonical(block_tables.dtype) != dt.int32:
        raise TypeError(f"block_tables are written in place: they must be of int32, got {dt.name(block_tables.dtype)}")
    return rows, width


def _check_assign(block_tables, context_lens, new_lens, pages, page_size, tokens):
    rows, width = _check_table(block_tables)
    _ints(context_lens, "context_lens", (rows,))
    _ints(new_lens, "new_lens", (rows,))
    pages = _whole(pages, "pages", 1, MAX_PAGES)
    page = _whole(page_size, "page_size", 1, 2**30)
    tokens = _whole(tokens, "tokens", 0, 2**30)
    if width * page >= 2**30 or pages * page >= 2**31:
        raise ValueError("block_tables or cache too large: positions and cache rows are 32-bit")
    if rows > 2**16:
        raise ValueError(f"{rows} sequences are too many: up to {2**16}")
    return pages, page, tokens


def _check_select(logits, scores, ended, end_token):
    groups, beams = _shape(scores, "scores", 2)
    rows, vocab = _shape(logits, "logits", 2)
    if groups < 1 or not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"scores must be of (groups, 1 to {MAX_BEAMS} beams), got {(groups, beams)}")
    if rows != groups * beams:
        raise ValueError(f"logits must have a row for each of {groups} x {beams} beams, got {rows}")
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"a vocabulary of {vocab}: from 1 to {MAX_VOCAB} tokens")
    if beams * vocab > MAX_CHOICES:
        raise ValueError(f"{beams} beams of {vocab} tokens are too many to choose from: up to {MAX_CHOICES} in all")
    _float(logits, "logits", _FLOATS)
    _float(scores, "scores", (dt.float32,))
    _ints(ended, "ended", (groups, beams))
    return groups, beams, vocab, _whole(end_token, "end_token", -1, vocab - 1)


def _check_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps, value_exps):
    groups, beams = _shape(parents, "parents", 2)
    if groups < 1 or not 1 <= beams <= MAX_BEAMS:
        raise ValueError(f"parents must be of (groups, 1 to {MAX_BEAMS} beams), got {(groups, beams)}")
    _ints(parents, "parents", (groups, beams))
    rows, width = _check_table(block_tables)
    if rows != groups * beams:
        raise ValueError(f"block_tables must have a row for each of {groups} x {beams} beams, got {rows}")
    _ints(context_lens, "context_lens", (rows,))
    pages, page, hkv, dim = _shape(key_cache, "key_cache", 4)
    if _shape(value_cache, "value_cache", 4) != (pages, page, hkv, dim):
        raise ValueError(f"value_cache must have key_cache's shape {(pages, page, hkv, dim)}, got {tuple(value_cache.shape)}")
    if min(pages, page, hkv, dim) < 1:
        raise ValueError("the cache holds no page")
    if width * page >= 2**30 or pages * page >= 2**31:
        raise ValueError("block_tables or cache too large: positions and cache rows are 32-bit")
    kinds = [dt.canonical(x.dtype) for x in (key_cache, value_cache)]
    for d in kinds:
        if d not in _FLOATS + (dt.float8_e4m3fn,):
            raise TypeError(f"caches must be of bfloat16 / float16 / float32 / float8_e4m3fn, got {dt.name(d)}")
    if kinds[0] != kinds[1]:
        raise TypeError(f"caches must share one type, got {dt.name(kinds[0])} and {dt.name(kinds[1])}")
    if (key_exps is None) != (value_exps is None):
        raise ValueError("give both of key_exps and value_exps, or neither")
    if (key_exps is not None) != (kinds[0] == dt.float8_e4m3fn):
        raise ValueError("caches of float8_e4m3fn have exponents, others none")
    if key_exps is not None:
        check_exps(key_exps, "key_exps", pages, hkv)
        check_exps(value_exps, "value_exps", pages, hkv)
    distinct(parents=parents, block_tables=block_tables, context_lens=context_lens, key_cache=key_cache,
             value_cache=value_cache, key_exps=key_exps, value_exps=value_exps)


# ---------------------------------------------------------------------------
# Traced forms
# ---------------------------------------------------------------------------
assign_pages = Op("assign_pages")


@assign_pages.impl("hip")
def _assign_pages_hip(block_tables, context_lens, new_lens, *, pages, page_size, tokens):
    pages, page, tokens = _check_assign(block_tables, context_lens, new_lens, pages, page_size, tokens)
    ops = [updated_argument(block_tables, "block_tables"), _int_value(context_lens), _int_value(new_lens)]
    rows = ops[0].shape[0]
    return tuple(build_updates("assign_pages", ops, [("starts", (rows + 1,), dt.int32), ("slots", (tokens,), dt.int32),
                                                     ("free", (1,), dt.int32)], [("tables", block_tables, 0)],
                               {"pages": pages, "page": page, "tokens": tokens}))


beam_select = Op("beam_select")


@beam_select.impl("hip")
def _beam_select_hip(logits, scores, ended, *, end_token):
    from nkipy_amd.core.ops._helpers import val

    groups, beams, _, end = _check_select(logits, scores, ended, end_token)
    ops = [val(logits), val(scores, dt.float32), _int_value(ended)]
    shape = (groups, beams)
    return tuple(build_updates("beam_select", ops, [("tokens", shape, dt.int32), ("parents", shape, dt.int32),
                                                    ("scores", shape, dt.float32), ("ended", shape, dt.int32)], [],
                               {"end": end}))


beam_reorder = Op("beam_reorder")


@beam_reorder.impl("hip")
def _beam_reorder_hip(parents, block_tables, context_lens, key_cache, value_cache, key_exps=None, value_exps=None):
    _check_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps, value_exps)
    arrays = {"tables": (block_tables, "block_tables"), "key_cache": (key_cache, "key_cache"),
              "value_cache": (value_cache, "value_cache")}
    if key_exps is not None:
        arrays.update(key_exps=(key_exps, "key_exps"), value_exps=(value_exps, "value_exps"))
    ops = [_int_value(parents), _int_value(context_lens)] + [updated_argument(x, name) for x, name in arrays.values()]
    build_updates("beam_reorder", ops, [], [(part, x, 2 + i) for i, (part, (x, _)) in enumerate(arrays.items())], {})


# ---------------------------------------------------------------------------
# CPU forms
# ---------------------------------------------------------------------------
@assign_pages.impl("cpu")
def _assign_pages_cpu(block_tables, context_lens, new_lens, *, pages, page_size, tokens):
    """Gives every sequence the pages for its new tokens: ``block_tables``
    (sequences, width) int32 is updated in place; returns (query_starts, slots,
    free), int32.

    Sequence b has context_lens[b] tokens, the last new_lens[b] of them new
    (both at least 0, where they are less).  It holds the pages of the tokens
    before those: entries 0 .. held-1 of its row, held = ceil((length - new) /
    page_size), which stay as they are.  The entries behind them, up to
    ceil(length / page_size), get the pages of 0 .. pages-1 that no row holds, the
    lowest first, in the order of rows and entries; where none is left they are
    -1, and so are all entries further behind.  A sequence of length 0 gives its
    pages back.

    query_starts (sequences + 1) are the running sums of the new lengths.  slots
    (tokens,) says for each token of the packed batch in which cache row (page *
    page_size + row) it lies, -1 where it has none: outside every sequence,
    before position 0, past the table, without a page.  free (1,) counts the
    pages left, below 0 those that lacked."""
    pages, page, tokens = _check_assign(block_tables, context_lens, new_lens, pages, page_size, tokens)
    rows, width = block_tables.shape
    length = np.clip(np.asarray(context_lens).astype(np.int64), 0, 2**30)
    new = np.clip(np.asarray(new_lens).astype(np.int64), 0, 2**30)
    held = np.minimum((np.maximum(length - new, 0) + page - 1) // page, width)
    need = np.minimum((length + page - 1) // page, width)
    kept = np.zeros(pages, bool)
    for b in range(rows):
        at = block_tables[b, :held[b]]
        kept[at[(at >= 0) & (at < pages)]] = True
    free = np.flatnonzero(~kept)
    given = 0
    for b in range(rows):
        want = max(int(need[b] - held[b]), 0)
        got = free[given:given + want]
        block_tables[b, held[b]:] = -1
        block_tables[b, held[b]:held[b] + len(got)] = got
        given += want
    starts = np.concatenate([[0], np.cumsum(new)])
    slots = np.full(tokens, -1, np.int32)
    for b in range(rows):
        for i in range(min(int(new[b]), max(tokens - int(starts[b]), 0))):
            p = int(length[b] - new[b]) + i
            if 0 <= p < width * page and 0 <= block_tables[b, p // page] < pages:
                slots[starts[b] + i] = block_tables[b, p // page] * page + p % page
    return (np.minimum(starts, 2**31 - 1).astype(np.int32), slots, np.array([len(free) - given], np.int32))


@beam_select.impl("cpu")
def _beam_select_cpu(logits, scores, ended, *, end_token):
    """One step of a beam search: of all beams' continuations by one token, the
    best as many as there are beams, for each group.  Returns (tokens, parents,
    scores, ended), all (groups, beams): tokens, parents and ended int32, scores
    float32.

    logits (groups * beams, vocab): a row for each beam; scores (groups, beams)
    float32: the beams' log probabilities so far; ended (groups, beams) int: not 0
    for a beam that has ended.  Token t continues beam b with

        scores[b] + logits[b, t] - log sum_u exp(logits[b, u])

    and a beam that has ended stands once, with ``end_token`` and its score
    unchanged.  The best come first; of equal ones the lower beam, then the lower
    token.  ``parents`` are beams of the same group; ``ended`` is 1 where the
    parent has ended or the token is ``end_token`` (-1: no token is).

    NaN and -inf logits, and beams whose score is NaN or -inf (those not begun
    yet), continue nothing; where too few continuations are left the rest have
    token -1, the parent at their own place, score -inf and that parent's
    ``ended``.  Logits of +inf share the weight of their row.

    On the GPU a row's sum has 32-bit terms, added up in 32 bits over up to
    8192 logits and in 64 over those sums; scores are compared in 64 bits."""
    groups, beams, vocab, end = _check_select(logits, scores, ended, end_token)
    x = _to64(logits).reshape(groups, beams, vocab)
    out = [np.zeros((groups, beams), d) for d in (np.int32, np.int32, np.float32, np.int32)]
    for g in range(groups):
        offers = []
        for b in range(beams):
            s = float(scores[g, b])
            if np.isnan(s) or s == -np.inf:
                continue
            if ended[g, b]:
                offers.append((-s, b, end))
                continue
            z = np.where(np.isnan(x[g, b]), -np.inf, x[g, b])
            best = z.max()
            if best == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                d = np.where(z == best, 0.0, z - best)
            d = d - np.log(np.exp(d).sum())
            for t in np.argsort(-d, kind="stable")[:beams]:
                if d[t] > -np.inf:
                    offers.append((-(s + d[t]), b, int(t)))
        offers.sort()
        for j in range(beams):
            s, b, t = offers[j] if j < len(offers) else (np.inf, j, -1)
            out[0][g, j], out[1][g, j], out[2][g, j] = t, b, -s
            out[3][g, j] = int(bool(ended[g, b]) or (t == end and t >= 0))
    return tuple(out)


@beam_reorder.impl("cpu")
def _beam_reorder_cpu(parents, block_tables, context_lens, key_cache, value_cache, key_exps=None, value_exps=None):
    """Every beam goes on from its parent's cache: ``block_tables`` (groups *
    beams, width) int32, the caches and their exponents are updated in place.

    parents (groups, beams): for each beam, which beam of its group it continues
    (one outside 0 .. beams-1: itself).  The beams of a group have one length, the
    one of its first in context_lens (groups * beams,).  A row of the table takes
    its parent's entries of the pages that are full, so rows come to share
    them.  The page behind, where the length leaves one in part filled, stays the
    row's own: its written rows (and its exponents) become copies of the
    parent's.  A row or a parent without such a page copies nothing; those of a
    group's rows must be different pages."""
    _check_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps, value_exps)
    groups, beams = parents.shape
    pages, page = key_cache.shape[:2]
    width = block_tables.shape[1]
    for g in range(groups):
        rows = np.arange(g * beams, g * beams + beams)
        up = np.asarray(parents[g]).astype(np.int64)
        up = np.where((up >= 0) & (up < beams), up, np.arange(beams))
        full, tail = divmod(min(max(int(context_lens[rows[0]]), 0), width * page), page)
        table = block_tables[rows]
        block_tables[rows, :full] = table[up, :full]
        if tail == 0:
            continue
        at = table[:, full]
        for cache, size in ((key_cache, tail), (value_cache, tail), (key_exps, None), (value_exps, None)):
            if cache is None:
                continue
            moves = [(int(at[b]), cache[at[up[b]], :size].copy()) for b in range(beams)
                     if 0 <= at[b] < pages and 0 <= at[up[b]] < pages]
            for pg, rows_ in moves:
                cache[pg, :size] = rows_
    return None
