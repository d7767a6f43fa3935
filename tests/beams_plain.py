"""Plain forms of the generation loop's operators, written from their contracts
(whole arrays, one sort), and the cases their tests share."""

import numpy as np

import serving_plain as P


def assign(tables, lens, new, pages, page, tokens):
    """(tables, starts, slots, free)."""
    rows, width = tables.shape
    lens, new = np.clip(lens, 0, 2**30).astype(int), np.clip(new, 0, 2**30).astype(int)
    held = np.minimum(-(-np.maximum(lens - new, 0) // page), width)
    need = np.minimum(-(-lens // page), width)
    used = {int(x) for b in range(rows) for x in tables[b, :held[b]] if 0 <= x < pages}
    free = sorted(set(range(pages)) - used)
    left = len(free)
    out = tables.copy()
    for b in range(rows):
        for i in range(held[b], width):
            out[b, i] = -1
            if i < need[b]:
                left -= 1
                if free:
                    out[b, i] = free.pop(0)
    starts = np.concatenate([[0], np.cumsum(new)])
    slots = np.full(tokens, -1)
    for t in range(min(tokens, starts[-1])):
        b = int(np.searchsorted(starts, t, side="right")) - 1
        p = lens[b] - new[b] + t - starts[b]
        if 0 <= p < width * page and 0 <= out[b, p // page] < pages:
            slots[t] = out[b, p // page] * page + p % page
    return out, starts, slots, np.array([left])


def continuations(logits, scores, ended, end):
    """Log probabilities (groups, beams, vocab) of every beam's continuations in
    float64, -inf where there is none."""
    g, k = scores.shape
    x = P.up(logits).reshape(g, k, -1)
    x = np.where(np.isnan(x), -np.inf, x)
    out = np.full(x.shape, -np.inf)
    for a in range(g):
        for b in range(k):
            s = float(scores[a, b])
            if np.isnan(s) or s == -np.inf:
                continue
            if ended[a, b]:
                out[a, b, max(end, 0)] = s
                continue
            top = x[a, b].max()
            if top == -np.inf:
                continue
            if top == np.inf:
                w = (x[a, b] == np.inf).astype(float)
            else:
                w = np.exp(x[a, b] - top)
            with np.errstate(divide="ignore", invalid="ignore"):
                d = np.log(w / w.sum()) if top == np.inf else x[a, b] - top - np.log(w.sum())
            out[a, b] = s + d
    return out


def check_select(got, logits, scores, ended, end, tol):
    """The outputs (tokens, parents, scores, ended) against the sorted
    continuations: each chosen one carries its own score, no other is better by
    more than twice ``tol`` (an error in each of two sums), the order is that of
    the scores and, between equal ones, of the places."""
    tokens, parents, new, over = (np.asarray(x) for x in got)
    g, k = scores.shape
    c = continuations(logits, scores, ended, end)
    vocab = c.shape[2]
    for a in range(g):
        flat = c[a].reshape(-1)
        n = min(k, int((flat > -np.inf).sum()))
        order = np.lexsort((np.arange(flat.size), -flat))[:n]
        at = []
        for j in range(n):
            b, t = int(parents[a, j]), int(tokens[a, j])
            assert 0 <= b < k
            if ended[a, b]:
                assert t == end and over[a, j] == 1 and new[a, j] == scores[a, b]
                t = max(end, 0)
            assert 0 <= t < vocab
            at.append(b * vocab + t)
            mine, best = flat[at[-1]], flat[order[j]]
            assert mine == best or abs(mine - best) <= 2 * tol, (a, j, mine, best)
            assert new[a, j] == np.float32(mine) or abs(new[a, j] - mine) <= tol + 2.0**-24 * abs(mine)
            assert over[a, j] == int(bool(ended[a, b]) or t == end)
            if mine == best and at[-1] != order[j]:  # equal ones stand in the order of their places
                assert flat[at[-1]] != flat[order[j]] or sorted(at[-1:] + [order[j]])[0] == order[j]
        assert len(set(at)) == len(at)
        for j in range(n, k):
            assert tokens[a, j] == -1 and parents[a, j] == j and new[a, j] == -np.inf and over[a, j] == int(ended[a, j] != 0)


def exact_ties(got, logits, scores, ended, end):
    """The outputs are exactly the first of the sorted continuations."""
    g, k = scores.shape
    c = continuations(logits, scores, ended, end)
    for a in range(g):
        order = np.lexsort((np.arange(c[a].size), -c[a].reshape(-1)))[:k]
        order = [x for x in order if c[a].reshape(-1)[x] > -np.inf]
        want = [(int(x) // c.shape[2], int(x) % c.shape[2]) for x in order]
        have = [(int(got[1][a, j]), int(got[0][a, j])) for j in range(len(want))]
        assert have == want


def reorder(parents, tables, lens, arrays):
    """(tables, arrays) after; arrays: (pages, page, ...) caches and (pages,
    heads) exponents."""
    g, k = parents.shape
    out_t, out = tables.copy(), [x.copy() for x in arrays]
    page, pages = arrays[0].shape[1], arrays[0].shape[0]
    for a in range(g):
        length = min(max(int(lens[a * k]), 0), tables.shape[1] * page)
        full, tail = length // page, length % page
        for b in range(k):
            up = int(parents[a, b]) if 0 <= parents[a, b] < k else b
            me, src = a * k + b, a * k + up
            out_t[me, :full] = tables[src, :full]
            if tail and 0 <= tables[me, full] < pages and 0 <= tables[src, full] < pages:
                for x, y in zip(out, arrays):
                    if y.ndim == 4:
                        x[tables[me, full], :tail] = y[tables[src, full], :tail]
                    else:
                        x[tables[me, full]] = y[tables[src, full]]
    return out_t, out


def logits(rng, rows, vocab, t, std=3.0):
    return P.cast(rng.standard_normal((rows, vocab)) * std, t)
