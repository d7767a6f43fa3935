"""Beams whose tables name pages that the cache does not have."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T

import beams_plain as B
import fp8_plain as Q

BEYOND = [(-1, 10**6), (10**6, -1), (7, 2**31 - 1), (-2**31, 0), (None, 10**6), (10**6, None), (0, 0)]


def tables_beyond(rng, g, k, width, extra, past):
    """Tables (g * k, width) over their own pages; in every second row the last
    pages of a length of ``width`` - 1/2 pages and the first ones are no pages
    (entries from the number of pages on; 0: that number itself), a row's own,
    its parents' or both."""
    rows = g * k
    pages = rows * width + extra
    tables = rng.permutation(pages)[:rows * width].reshape(rows, width).astype(np.int32)
    parents = rng.integers(0, k, (g, k)).astype(np.int32)
    last, first = past
    if last is not None:
        tables[::2, -1] = pages if last == 0 else last
    if first is not None:
        tables[1::2, 0] = pages if first == 0 else first
        tables[1::2, -1] = tables[1::2, 0]
    return tables, parents, pages


def cache_arrays(rng, kind, pages, page, hkv, d):
    if kind == "fp8":
        (kc, ke), (vc, ve) = Q.random_cache(rng, pages, page, hkv, d), Q.random_cache(rng, pages, page, hkv, d)
        return [kc, vc, ke, ve]
    return [B.logits(rng, pages * page * hkv, d, kind).reshape(pages, page, hkv, d) for _ in range(2)]


@pytest.mark.parametrize("past", BEYOND)
@pytest.mark.parametrize("kind", ["fp8", "bf16", "f16", "f32"])
def test_reorder_of_no_pages(kind, past):
    """They are copied neither from nor to."""
    rng = np.random.default_rng(81)
    for g, k, page in ((2, 4, 16), (1, 7, 3)):
        tables, parents, pages = tables_beyond(rng, g, k, 3, 2, past)
        arrays = cache_arrays(rng, kind, pages, page, 2, 8)
        lens = np.full(g * k, 2 * page + page // 2, np.int32)
        t, want = B.reorder(parents, tables, lens, arrays)
        T.beam_reorder(parents, tables, lens, *arrays)
        assert (tables == t).all()
        for x, y in zip(arrays, want):
            assert x.tobytes() == y.tobytes()
