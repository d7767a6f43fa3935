"""Beams whose tables name pages that the cache does not have, on the GPU."""

import numpy as np
import pytest

import beams_plain as B
from test_beam_pages import BEYOND, cache_arrays, tables_beyond
from test_gpu_beams import f_reorder
from test_gpu_serving import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("past", BEYOND)
@pytest.mark.parametrize("kind", ["fp8", "bf16", "f16", "f32"])
def test_reorder_of_no_pages(kind, past):
    """Bit for bit what the plain form leaves, in every array."""
    rng = np.random.default_rng(81)
    for g, k, page, d in ((2, 4, 16, 64), (1, 7, 3, 8), (1, 32, 16, 5), (3, 8, 5, 16)):
        tables, parents, pages = tables_beyond(rng, g, k, 3, 2, past)
        arrays = cache_arrays(rng, kind, pages, page, 2, d)
        lens = np.full(g * k, 2 * page + page // 2, np.int32)
        t, want = B.reorder(parents, tables, lens, arrays)
        got = run(f_reorder, parents, tables, lens, *arrays)
        assert (got["block_tables"] == t).all()
        for name, x in zip(("key_cache", "value_cache", "key_exps", "value_exps"), want):
            assert got[name].tobytes() == x.tobytes(), name
