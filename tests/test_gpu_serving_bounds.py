"""Serving operators given arrays that make no sense: nothing outside the
tensors is read or written, and what is left whole keeps its result."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T

import serving_plain as P
from test_gpu_serving import close, draw, f_paged, run
from test_serving_layouts import values_alone

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 48])
def test_long_batches_of_unordered_starts(d):
    """Starts that decrease over batches of many tiles: sequences that lie in order
    at the end of the batch are right all the same."""
    rng = np.random.default_rng(71)
    tables, lens, _, pages = P.batch(rng, [100, 100, 100, 330], [1, 1, 1, 300], 16)
    q = draw(rng, (1000, 8, d), "bf16")
    kc, vc = draw(rng, (pages, 16, 4, d), "bf16"), draw(rng, (pages, 16, 4, d), "bf16")
    for first in ([0, 700, 0], [700, 0, 0], [650, 3, 690], [2**31 - 1, -2**31, 0]):
        starts = np.array(first + [700, 1000], np.int32)
        got = P.up(run(f_paged, q, kc, vc, tables, lens, starts, window=40, sinks=1)["output0"])
        last = P.paged(q[700:], kc, vc, tables[3:], lens[3:], np.array([0, 300], np.int32), 40, 1, "bf16")
        if first[0] <= 700 and first[1] <= 700:  # (each tile behind row 700 finds its sequence)
            close(P.cast(got[700:], "f32"), *last)


@pytest.mark.parametrize("new", [None, [9, 40]])
def test_caches_whose_pages_are_one(new):
    rng = np.random.default_rng(72)
    tables, lens, starts, pages = P.batch(rng, [70, 45], new, 16)
    q = draw(rng, (2 if new is None else sum(new), 4, 64), "bf16")
    k, v = draw(rng, (1, 16, 2, 64), "bf16"), draw(rng, (1, 16, 2, 64), "bf16")
    shape = (pages, 16, 2, 64)
    f = lambda q, k, v, tables, lens, starts=None: T.paged_attention(  # noqa: E731
        q, np.broadcast_to(k, shape), np.broadcast_to(v, shape), tables, lens, starts)
    kc, vc = (np.ascontiguousarray(np.broadcast_to(x, shape)) for x in (k, v))
    close(run(f, q, k, v, tables, lens, starts)["output0"], *P.paged(q, kc, vc, tables, lens, starts, 0, 0, "bf16"))


@pytest.mark.parametrize("new", [None, [3, 9, 1]])
def test_values_written_alone(new):
    """Tokens whose position has no row in the tables are dropped also where the
    value cache is all that is written."""
    rng = np.random.default_rng(73)
    tables, lens, starts, pages = P.batch(rng, [12, 20, 14], new, 4)
    n = 3 if new is None else sum(new)
    q, k, v = (draw(rng, (n, h, 64), "f32") for h in (4, 2, 2))
    vc = draw(rng, (pages, 4, 2, 64), "f32")
    ang = np.arange(13 * 32, dtype=np.float32).reshape(13, 32)  # positions 0 to 12
    cos, sin = np.cos(ang), np.sin(ang)
    want = P.append(q, k, v, cos, sin, vc, vc, tables, lens, starts, "f32")[0][2]
    got = run(values_alone, q, k, v, cos, sin, vc, tables, lens, starts)
    assert (got["vc"] == want).all()
