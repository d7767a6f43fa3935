"""Serving operators given arrays that make no sense: nothing outside the
tensors is read or written, and what is left whole keeps its result."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T

import serving_plain as P
from test_gpu_serving import close, draw, f_paged, run

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
