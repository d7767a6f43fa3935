"""Draws at the borders of their filters on the GPU."""

import numpy as np
import pytest

import serving_plain as P
from test_gpu_serving import f_sample, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1000, 20000])
def test_nucleus_that_ends_on_a_tie(t, vocab):
    """Ten equal logits and a share that whole numbers of them have exactly: the
    share given is the share kept, in 64 bits."""
    rng = np.random.default_rng(91)
    x = np.full((1, vocab), -np.inf, np.float32)
    at = np.sort(rng.permutation(vocab)[:10])
    x[0, at] = 1.5
    x = P.cast(x, t)
    u = np.array([1 - 2.0**-24], np.float32)  # (the last kept)
    for top_p in (0.1, 0.2, 0.3, 0.5, 0.6, 0.7, 0.8, 0.9):
        for top_k in (None, 10, 500):
            n = len(P.kept(P.up(x)[0], 1.0, top_k, top_p, None)[0])
            assert n == round(10 * top_p)
            assert run(f_sample, x, u, top_k=top_k, top_p=top_p)["output0"][0] == at[n - 1], (top_p, top_k)


def test_temperatures_below_32_bits():
    """The largest logits share the draw at any temperature above 0."""
    x = np.zeros((2, 50), np.float32)
    x[:, 10:20] = 1.0
    u = np.array([0.05, 0.95], np.float32)
    for temperature in (1e-3, 1e-38, 1e-45, 1e-60, 1e-300):
        assert list(f_sample(x, u, temperature)) == [10, 19]
        assert list(run(f_sample, x, u, temperature=temperature)["output0"]) == [10, 19], temperature
    for temperature in (1e38, 1e60, np.inf):
        assert list(f_sample(x, u, temperature)) == [2, 47]
        assert list(run(f_sample, x, u, temperature=temperature)["output0"]) == [2, 47], temperature


@pytest.mark.parametrize("vocab", [4000, 17001])
def test_rows_without_temperature(vocab):
    """A temperature of 0, below it or NaN takes the largest logit, the first of equal
    ones, whatever the filters of its row say."""
    rng = np.random.default_rng(92)
    x = (rng.standard_normal((6, vocab)) * 3).astype(np.float32)
    x[2, [70, 3000]] = 50.0
    x[3, :5] = np.nan
    x[4] = -np.inf
    temp = np.array([0, np.nan, 0, -1, 0, 0.0], np.float32)
    k = np.array([5, 7, 0, -3, 1, 900], np.int32)
    p = np.array([0.5, 0.3, 1.0, 0.1, 0.2, np.nan], np.float32)
    m = np.array([0, np.nan, 0.5, 0, 0, 1], np.float32)
    u = np.full(6, 0.999, np.float32)
    want = [int(np.nanargmax(r)) if (r > -np.inf).any() else -1 for r in x]
    assert want[2] == 70 and want[4] == -1
    assert list(run(f_sample, x, u, temp, k, p, m)["output0"]) == want
    assert list(f_sample(x, u, temp, k, p, m)) == want
