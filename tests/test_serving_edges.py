"""Edges of the serving operators on the CPU."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T


@pytest.mark.parametrize("far", [30.0, 100.0, 1000.0])
def test_infinite_values_of_small_weight(far):
    q, k, v = np.ones((1, 2, 2, 1), np.float32), np.zeros((1, 2, 1, 1), np.float32), np.ones((1, 2, 1, 1), np.float32)
    k[0, 0], v[0, 0] = -far, np.inf
    assert (T.window_attention(q, k, v, scale=1.0) == np.inf).all()
    v[0, 0] = 3e38  # (a finite one by its weight: nothing at e^-1000)
    w = np.exp(-far)
    want = (w * 3e38 + 1) / (w + 1)
    assert np.allclose(T.window_attention(q, k, v, scale=1.0)[0, 1], want, rtol=2.0**-22, atol=0)
