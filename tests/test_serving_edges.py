"""Edges of the serving operators on the CPU."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel


@pytest.mark.parametrize("far", [30.0, 100.0, 1000.0])
def test_infinite_values_of_small_weight(far):
    q, k, v = np.ones((1, 2, 2, 1), np.float32), np.zeros((1, 2, 1, 1), np.float32), np.ones((1, 2, 1, 1), np.float32)
    k[0, 0], v[0, 0] = -far, np.inf
    assert (T.window_attention(q, k, v, scale=1.0) == np.inf).all()
    v[0, 0] = 3e38  # (a finite one by its weight: nothing at e^-1000)
    w = np.exp(-far)
    want = (w * 3e38 + 1) / (w + 1)
    assert np.allclose(T.window_attention(q, k, v, scale=1.0)[0, 1], want, rtol=2.0**-22, atol=0)


def _append(kc, vc, q, k, cos, tables, lens):
    return T.rotary_append(q, k, k, cos, cos, kc, vc, tables, lens)


ARGS = dict(q=np.zeros((2, 4, 8), np.float32), k=np.zeros((2, 2, 8), np.float32), cos=np.zeros((9, 4), np.float32),
            tables=np.zeros((2, 3), np.int32), lens=np.zeros(2, np.int32))


def test_append_refuses_parts_of_arguments():
    """A traced slice or reshape is an array of its own, so a write into one would not
    reach the argument; on the CPU it does."""
    c = np.zeros((2, 5, 4, 2, 8), np.float32)
    whole = np.zeros((5, 4, 2, 8), np.float32)

    def parts(c, **a):
        return _append(c[0], c[1], **a)

    def shapes(c, d, **a):
        return _append(c, d.reshape(5, 4, 2, 8), **a)

    def turned(c, d, **a):
        return _append(c.transpose(1, 0, 2, 3), d, **a)

    def after_a_write(c, **a):
        c[0, 0, 0] = 1.0
        return _append(c[0], c[1], **a)

    for f, args, name in ((parts, (c,), "key_cache"), (shapes, (whole, whole.reshape(20, 2, 8)), "value_cache"),
                          (turned, (np.zeros((4, 5, 2, 8), np.float32), whole), "key_cache"), (after_a_write, (c,), "key_cache")):
        with pytest.raises(ValueError, match=f"{name}.*would not reach"):
            NKIPyKernel.trace(f).specialize(*args, **ARGS)
    a = dict(ARGS, lens=np.ones(2, np.int32), tables=np.array([[1, 0, 0], [3, 0, 0]], np.int32), k=ARGS["k"] + 2,
             cos=np.ones((9, 4), np.float32))
    parts(c, **a)
    assert (c[1, 1, 0] == 2).all() and (c[1, 3, 0] == 2).all() and c[1].sum() == 2 * 2 * 2 * 8

    def of_their_own(c, **a):  # arrays that the kernel makes
        return _append(c[0] + 0, np.copy(c[1]), **a)

    NKIPyKernel.trace(of_their_own).specialize(c, **ARGS)
    NKIPyKernel.trace(_append).specialize(whole, whole.copy(), **ARGS)
