"""Calls over the same operands in one kernel: each is its own."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch.lower import lower

X = dict(logits=np.zeros((6, 40), np.float32), scores=np.zeros((2, 3), np.float32), ended=np.zeros((2, 3), np.int32))


def two_ends(logits, scores, ended):
    """Two of each call's results, none of them the same."""
    a = T.beam_select(logits, scores, ended, end_token=2)
    b = T.beam_select(logits, scores, ended, end_token=3)
    return a[0], a[2], b[1], b[3]


def many_ends(logits, scores, ended):
    return [T.beam_select(logits, scores, ended, end_token=i)[3] for i in (-1, 0, 7, 0)]


def draw(rng):
    """Logits whose largest are the tokens 2, 3 and 7 in turn, some beams ended."""
    x = rng.standard_normal((6, 40)).astype(np.float32)
    for r in range(6):
        x[r, [2, 3, 7][r % 3]] = 9
    ended = np.array([[0, 0, 1], [0, 0, 0]], np.int32)
    return x, -rng.random((2, 3)).astype(np.float32), ended


def test_calls_of_other_end_tokens_are_launches_of_their_own():
    assert lower(NKIPyKernel.trace(two_ends).specialize(**X)).kernel_kinds == ["beam_select"] * 2
    kinds = lower(NKIPyKernel.trace(many_ends).specialize(**X)).kernel_kinds
    assert kinds == ["beam_select"] * 4


def test_calls_of_other_sizes_are_launches_of_their_own():
    """Tables of one call are the next one's: the results are those of either."""

    def f(tables, lens, new):
        a = T.assign_pages(tables, lens, new, pages=9, page_size=4, tokens=7)
        b = T.assign_pages(tables, lens, new, pages=9, page_size=4, tokens=8)
        return a[1], b[1]

    kw = dict(tables=np.full((2, 3), -1, np.int32), lens=np.array([5, 3], np.int32), new=np.array([5, 3], np.int32))
    assert lower(NKIPyKernel.trace(f).specialize(**kw)).kernel_kinds == ["assign_pages"] * 2


def test_the_end_token_matters_here():
    x, scores, ended = draw(np.random.default_rng(91))
    with_2, with_3 = (T.beam_select(x, scores, ended, end_token=e)[3] for e in (2, 3))
    assert (with_2 != with_3).any()


@pytest.mark.gpu
@pytest.mark.parametrize("f", [two_ends, many_ends])
def test_calls_of_other_end_tokens(f):
    from test_gpu_serving import run

    x, scores, ended = draw(np.random.default_rng(91))
    want = f(x, scores, ended)
    got = run(f, x, scores, ended)
    for i, y in enumerate(want):
        if y.dtype == np.int32:
            assert (got[f"output{i}"] == y).all()
        else:  # (as test_gpu_beams.select_tolerance, and the CPU form's own rounding)
            assert np.abs(got[f"output{i}"] - y).max() <= 198 * 2.0**-23 + 2.0**-23 * np.abs(y).max()
