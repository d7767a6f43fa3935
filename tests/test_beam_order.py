"""The order of a beam choice: equal logits, and beams that have ended."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T

import beams_plain as B
import serving_plain as P


def check_order(got, x, scores, ended, end):
    """The tokens chosen of one parent are its first by the largest logit and,
    of equal ones, by the lowest token, in that order; scores do not rise.  The
    same score by the same sum: no tolerance."""
    tokens, parents, new, over = (np.asarray(y) for y in got)
    g, k = scores.shape
    x = P.up(x).reshape(g, k, -1)
    for a in range(g):
        assert (np.diff(new[a]) <= 0).all()
        for b in range(k):
            mine = [int(t) for t, p in zip(tokens[a], parents[a]) if p == b and t >= 0]
            if ended[a, b]:
                assert mine in ([], [end])
                continue
            z = np.where(np.isnan(x[a, b]), -np.inf, x[a, b])
            assert mine == np.argsort(-z, kind="stable")[:len(mine)].tolist(), (a, b, mine)


def draw_ties(rng, g, k, vocab, t):
    """Logits of a few whole values, so that every place of the choice is among
    equal ones, and beams whose scores are whole numbers apart."""
    x = P.cast(rng.integers(-3, 3, (g * k, vocab)), t)
    scores = -rng.permutation(g * k).reshape(g, k).astype(np.float32) / 4
    ended = (rng.random((g, k)) < 0.3).astype(np.int32)
    return x, scores, ended


SIZES = [(1, 4, 40), (3, 8, 500), (2, 32, 900), (1, 1, 3000), (2, 5, 9000), (4, 16, 20000)]


@pytest.mark.parametrize("g,k,vocab", SIZES[:3])
def test_equal_logits_cpu(g, k, vocab):
    x, scores, ended = draw_ties(np.random.default_rng(101), g, k, vocab, "f32")
    check_order(T.beam_select(x, scores, ended, end_token=5), x, scores, ended, 5)
    check_order(T.beam_select(x, scores, 0 * ended, end_token=5), x, scores, 0 * ended, 5)


def test_wrong_orders_are_noticed():
    """The check itself: a higher token in place of an equal lower one, last or
    first, and two equal ones the wrong way round."""
    x, scores, ended = draw_ties(np.random.default_rng(102), 1, 8, 300, "f32")
    good = [y.copy() for y in T.beam_select(x, scores, 0 * ended, end_token=5)]
    check_order(good, x, scores, 0 * ended, 5)
    b = int(good[1][0, -1])  # the last one's parent
    z = P.up(x).reshape(1, 8, -1)[0, b]
    last = good[0][0, -1]
    higher = [t for t in np.flatnonzero(z == z[last]) if t > last]
    wrong = [y.copy() for y in good]
    wrong[0][0, -1] = higher[0]
    with pytest.raises(AssertionError):
        check_order(wrong, x, scores, 0 * ended, 5)
    of = np.flatnonzero(good[1][0] == good[1][0, 0])[:2]
    wrong = [y.copy() for y in good]
    wrong[0][0, of] = wrong[0][0, of[::-1]]
    with pytest.raises(AssertionError):
        check_order(wrong, x, scores, 0 * ended, 5)


def ended_case():
    """An ended beam in each place of the order: its score between those of the
    others' best continuations."""
    x = np.full((3 * 4, 50), -20, np.float32)
    x[:, 7] = 20  # (one continuation of each other beam weighs about 1)
    ended = np.zeros((3, 4), np.int32)
    scores = np.array([[-3, -1, -2, -4], [-1, -5, -2, -4], [-1, -2, -3, -2.5]], np.float32)
    ended[0, 1], ended[1, 2], ended[2, 2] = 1, 5, -1
    parents = [[1, 2, 0, 3], [0, 2, 3, 1], [0, 1, 3, 2]]
    return x, scores, ended, np.array(parents)


def check_ended(got, scores, ended, parents, end):
    assert (got[1] == parents).all()
    over = np.take_along_axis(ended, parents, 1) != 0
    assert (got[0] == np.where(over, end, 7)).all()
    assert (got[3] == (over | (got[0] == end))).all()
    assert (np.asarray(got[2])[over] == np.take_along_axis(scores, parents, 1)[over]).all()


@pytest.mark.parametrize("end", [-1, 0, 7, 49])
def test_ended_beams_stand_in_their_place_cpu(end):
    x, scores, ended, parents = ended_case()
    check_ended(T.beam_select(x, scores, ended, end_token=end), scores, ended, parents, end)


@pytest.mark.gpu
@pytest.mark.parametrize("end", [-1, 0, 7, 49])
def test_ended_beams_stand_in_their_place(end):
    from test_gpu_beam_sums import select

    x, scores, ended, parents = ended_case()
    check_ended(select(x, scores, ended, end), scores, ended, parents, end)


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("g,k,vocab", SIZES)
def test_equal_logits(t, g, k, vocab):
    from test_gpu_beam_sums import select

    x, scores, ended = draw_ties(np.random.default_rng(103), g, k, vocab, t)
    for e in (0 * ended, ended):
        check_order(select(x, scores, e, 5), x, scores, e, 5)
    x = B.logits(np.random.default_rng(104), g * k, vocab, t)
    check_order(select(x, scores, ended, 5), x, scores, ended, 5)
