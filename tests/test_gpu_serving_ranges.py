"""Attention at the ends of 32 bits on the GPU: scores of any finite size."""

import numpy as np
import pytest

import serving_plain as P
from test_gpu_serving import close, draw, f_paged, f_window, run

pytestmark = pytest.mark.gpu


# (type, head dim, q, k, scale): each score is -|q k| d scale, a power of two or a few
# bits more, so that sums of the products are exact in any order.  The last of each
# type: a score that is in range and its product with log2 e that is not.
LOW = [("bf16", 64, 2.0**46, 2.0**46, 0.125), ("bf16", 64, 2.0**48, 2.0**48, 0.125), ("bf16", 64, 2.0**49, 2.0**48, 0.125),
       ("bf16", 64, 2.0**55, 2.0**55, 0.125), ("bf16", 64, 2.0**60, 2.0**60, 2.0**-64),
       ("bf16", 64, 1.75 * 2.0**60, 1.75 * 2.0**60, 1.0),
       ("bf16", 128, 2.0**50, 2.0**50, 0.125), ("bf16", 128, 1.75 * 2.0**59, 1.75 * 2.0**60, 1.0),
       ("f16", 64, 2.0**15, 2.0**15, 2.0**63), ("f16", 128, 2.0**15, 2.0**15, 2.0**64),
       ("f32", 48, 2.0**55, 2.0**55, 0.125)]


@pytest.mark.parametrize("t,d,big_q,big_k,scale", LOW)
@pytest.mark.parametrize("S", [1, 40, 130])
@pytest.mark.parametrize("K", [130, 3000])
def test_window_lowest_scores(t, d, big_q, big_k, scale, S, K):
    """Scores far below 0 alone: the largest has all the weight, equal ones share it,
    also where a row's keys lie in several splits."""
    rng = np.random.default_rng(81)
    v = P.cast(rng.integers(-8, 8, (2, K, 2, d)).astype(np.float32), t)
    q, k = np.full((2, S, 4, d), -big_q, np.float32), np.full((2, K, 2, d), big_k, np.float32)
    k[0, 70] /= 2  # (every query sees it where S < 60)
    q, k = P.cast(q, t), P.cast(k, t)
    want, tol = P.dense(q, k, v, None, None, 0, 0, t, scale)
    # among equal scores: at most 8, by the roundings of weights, sums and result
    close(run(f_window, q, k, v, scale=scale)["output0"], want, np.minimum(tol, 8 * 4 * 2.0**-8))


@pytest.mark.parametrize("new", [None, [40, 300]])
def test_paged_lowest_scores(new):
    rng = np.random.default_rng(82)
    tables, lens, starts, pages = P.batch(rng, [2500, 700], new, 16)
    tables[0, 3] = -1
    n = 2 if new is None else sum(new)
    q = P.cast(np.full((n, 4, 128), -2.0**52, np.float32), "bf16")
    kc = P.cast(np.full((pages, 16, 2, 128), 2.0**52, np.float32), "bf16")
    kc[tables[0, 1], 5] = P.cast(np.float32(2.0**51), "bf16")
    vc = P.cast(rng.integers(-8, 8, kc.shape).astype(np.float32), "bf16")
    for window, sinks in ((0, 0), (500, 3)):
        want, tol = P.paged(q, kc, vc, tables, lens, starts, window, sinks, "bf16")
        got = run(f_paged, q, kc, vc, tables, lens, starts, window=window or None, sinks=sinks)["output0"]
        close(got, want, np.minimum(tol, 8 * 4 * 2.0**-8))


def test_only_scores_of_minus_infinity():
    """Rows whose keys are all -inf, beside rows with one that is not."""
    rng = np.random.default_rng(83)
    for S, K in ((1, 3000), (70, 90)):
        q, v = np.abs(P.up(draw(rng, (2, S, 4, 64), "bf16"))) + 1, draw(rng, (2, K, 2, 64), "bf16")
        k = np.full((2, K, 2, 64), -np.inf, np.float32)
        k[1, 11] = 1.0
        q, k = P.cast(q, "bf16"), P.cast(k, "bf16")
        got = P.up(run(f_window, q, k, v)["output0"])
        assert (got[0] == 0).all()
        first = max(0, 11 - (K - S))  # (the query at position 11)
        assert (got[1, :first] == 0).all() and (got[1, first:] == np.repeat(P.up(v)[1, 11], 2, 0)).all()


@pytest.mark.parametrize("t,d,far", [("bf16", 64, 60.0), ("bf16", 128, 95.0), ("f16", 64, 30.0), ("f16", 128, 60.0), ("f32", 48, 95.0)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("S,K", [(1, 130), (1, 3000), (40, 300)])
def test_infinite_values_of_small_weight(t, d, far, value, S, K):
    """A value that is not finite reaches each query that sees its key, also where the
    weight e^-far is nothing in the operands' type, and no other element."""
    rng = np.random.default_rng(84)
    q, k = np.zeros((2, S, 4, d), np.float32), np.zeros((2, K, 2, d), np.float32)
    q[..., 0], k[..., 0] = 1.0, rng.random((2, K, 2)) * 0.5
    at = K - S - 5  # (seen by all)
    k[0, at, 1, 0] = -far
    v = rng.standard_normal((2, K, 2, d)).astype(np.float32)
    q, k, v = P.cast(q, t), P.cast(k, t), P.cast(v, t)
    clean = v.copy()
    clean[0, at, 1, 7] = P.cast(np.float32(0), t)
    v[0, at, 1, 7] = P.cast(np.float32(value), t)
    want, tol = P.dense(q, k, clean, None, None, 0, 0, t, 1.0)
    got = P.up(run(f_window, q, k, v, scale=1.0)["output0"])
    hit = np.zeros(got.shape, bool)
    hit[0, :, 2:, 7] = True
    assert np.isnan(got[hit]).all() if np.isnan(value) else (got[hit] == value).all()
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("hq,hkv", [(4, 2), (40, 1)])
def test_paged_infinite_values_of_small_weight(hq, hkv):
    rng = np.random.default_rng(85)
    tables, lens, _, pages = P.batch(rng, [2500, 40, 300], None, 16)
    q, kc = np.zeros((3, hq, 64), np.float32), np.zeros((pages, 16, hkv, 64), np.float32)
    q[..., 0], kc[..., 0] = 1.0, rng.random((pages, 16, hkv)) * 0.5
    q[:, 0, 0] = 2.0
    kc[tables[0, 70], 3, 0, 0] = -30.0
    kc[tables[2, 18], 11, 0, 0] = -30.0
    q, kc, vc = P.cast(q, "f16"), P.cast(kc, "f16"), draw(rng, kc.shape, "f16")
    clean = vc.copy()
    clean[tables[0, 70], 3, 0, 5] = clean[tables[2, 18], 11, 0, 60] = 0
    vc[tables[0, 70], 3, 0, 5], vc[tables[2, 18], 11, 0, 60] = np.inf, -np.inf
    want, tol = P.paged(q, kc, clean, tables, lens, None, 0, 0, "f16", 1.0)
    got = P.up(run(f_paged, q, kc, vc, tables, lens, scale=1.0)["output0"])
    hit = np.zeros(got.shape, bool)
    hit[0, :hq // hkv, 5] = hit[2, :hq // hkv, 60] = True
    assert (got[0, :hq // hkv, 5] == np.inf).all() and (got[2, :hq // hkv, 60] == -np.inf).all()
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("S,K", [(1, 130), (1, 3000), (40, 300)])
@pytest.mark.parametrize("t,d", [("bf16", 64), ("f16", 128), ("f32", 48)])
def test_scores_that_are_no_number(t, d, S, K):
    """A NaN query, and a NaN key, make the rows that meet them NaN, whole, and no other."""
    rng = np.random.default_rng(86)
    q, k, v = draw(rng, (3, S, 4, d), t), draw(rng, (3, K, 2, d), t), draw(rng, (3, K, 2, d), t)
    want, tol = P.dense(q, k, v, None, None, 0, 0, t)
    q[0, S - 1, 2, 3] = P.cast(np.float32(np.nan), t)
    k[1, K - 1, 0, 5] = P.cast(np.float32(np.nan), t)
    v[0, 2, 1, 9] = P.cast(np.float32(np.inf), t)  # (seen by the NaN query as well)
    hit = np.zeros(want.shape, bool)
    hit[0, S - 1, 2] = hit[1, S - 1, :2] = True
    got = P.up(run(f_window, q, k, v)["output0"])
    assert np.isnan(got[hit]).all()
    inf = np.zeros(want.shape, bool)
    inf[0, :, 2:, 9] = True
    inf &= ~hit
    assert (got[inf] == np.inf).all()
    assert (np.abs(got - want)[~hit & ~inf] <= tol[~hit & ~inf]).all()
