"""The generation loop's operators on the GPU against plain forms."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T

import beams_plain as B
import fp8_plain as Q
import serving_plain as P
from test_gpu_serving import load, run

pytestmark = pytest.mark.gpu


def f_assign(block_tables, context_lens, new_lens, pages=9, page_size=4, tokens=7):
    return T.assign_pages(block_tables, context_lens, new_lens, pages=pages, page_size=page_size, tokens=tokens)


def f_select(logits, scores, ended, end_token=2):
    return T.beam_select(logits, scores, ended, end_token=end_token)


def f_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps=None, value_exps=None):
    T.beam_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps, value_exps)


# ---------------------------------------------------------------------------
# Tables
# ---------------------------------------------------------------------------
def check_assign(tables, lens, new, pages, page, tokens):
    lens, new = np.asarray(lens, np.int32), np.asarray(new, np.int32)
    t, starts, slots, free = B.assign(tables, lens, new, pages, page, tokens)
    got = run(f_assign, tables, lens, new, pages=pages, page_size=page, tokens=tokens)
    assert (got["block_tables"] == t).all()
    assert (got["output0"] == starts).all()
    if tokens:
        assert (got["output1"] == slots).all()
    assert (got["output2"] == free).all()


def test_assign_small():
    rng = np.random.default_rng(1)
    tables = rng.permutation(60)[:40].reshape(5, 8).astype(np.int32)
    check_assign(tables.copy(), [9, 0, 30, 17, 32], [1, 0, 12, 17, 3], 60, 4, 40)
    check_assign(tables.copy(), [9, 0, 30, 17, 32], [1, 0, 12, 17, 3], 42, 4, 20)
    check_assign(tables.copy(), [9, 5, 30, 100, -3], [20, 5, -2, 90, 4], 60, 4, 200)
    tables[0, :2] = [-1, 70]
    check_assign(tables.copy(), [9, 8, 30, 17, 32], [1, 0, 12, 17, 3], 60, 4, 33)
    tables[2] = tables[4]
    check_assign(tables.copy(), [9, 8, 30, 17, 32], [1, 0, 2, 17, 3], 60, 4, 33)
    check_assign(np.zeros((1, 1), np.int32), [1], [1], 1, 1, 1)
    check_assign(np.zeros((1, 1), np.int32), [0], [0], 33, 1, 0)


@pytest.mark.parametrize("rows,page,pages,most,new", [(64, 16, 5000, 1000, 1), (1, 16, 200, 3000, 2900), (200, 1, 9000, 40, 3),
                                                      (1500, 8, 40000, 150, 2), (30, 24, 900, 600, 300), (70, 128, 2**20, 4000, 0),
                                                      (3000, 16, 3000, 30, 1), (2**16, 16, 2**20, 40, 1), (64, 16, 40000, 8000, 3),
                                                      (65, 16, 40000, 8000, 3), (7, 16, 20000, 40000, 100)])
def test_assign_batches(rows, page, pages, most, new):
    """Rows of many lengths, some ended, some without new tokens; more pages
    wanted than there are."""
    rng = np.random.default_rng(rows)
    lens = rng.integers(1, most + 1, rows)
    n = np.minimum(rng.integers(0, 2 * new + 1, rows), lens)
    lens[rng.random(rows) < 0.1] = 0
    n = np.minimum(n, lens)
    width = -(-most // page) + 1
    tables = np.full((rows, width), -1, np.int32)
    held = -(-(lens - n) // page)
    ids, at = rng.permutation(pages), 0
    for b in range(rows):
        k = min(int(held[b]), max(pages - at, 0))
        tables[b, :k] = ids[at:at + k]
        at += k
    tables[:, -1] = 12345  # (old entries)
    check_assign(tables, lens, n, pages, page, int(n.sum()) + 5)


# ---------------------------------------------------------------------------
# The choice of beams
# ---------------------------------------------------------------------------
def select_tolerance(x, vocab):
    """Of a log sum: terms 2^t with t rounded at up to 2^-23 of itself (two
    roundings, one of the constant) and |t| of up to 150 where a term counts, an
    instruction's ulp, and a running sum of 32 and 64 terms: each within 2^-23 of
    its own, so the sum within (150 + 1 + 7 + 40) 2^-23 of itself; the score is
    rounded behind the comparison."""
    return (150 + 1 + 7 + 40) * 2.0**-23


def check_select(x, scores, ended, end):
    got = run(f_select, x, scores, ended, end_token=end)
    got = [got[f"output{j}"] for j in range(4)]
    B.check_select(got, x, scores, ended, end, select_tolerance(x, x.shape[1]))
    return got


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("g,k,vocab", [(1, 1, 1), (1, 4, 3), (3, 4, 50), (2, 32, 40), (1, 4, 32000), (2, 3, 2047), (5, 8, 8193),
                                       (2, 5, 8191), (1, 2, 16385), (3, 16, 50257), (1, 32, 20000), (33, 2, 1000), (2, 25, 90000),
                                       (1, 7, 300000), (1, 2, 2**22), (1, 32, 2**18), (4000, 2, 5)])
def test_select(t, g, k, vocab):
    rng = np.random.default_rng(vocab)
    x, scores = B.logits(rng, g * k, vocab, t), (-5 - 3 * rng.random((g, k))).astype(np.float32)
    ended = (rng.random((g, k)) < 0.3).astype(np.int32)
    check_select(x, scores, 0 * ended, 0)
    check_select(x, scores, ended, vocab - 1)
    scores[:, 1:] = -np.inf  # the first step: one beam
    check_select(x, scores, 0 * ended, -1)


def test_select_special_values():
    rng = np.random.default_rng(3)
    for vocab in (20, 9000):
        x = rng.standard_normal((12, vocab)).astype(np.float32)
        x[0] = np.nan
        x[1] = -np.inf
        x[2, 3:6] = np.inf
        x[3, ::2] = np.nan
        x[4] = 1.0
        x[9] = -3e38
        x[9, 7] = 3e38
        x[10] = -1e30
        scores = np.array([[-1, -2, -3, -4], [-1, np.nan, -np.inf, -1], [-2, -2, -2, -2]], np.float32)
        ended = np.array([[0, 0, 0, 0], [0, 0, 1, 0], [1, 0, 0, 0]], np.int32)
        check_select(x, scores, ended, 4)
        got = run(f_select, x[:4], np.full((1, 4), -np.inf, np.float32), ended[:1], end_token=4)
        assert (got["output0"] == -1).all() and (got["output1"] == [0, 1, 2, 3]).all() and (got["output2"] == -np.inf).all()


@pytest.mark.parametrize("k,vocab", [(4, 20), (8, 9000), (32, 40000), (32, 70000), (1, 2500)])
def test_select_ties(k, vocab):
    """Equal logits, whole rows of them: the lower beam, then the lower token."""
    x = np.zeros((2 * k, vocab), np.float32)
    x[:, vocab // 2:vocab // 2 + 3] = 2.0
    scores, ended = np.zeros((2, k), np.float32), np.zeros((2, k), np.int32)
    got = run(f_select, x, scores, ended, end_token=1)
    B.exact_ties([got[f"output{j}"] for j in range(4)], x, scores, ended, 1)
    x[:] = 0
    got = run(f_select, x, scores, ended, end_token=1)
    B.exact_ties([got[f"output{j}"] for j in range(4)], x, scores, ended, 1)


def test_select_ended_beams_are_not_read():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((8, 3000)).astype(np.float32)
    x[[1, 6]] = np.nan
    scores = -rng.random((2, 4)).astype(np.float32)
    ended = np.array([[0, 1, 0, 0], [0, 0, 7, 0]], np.int32)
    got = check_select(x, scores, ended, 9)
    assert (got[1][0, 0] == 1 or scores[0, 1] < 0) and got[3].max() == 1
    every = np.ones((2, 4), np.int32)
    got = check_select(x, scores, every, -1)
    assert (got[0] == -1).all() and (got[2] == -np.sort(-scores, axis=1)).all()


def test_select_strided_rows():
    """Rows apart and at odd addresses."""
    rng = np.random.default_rng(6)
    for t, cut in (("bf16", 3), ("f32", 1), ("bf16", 8)):
        big = B.logits(rng, 6, 9100, t)

        def f(big, scores, ended):
            return T.beam_select(big[:, cut:], scores, ended, end_token=0)

        scores, ended = -rng.random((2, 3)).astype(np.float32), np.zeros((2, 3), np.int32)
        got = run(f, big, scores, ended)
        B.check_select([got[f"output{j}"] for j in range(4)], big[:, cut:], scores, ended, 0, select_tolerance(big, 9100))


# ---------------------------------------------------------------------------
# Caches behind their parents
# ---------------------------------------------------------------------------
def check_reorder(rng, kind, g, k, page, hkv, d, lens, width):
    rows = g * k
    pages = rows * width + 3
    tables = rng.permutation(pages)[:rows * width].reshape(rows, width).astype(np.int32)
    tables[rng.random(tables.shape) < 0.05] = -1
    parents = rng.integers(-1, k + 1, (g, k)).astype(np.int32)
    lens = np.repeat(np.asarray(lens, np.int32), k)
    if kind == "fp8":
        (kc, ke), (vc, ve) = Q.random_cache(rng, pages, page, hkv, d), Q.random_cache(rng, pages, page, hkv, d)
        arrays = [kc, vc, ke, ve]
    else:
        arrays = [B.logits(rng, pages * page * hkv, d, kind).reshape(pages, page, hkv, d) for _ in range(2)]
    t, want = B.reorder(parents, tables, lens, arrays)
    got = run(f_reorder, parents, tables, lens, *arrays)
    assert (got["block_tables"] == t).all()
    for name, x in zip(("key_cache", "value_cache", "key_exps", "value_exps"), want):
        assert got[name].tobytes() == x.tobytes(), name


@pytest.mark.parametrize("kind", ["fp8", "bf16", "f16", "f32"])
@pytest.mark.parametrize("g,k", [(1, 1), (1, 4), (3, 5), (2, 8), (2, 9), (1, 32)])
def test_reorder(kind, g, k):
    rng = np.random.default_rng(7)
    check_reorder(rng, kind, g, k, 16, 2, 64, [37, 64, 5][:g], 4)
    check_reorder(rng, kind, g, k, 3, 1, 5, [0, 8, 100][:g], 3)


def test_reorder_long_tables_and_large_pages():
    rng = np.random.default_rng(8)
    check_reorder(rng, "fp8", 2, 4, 1, 1, 16, [700, 531], 701)
    check_reorder(rng, "bf16", 2, 4, 200, 2, 128, [399, 1], 2)
    check_reorder(rng, "fp8", 1, 7, 64, 300, 16, [63], 1)


def test_reorder_of_one_array_as_both_caches():
    """Keys and values in the same memory: both results are the same."""
    from nkipy_amd.runtime import DeviceTensor

    rng = np.random.default_rng(9)
    tables = rng.permutation(12).reshape(6, 2).astype(np.int32)
    parents, lens = np.array([[2, 0, 0], [1, 1, 2]], np.int32), np.full(6, 21, np.int32)
    cache = B.logits(rng, 12 * 16, 64, "bf16").reshape(12, 16, 1, 64)
    t, (want, _) = B.reorder(parents, tables, lens, [cache, cache])
    both = DeviceTensor.from_numpy(cache)
    dk, ins, outs = load(f_reorder, parents, tables, lens, both, both)
    for graph in (False, True, True):
        both.write_from_numpy(cache)
        outs["block_tables"].write_from_numpy(tables)
        dk(ins, outs, graph=graph)
        assert (outs["block_tables"].numpy() == t).all()
        assert both.numpy().tobytes() == want.tobytes()


def test_two_sets_of_tensors_replayed_in_turns():
    """Two graphs of one kernel share its workspace."""
    rng = np.random.default_rng(10)
    dk, sets = None, []
    for _ in range(2):
        x = B.logits(rng, 12, 20000, "bf16")
        scores, ended = -rng.random((3, 4)).astype(np.float32), (rng.random((3, 4)) < 0.2).astype(np.int32)
        one, ins, outs = load(f_select, x, scores, ended, end_token=2)
        dk = dk or one
        sets.append((ins, outs, (x, scores, ended)))
    for _ in range(3):
        for ins, outs, _ in sets:
            dk(ins, outs, graph=True, sync=False)
        for ins, outs, (x, scores, ended) in sets:
            B.check_select([outs[f"output{j}"].numpy() for j in range(4)], x, scores, ended, 2, select_tolerance(x, 20000))
