"""The generation loop's operators on the CPU: their NumPy forms against plain
ones, what they refuse, and what they lower to."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch import beams as D
from nkipy_amd.dispatch.launchers import LaunchError
from nkipy_amd.dispatch.lower import lower

import beams_plain as B
import fp8_plain as Q


def check_assign(tables, lens, new, pages, page, tokens):
    t, starts, slots, free = B.assign(tables, np.asarray(lens), np.asarray(new), pages, page, tokens)
    got = T.assign_pages(tables, np.asarray(lens), np.asarray(new), pages=pages, page_size=page, tokens=tokens)
    assert (tables == t).all()
    for x, y in zip(got, (starts, slots, free)):
        assert x.dtype == np.int32 and x.shape == y.shape and (x == y).all()


def test_assign_cpu():
    rng = np.random.default_rng(1)
    tables = rng.permutation(60)[:40].reshape(5, 8).astype(np.int32)
    check_assign(tables.copy(), [9, 0, 30, 17, 32], [1, 0, 12, 17, 3], 60, 4, 40)
    check_assign(tables.copy(), [9, 0, 30, 17, 32], [1, 0, 12, 17, 3], 42, 4, 20)  # too few pages, too few rows
    check_assign(tables.copy(), [9, 5, 30, 100, -3], [20, 5, -2, 90, 4], 60, 4, 200)  # past the table, before 0
    tables[0, :2] = [-1, 70]  # held pages that are none
    check_assign(tables.copy(), [9, 8, 30, 17, 32], [1, 0, 12, 17, 3], 60, 4, 33)
    tables[2] = tables[4]  # shared pages
    check_assign(tables.copy(), [9, 8, 30, 17, 32], [1, 0, 2, 17, 3], 60, 4, 33)
    check_assign(np.zeros((1, 1), np.int32), [1], [1], 1, 1, 1)


def test_assign_gives_pages_back():
    tables = np.full((2, 4), -1, np.int32)
    for step, (lens, new, held) in enumerate([([5, 3], [5, 3], 3), ([6, 4], [1, 1], 3), ([0, 5], [0, 1], 2), ([9, 6], [9, 1], 5)]):
        _, _, free = T.assign_pages(tables, np.array(lens), np.array(new), pages=8, page_size=4, tokens=16)
        assert free[0] == 8 - held, step
        mine = tables[tables >= 0]
        assert len(mine) == held == len(set(mine.tolist()))


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("g,k,vocab", [(1, 1, 1), (1, 4, 3), (3, 4, 50), (2, 32, 40), (2, 3, 700)])
def test_select_cpu(t, g, k, vocab):
    rng = np.random.default_rng(2)
    x, scores = B.logits(rng, g * k, vocab, t), (-5 - 3 * rng.random((g, k))).astype(np.float32)
    ended = (rng.random((g, k)) < 0.3).astype(np.int32)
    for e, end in [(0 * ended, 0), (ended, vocab - 1), (ended, -1)]:
        B.check_select(T.beam_select(x, scores, e, end_token=end), x, scores, e, end, 1e-12)
    scores[:, 1:] = -np.inf  # the first step: one beam
    B.check_select(T.beam_select(x, scores, 0 * ended, end_token=-1), x, scores, 0 * ended, -1, 1e-12)


def test_select_special_values():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, 20)).astype(np.float32)
    x[0] = np.nan
    x[1] = -np.inf
    x[2, 3:6] = np.inf
    x[3, ::2] = np.nan
    x[4] = 1.0  # ties
    scores = np.array([[-1, -2, -3, -4], [-1, np.nan, -np.inf, -1]], np.float32)
    ended = np.array([[0, 0, 0, 0], [0, 0, 1, 0]], np.int32)
    got = T.beam_select(x, scores, ended, end_token=4)
    B.check_select(got, x, scores, ended, 4, 1e-12)
    got = T.beam_select(x[:4], np.full((1, 4), -np.inf, np.float32), ended[:1], end_token=4)
    assert (got[0] == -1).all() and (got[1] == [0, 1, 2, 3]).all() and (got[2] == -np.inf).all()


@pytest.mark.parametrize("kind", ["bf16", "f32", "fp8"])
def test_reorder_cpu(kind):
    rng = np.random.default_rng(4)
    for lens in ([9, 9, 9, 4, 4, 4], [0] * 6, [16] * 6, [3] * 6, [100] * 6):
        tables = rng.permutation(30)[:24].reshape(6, 4).astype(np.int32)
        tables[1, 2] = -1
        parents = np.array([[1, 0, 0], [2, 7, 2]], np.int32)
        if kind == "fp8":
            (kc, ke), (vc, ve) = Q.random_cache(rng, 30, 4, 2, 8), Q.random_cache(rng, 30, 4, 2, 8)
            arrays = [kc, vc, ke, ve]
        else:
            arrays = [B.logits(rng, 30 * 8, 8, kind).reshape(30, 4, 2, 8) for _ in range(2)]
        t, want = B.reorder(parents, tables, np.array(lens), arrays)
        T.beam_reorder(parents, tables, np.array(lens), *arrays)
        assert (tables == t).all()
        for a, b in zip(arrays, want):
            assert a.tobytes() == b.tobytes()


# ---------------------------------------------------------------------------
def i(*s):
    return np.zeros(s, np.int32)


def z(*s):
    return np.zeros(s, np.float32)


def c8(*s):
    return np.zeros(s, dt.float8_e4m3fn)


def f_assign(block_tables, context_lens, new_lens, pages=9, page_size=4, tokens=7):
    return T.assign_pages(block_tables, context_lens, new_lens, pages=pages, page_size=page_size, tokens=tokens)


def f_select(logits, scores, ended, end_token=2):
    return T.beam_select(logits, scores, ended, end_token=end_token)


def f_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps=None, value_exps=None):
    T.beam_reorder(parents, block_tables, context_lens, key_cache, value_cache, key_exps, value_exps)


ASSIGN = dict(block_tables=i(3, 2), context_lens=i(3), new_lens=i(3))
SELECT = dict(logits=z(6, 10), scores=z(2, 3), ended=i(2, 3))
REORDER = dict(parents=i(2, 3), block_tables=i(6, 4), context_lens=i(6), key_cache=c8(9, 4, 2, 8), value_cache=c8(9, 4, 2, 8),
               key_exps=i(9, 2), value_exps=i(9, 2))


@pytest.mark.parametrize("f,ok,error,text,change", [
    (f_assign, ASSIGN, TypeError, "must be of int32", dict(block_tables=np.zeros((3, 2), np.int16))),
    (f_assign, ASSIGN, ValueError, "name no page", dict(block_tables=i(3, 0))),
    (f_assign, ASSIGN, ValueError, "context_lens must have", dict(context_lens=i(2))),
    (f_assign, ASSIGN, TypeError, "integers", dict(new_lens=z(3))),
    (f_assign, ASSIGN, ValueError, "pages must be", dict(pages=0)),
    (f_assign, ASSIGN, ValueError, "pages must be", dict(pages=2**20 + 1)),
    (f_assign, ASSIGN, ValueError, "page_size must be", dict(page_size=0)),
    (f_assign, ASSIGN, ValueError, "tokens must be", dict(tokens=-1)),
    (f_assign, ASSIGN, ValueError, "tokens must be", dict(tokens=2.0)),
    (f_assign, ASSIGN, ValueError, "too large", dict(page_size=2**29)),
    (f_select, SELECT, ValueError, "row for each", dict(logits=z(5, 10))),
    (f_select, SELECT, ValueError, "2 dimensions", dict(scores=z(6))),
    (f_select, SELECT, ValueError, "1 to 32 beams", dict(scores=z(1, 33), logits=z(33, 10), ended=i(1, 33))),
    (f_select, SELECT, ValueError, "vocabulary", dict(logits=z(6, 0))),
    (f_select, SELECT, TypeError, "must be of", dict(logits=i(6, 10))),
    (f_select, SELECT, TypeError, "must be of", dict(scores=z(2, 3).astype(np.float16))),
    (f_select, SELECT, TypeError, "integers", dict(ended=z(2, 3))),
    (f_select, SELECT, ValueError, "end_token must be", dict(end_token=10)),
    (f_select, SELECT, ValueError, "end_token must be", dict(end_token=None)),
    (f_reorder, REORDER, ValueError, "row for each", dict(parents=i(2, 2))),
    (f_reorder, REORDER, ValueError, "1 to 32 beams", dict(parents=i(6, 0))),
    (f_reorder, REORDER, TypeError, "integers", dict(parents=z(2, 3))),
    (f_reorder, REORDER, TypeError, "must be of int32", dict(block_tables=np.zeros((6, 4), np.int16))),
    (f_reorder, REORDER, ValueError, "value_cache must have", dict(value_cache=c8(9, 4, 2, 4))),
    (f_reorder, REORDER, TypeError, "share one type", dict(value_cache=z(9, 4, 2, 8))),
    (f_reorder, REORDER, TypeError, "caches must be", dict(key_cache=i(9, 4, 2, 8), value_cache=i(9, 4, 2, 8))),
    (f_reorder, REORDER, ValueError, "give both", dict(key_exps=None)),
    (f_reorder, REORDER, ValueError, "have exponents", dict(key_exps=None, value_exps=None)),
    (f_reorder, REORDER, ValueError, "have exponents", dict(key_cache=z(9, 4, 2, 8), value_cache=z(9, 4, 2, 8))),
    (f_reorder, REORDER, ValueError, "key_exps must have", dict(key_exps=i(9, 3)))])
def test_refused(f, ok, error, text, change):
    f(**ok)
    for call in (f, lambda **k: NKIPyKernel.trace(f).specialize(**k)):
        with pytest.raises(error, match=text):
            call(**{**ok, **change})


def test_select_refuses_more_than_it_ranks():
    with pytest.raises(ValueError, match="too many"):
        f_select(np.broadcast_to(z(1, 1), (32, 2**22)), z(1, 32), i(1, 32))


def test_lowering():
    def plan(f, **kw):
        return lower(NKIPyKernel.trace(f).specialize(**kw))

    assert plan(f_assign, **ASSIGN).kernel_kinds == ["assign_pages"]
    assert plan(f_select, **SELECT).kernel_kinds == ["beam_select"]
    p = plan(f_reorder, **REORDER)
    assert p.kernel_kinds == ["beam_reorder"]
    assert set(p.alias_outputs) == {"block_tables", "key_cache", "value_cache", "key_exps", "value_exps"}

    def some(logits, scores, ended):  # two of four results
        tokens, _, new, _ = f_select(logits, scores, ended)
        return tokens, new

    assert plan(some, **SELECT).kernel_kinds == ["beam_select"]


def test_launch_helpers_refuse():
    ptr = dict(tables=16, lens=16, news=16, starts=16, slots=16, free=16, ws=16)
    D.assign_pages(3, 4, 16, 100, 2000, **ptr)
    for args in [(0, 4, 16, 100, 20), (3, 0, 16, 100, 20), (3, 4, 16, 2**20 + 1, 20), (3, 4, 0, 100, 20), (3, 4, 2**28, 7, 20),
                 (2**16 + 1, 4, 16, 100, 20)]:
        with pytest.raises(LaunchError):
            D.assign_pages(*args, **ptr)
    ptr = dict(x=16, scores=16, ended=16, tokens=16, parents=16, out=16, ends=16)
    D.beam_select(dt.float32, 1, 32, 2**18, 2**18, 2, **ptr, ws=16)
    for args in [(0, 4, 100), (1, 33, 100), (1, 4, 0), (1, 32, 2**22)]:
        with pytest.raises(LaunchError):
            D.beam_select(dt.float32, *args, 100, 2, **ptr, ws=16)
    with pytest.raises(LaunchError, match="workspace"):
        D.beam_select(dt.float32, 1, 4, 100, 100, 2, **ptr, ws=0)
    ptr = dict(parents=16, lens=16, tables=16, k=16, v=16)
    assert D.beam_reorder(2, 3, 4, 16, 9, 2, 1024, **ptr).symbol == "nk_beam_reorder16_k4"
    assert D.beam_reorder(2, 9, 4, 16, 9, 2, 24, **ptr).symbol == "nk_beam_reorder1_k32"
    for args in [(0, 3, 4, 16, 9, 2, 64), (2, 33, 4, 16, 9, 2, 64), (2, 3, 4, 0, 9, 2, 64), (2, 3, 4, 16, 0, 2, 64),
                 (2, 3, 4, 2**20, 9, 2, 2**15 + 1)]:
        with pytest.raises(LaunchError):
            D.beam_reorder(*args, **ptr)
