"""What calls that update arguments say to another name of one."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel

CODES = np.zeros((6, 4, 1, 8), np.uint8).view(dt.float8_e4m3fn)
EXPS = np.zeros((6, 1), np.int32)
TABLES, LENS = np.zeros((2, 3), np.int32), np.zeros(2, np.int32)
Q, ANGLES = np.zeros((2, 1, 8), np.float32), np.zeros((12, 4), np.float32)


def assign(tables, lens, other):
    return T.assign_pages(other(tables), lens, lens, pages=6, page_size=4, tokens=3)


def reorder_tables(parents, tables, lens, k, v, other):
    T.beam_reorder(parents, other(tables), lens, k, v)


def reorder_cache(parents, tables, lens, k, v, other):
    T.beam_reorder(parents, tables, lens, k, other(v))


def reorder_twice(parents, tables, lens, k, other):
    T.beam_reorder(parents, tables, lens, k, other(k))


def append_cache(q, c, kc, vc, ke, ve, tables, lens, other):
    return T.rotary_append_fp8(q, q, q, c, c, other(kc), vc, ke, ve, tables, lens)


def append_exps(q, c, kc, vc, ke, ve, tables, lens, other):
    return T.rotary_append_fp8(q, q, q, c, c, kc, vc, ke, other(ve), tables, lens)


PARENTS, CACHE = np.zeros((1, 2), np.int32), np.zeros((6, 4, 1, 8), np.float32)
CALLS = [(assign, dict(tables=TABLES, lens=LENS)),
         (reorder_tables, dict(parents=PARENTS, tables=TABLES, lens=LENS, k=CACHE, v=CACHE)),
         (reorder_cache, dict(parents=PARENTS, tables=TABLES, lens=LENS, k=CACHE, v=CACHE)),
         (reorder_twice, dict(parents=PARENTS, tables=TABLES, lens=LENS, k=CACHE)),
         (append_cache, dict(q=Q, c=ANGLES, kc=CODES, vc=CODES, ke=EXPS, ve=EXPS, tables=TABLES, lens=LENS)),
         (append_exps, dict(q=Q, c=ANGLES, kc=CODES, vc=CODES, ke=EXPS, ve=EXPS, tables=TABLES, lens=LENS))]


@pytest.mark.parametrize("other", [lambda x: x[:], lambda x: x.reshape(x.shape), lambda x: x[...]])
@pytest.mark.parametrize("f,kw", CALLS)
def test_whole_views_are_refused(f, kw, other):
    """A write into a view of the whole argument would be lost."""
    with pytest.raises(ValueError, match="pass the argument itself"):
        NKIPyKernel.trace(lambda *a: f(*a, other=other)).specialize(*kw.values())


@pytest.mark.parametrize("f,kw", CALLS[:3] + CALLS[4:])
def test_the_arguments_themselves_are_taken(f, kw):
    NKIPyKernel.trace(lambda *a: f(*a, other=lambda x: x)).specialize(*kw.values())
