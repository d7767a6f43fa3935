"""What the serving operators' launches are given for caches and tensors of
unusual layouts, read from the plans on the CPU."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch import serving as S
from nkipy_amd.dispatch.launchers import LaunchError
from nkipy_amd.dispatch.lower import lower

bf = lambda *s: np.zeros(s, dt.bfloat16)  # noqa: E731
i32 = lambda *s: np.zeros(s, np.int32)  # noqa: E731
f32 = lambda *s: np.zeros(s, np.float32)  # noqa: E731


def plan(f, *args, **kw):
    return lower(NKIPyKernel.trace(f).specialize(*args, **kw))


def launches(p, kind):
    """The launches of a plan's steps of one kind, with every buffer at an address of its own."""
    at = {}
    return [x for s in p.steps if getattr(s, "kind", None) == kind
            for x in s.launches(lambda v: at.setdefault(id(v), 2**20 * (len(at) + 1)))]


@pytest.mark.parametrize("starts", [None, i32(3)])
@pytest.mark.parametrize("shared", ["pages", "rows", "keys"])
def test_caches_whose_pages_share_memory(starts, shared):
    """A cache broadcast over its pages, or its rows, is laid out before the launch;
    every page has rows of its own there."""

    def f(q, k, t, n, s=None):
        c = np.broadcast_to(k, (5, 16, 2, 64))
        return T.paged_attention(q, c, c if shared != "keys" else c + 0, t, n, s)

    k = bf(1, 16, 2, 64) if shared != "rows" else bf(5, 1, 2, 64)
    kw = {} if starts is None else {"s": starts}
    for x in launches(plan(f, bf(2, 4, 64), k, i32(2, 3), i32(2), **kw), "attend"):
        assert x.args.pitch >= x.args.page == 16 and x.args.k_ss >= 64 and x.args.v_ss >= 64


def test_attention_refuses_overlapping_pages_and_rows_backwards():
    kw = dict(B=1, N=1, Hq=4, Hkv=2, D=64, q_str=(0, 256, 64), k_str=(0, 128, 64), v_str=(0, 128, 64), scale=1.0)
    paged = dict(kw, tables=256, lens=256, page=16, pages=3, width=4)
    for zeros in (0, 256):
        S.attend(dt.bfloat16, 256, 256, 256, 256, **paged, pitch=16, zeros=zeros, ws=256)
        for pitch in (0, 15, -16):
            with pytest.raises(LaunchError, match="pitch"):
                S.attend(dt.bfloat16, 256, 256, 256, 256, **paged, pitch=pitch, zeros=zeros, ws=256)
        for name in ("k_str", "v_str"):
            for row in (0, -128):
                with pytest.raises(LaunchError, match="stride"):
                    S.attend(dt.bfloat16, 256, 256, 256, 256, **{**paged, name: (0, row, 64)}, pitch=16, zeros=zeros, ws=256)
            with pytest.raises(LaunchError, match="stride"):
                S.attend(dt.bfloat16, 256, 256, 256, 256, **{**kw, name: (0, -128, 64)}, T=4, zeros=zeros, ws=256)
            S.attend(dt.bfloat16, 256, 256, 256, 256, **{**kw, name: (0, 0, 64)}, T=4, zeros=zeros, ws=256)  # (one row is every key)


def values_alone(q, k, v, cos, sin, vc, tables, lens, starts=None):
    """The rotated q and keys are used by nothing: one launch, of the values."""
    T.rotary_append(q, k, v, cos, sin, vc * np.float32(2), vc, tables, lens, starts)


def test_values_written_alone_know_the_positions():
    p = plan(values_alone, f32(3, 4, 8), f32(3, 2, 8), f32(3, 2, 8), f32(7, 4), f32(7, 4), f32(5, 4, 2, 8), i32(3, 2), i32(3))
    (x,) = launches(p, "rotary_append")
    assert not x.args.oq and not x.args.ok and x.args.ov and x.args.P == 7
