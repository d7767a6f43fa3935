"""Appends into the same caches one after the other, read from the plans on the
CPU."""

import numpy as np

from nkipy_amd.core import tensor_apis as T

from test_serving_layouts import f32, i32, plan

A = dict(q=f32(2, 4, 8), k=f32(2, 2, 8), cos=f32(9, 4), kc=f32(5, 4, 2, 8), vc=f32(5, 4, 2, 8), tables=i32(2, 3), lens=i32(2))


def append(q, k, cos, kc, vc, tables, lens):
    return T.rotary_append(q, k, k, cos, cos, kc, vc, tables, lens)


def test_appends_in_turn_stay_in_the_caller_s_buffers():
    def two(later, q, **a):
        x = append(q=q, **a)
        o = T.paged_attention(x, a["kc"], a["vc"], a["tables"], a["lens"])
        return o, T.paged_attention(append(q=q, **{**a, "lens": later}), a["kc"], a["vc"], a["tables"], later)

    p = plan(two, i32(2), **A)
    assert p.kernel_kinds == ["rotary_append", "attend", "rotary_append", "attend"]
    assert p.alias_outputs == {"kc": "kc.must_alias_input", "vc": "vc.must_alias_input"}

    def three(later, **a):
        append(**a)
        append(**{**a, "lens": later})
        return append(**a)

    assert plan(three, i32(2), **A).kernel_kinds == ["rotary_append"] * 3


def test_appends_in_turn_copy_what_is_still_read():
    """The cache between two calls, read after the second or returned; the old cache,
    read between the two."""

    def between(later, kc, **a):
        append(kc=kc, **a)
        old = kc * np.float32(2)
        append(kc=kc, **{**a, "lens": later})
        return old + kc, kc

    kinds = plan(between, i32(2), **A).kernel_kinds
    assert kinds.count("rotary_append") == 2 and len(kinds) > 2

    def before(later, kc, **a):
        old = kc + 0
        append(kc=kc, **a)
        x = old * np.float32(2)
        append(kc=kc, **{**a, "lens": later})
        return x + kc

    kinds = plan(before, i32(2), **A).kernel_kinds
    assert kinds.count("rotary_append") == 2 and len(kinds) > 3
