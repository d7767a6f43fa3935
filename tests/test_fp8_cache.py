"""The 8-bit paged cache on the CPU: its NumPy forms against plain 64-bit ones,
what they refuse, and what they lower to."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.ops import serving_fp8 as OPS
from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch import serving_fp8 as F
from nkipy_amd.dispatch.launchers import LaunchError
from nkipy_amd.dispatch.lower import lower

import fp8_plain as Q
import serving_plain as P


def draw(rng, shape, t, std=1.0):
    return P.cast(rng.standard_normal(shape) * std, t)


def close(got, want, tol):
    bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) - tol)}"


def test_codes_are_nearest():
    t = Q.TABLE[:127]
    mids = (t[:-1] + t[1:]) / 2
    x = np.concatenate([t, mids, np.nextafter(mids, 0), np.nextafter(mids, 500), [1e-30]])
    x = np.concatenate([x, -x])
    assert (Q.TABLE[Q.bits(OPS._codes(x))] == Q.nearest(x)).all()
    assert np.isnan(Q.TABLE[Q.bits(OPS._codes(np.array([np.nan, np.inf, -np.inf])))]).all()


@pytest.mark.parametrize("top,e", [(448.0, 0), (449.0, 1), (224.0, -1), (0.0, -120), (2.0**-140, -120), (3.4e38, 120)])
def test_exponents(top, e):
    assert OPS._exponent(np.array([top, -top / 2])) == e


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_append_cpu(t):
    rng = np.random.default_rng(5)
    tables, lens, starts, pages = P.batch(rng, [13, 2, 9, 6], [4, 3, 9, 1], 4)  # (a token before position 0)
    q, k, v = draw(rng, (17, 4, 16), t), draw(rng, (17, 2, 16), t), draw(rng, (17, 2, 16), t, 3)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 4, 2, 16), Q.random_cache(rng, pages, 4, 2, 16, -14, 3)
    tables[2, 1] = -1
    ang = rng.standard_normal((12, 6)).astype(np.float32)  # (positions 12 and up have no row)
    cos, sin = np.cos(ang), np.sin(ang)
    (rq, tq), parts = Q.append(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts, t)
    got = T.rotary_append_fp8(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts)
    close(P.up(got), rq, tq)
    for codes, exps, (e, val, tol, _) in ((kc, ke, parts[0]), (vc, ve, parts[1])):
        assert (exps == e).all()
        close(Q.values(codes, exps), val, tol)


def test_append_one_at_a_time_is_the_prompt():
    """Tokens appended one by one hold the exponent of the whole page, and
    values within a rounding of those appended at once."""
    rng = np.random.default_rng(6)
    x = draw(rng, (24, 2, 16), "f32", 1.0) * (1 + np.arange(24, dtype=np.float32))[:, None, None]
    cos, sin = np.ones((24, 8), np.float32), np.zeros((24, 8), np.float32)
    tables = np.array([[2, 0]], np.int32)
    a = [*Q.random_cache(rng, 3, 12, 2, 16), *Q.random_cache(rng, 3, 12, 2, 16)]
    b = [y.copy() for y in a]
    T.rotary_append_fp8(x, x, x, cos, sin, a[0], a[2], a[1], a[3], tables, np.array([24]), np.array([0, 24]))
    for i in range(24):
        T.rotary_append_fp8(x[i:i + 1], x[i:i + 1], x[i:i + 1], cos, sin, b[0], b[2], b[1], b[3], tables, np.array([i + 1]))
    for s in (0, 2):
        assert (a[s + 1] == b[s + 1]).all()
        u, w = Q.values(a[s], a[s + 1])[[0, 2]], Q.values(b[s], b[s + 1])[[0, 2]]
        # rounded once more where the scale grew: half a step of normal codes is
        # kept, subnormal ones move by half a step (2^-10 of the scale) at most twice
        assert (np.abs(u - w) <= 2 * 2.0 ** (a[s + 1][[0, 2]][:, None, :, None] - 10.0)).all()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
@pytest.mark.parametrize("packed", [True, False])
def test_attention_cpu(t, window, sinks, packed):
    rng = np.random.default_rng(3)
    lens, new = ([13, 0, 9, 21], [4, 0, 2, 21]) if packed else ([13, 0, 9, 21], None)
    tables, lens, starts, pages = P.batch(rng, lens, new, 4)
    n = int(starts[-1]) if packed else 4
    q = draw(rng, (n, 4, 16), t)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 4, 2, 16), Q.random_cache(rng, pages, 4, 2, 16)
    tables[3, 2] = 1000  # a page that is none
    got = T.paged_attention_fp8(q, kc, vc, ke, ve, tables, lens, starts, window=window or None, sinks=sinks)
    assert got.dtype == q.dtype
    close(P.up(got), *Q.paged(q, kc, vc, ke, ve, tables, lens, starts, window, sinks, t))


# ---------------------------------------------------------------------------
def _refused(f, error, text, *args, **kw):
    for call in (f, lambda *a, **k: NKIPyKernel.trace(f).specialize(*a, **k)):
        with pytest.raises(error, match=text):
            call(*args, **kw)


def z(*s):
    return np.zeros(s, np.float32)


def i(*s):
    return np.zeros(s, np.int32)


def c8(*s):
    return np.zeros(s, dt.float8_e4m3fn)


def f_append(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens, query_starts=None):
    return T.rotary_append_fp8(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens,
                               query_starts)


def f_attend(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens, query_starts=None, **kw):
    return T.paged_attention_fp8(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens, query_starts, **kw)


APPEND = dict(q=z(3, 4, 8), k=z(3, 2, 8), v=z(3, 2, 8), cos=z(5, 4), sin=z(5, 4), key_cache=c8(6, 2, 2, 8),
              value_cache=c8(6, 2, 2, 8), key_exps=i(6, 2), value_exps=i(6, 2), block_tables=i(3, 2), context_lens=i(3))
CACHE = {n: APPEND[n] for n in ("q", "key_cache", "value_cache", "key_exps", "value_exps", "block_tables", "context_lens")}


@pytest.mark.parametrize("error,text,change", [
    (ValueError, "k must have shape", dict(k=z(3, 2, 4))),
    (ValueError, "v must have shape", dict(v=z(2, 2, 8))),
    (ValueError, "3 dimensions", dict(q=z(3, 32))),
    (ValueError, "no multiple", dict(q=z(3, 3, 8))),
    (ValueError, "value_cache must have", dict(value_cache=c8(6, 2, 2, 4))),
    (ValueError, "no page", dict(key_cache=c8(0, 2, 2, 8), value_cache=c8(0, 2, 2, 8))),
    (ValueError, "key_exps must have", dict(key_exps=i(5, 2))),
    (ValueError, "value_exps must have", dict(value_exps=i(6, 1))),
    (TypeError, "must be of int32", dict(key_exps=np.zeros((6, 2), np.int16))),
    (TypeError, "must be of float8_e4m3fn", dict(key_cache=z(6, 2, 2, 8), value_cache=z(6, 2, 2, 8))),
    (ValueError, "one new token", dict(context_lens=i(2), block_tables=i(2, 2))),
    (ValueError, "query_starts must have", dict(query_starts=i(3))),
    (TypeError, "integers", dict(block_tables=z(3, 2))),
    (TypeError, "share one type", dict(q=z(3, 4, 8).astype(np.float16))),
    (ValueError, "do not fit", dict(cos=z(5, 5), sin=z(5, 5))),
    (ValueError, "sin must have", dict(sin=z(4, 4)))])
def test_append_refuses(error, text, change):
    f_append(**APPEND)
    _refused(f_append, error, text, **{**APPEND, **change})


def test_append_refuses_caches_it_cannot_write():
    same = dict(APPEND, value_cache=APPEND["key_cache"])
    with pytest.raises(ValueError, match="same array"):
        f_append(**same)
    with pytest.raises(ValueError, match="same array"):
        f_append(**dict(APPEND, value_exps=APPEND["key_exps"]))

    def part(big, **kw):
        return f_append(key_cache=big[0], **kw)

    rest = {n: x for n, x in APPEND.items() if n != "key_cache"}
    with pytest.raises(ValueError, match="part or another layout"):
        NKIPyKernel.trace(part).specialize(big=c8(2, 6, 2, 2, 8), **rest)

    def computed(key_exps, **kw):
        return f_append(key_exps=key_exps + 1, **kw)

    rest = {n: x for n, x in APPEND.items() if n != "key_exps"}
    with pytest.raises(TypeError, match="not computed"):
        NKIPyKernel.trace(computed).specialize(key_exps=APPEND["key_exps"], **rest)
    with pytest.raises(TypeError, match="written in place"):
        NKIPyKernel.trace(lambda q: f_append(**dict(APPEND, q=q))).specialize(APPEND["q"])


@pytest.mark.parametrize("error,text,change", [
    (ValueError, "head_dim 4", dict(q=z(3, 4, 4))),
    (ValueError, "no multiple", dict(q=z(3, 5, 8))),
    (ValueError, "window", dict(window=0)),
    (ValueError, "sinks", dict(window=4, sinks=-1)),
    (ValueError, "give one", dict(sinks=2)),
    (ValueError, "scale", dict(scale=0.0)),
    (ValueError, "key_exps must have", dict(key_exps=i(6, 3))),
    (TypeError, "must be of int32", dict(value_exps=np.zeros((6, 2), np.int16))),
    (TypeError, "must be of float8_e4m3fn", dict(key_cache=z(6, 2, 2, 8), value_cache=z(6, 2, 2, 8))),
    (TypeError, "must be of", dict(q=i(3, 4, 8)))])
def test_attention_refuses(error, text, change):
    f_attend(**CACHE)
    _refused(f_attend, error, text, **{**CACHE, **change})


def steps(f, **kw):
    return lower(NKIPyKernel.trace(f).specialize(**kw))


def test_one_launch_and_no_copies():
    plan = steps(f_append, **APPEND)
    assert plan.kernel_kinds == ["rotary_append_fp8"]
    assert set(plan.alias_outputs) == {"key_cache", "value_cache", "key_exps", "value_exps"}
    assert steps(f_attend, **CACHE).kernel_kinds == ["attend8"]


def test_layer_lowers_without_copies():
    """Append and attention, twice over the same caches."""

    def layer(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens):
        for _ in range(2):
            q = T.rotary_append_fp8(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens)
            q = T.paged_attention_fp8(q, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens)
        return q

    plan = steps(layer, **APPEND)
    assert plan.kernel_kinds == ["rotary_append_fp8", "attend8"] * 2


def test_old_cache_returned_stays_old():
    """A caller that reads a cache's old exponents after the append gets them."""

    def f(**kw):
        before = kw["key_exps"] + 0
        out = f_append(**kw)
        return out, before

    def g(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, block_tables, context_lens):
        return f(q=q, k=k, v=v, cos=cos, sin=sin, key_cache=key_cache, value_cache=value_cache, key_exps=key_exps,
                 value_exps=value_exps, block_tables=block_tables, context_lens=context_lens)

    assert "rotary_append_fp8" in steps(g, **APPEND).kernel_kinds


def test_launch_helpers_refuse():
    ok = dict(q=0, k=0, v=0, oq=0, kc=0, vc=0, ke=0, ve=0, cos=0, sin=0, tables=0, lens=0)
    F.rotary_append_fp8(dt.bfloat16, 2, 4, 4, 2, 128, 64, 10, 16, 5, 3, **ok, starts=16)
    for args in [(0, 4, 4, 2, 128, 64, 10, 16, 5, 3), (2, 0, 4, 2, 128, 64, 10, 16, 5, 3), (2, 4, 4, 2, 128, 65, 10, 16, 5, 3),
                 (2, 4, 4, 2, 128, 64, 10, 0, 5, 3), (2, 4, 4, 2, 128, 64, 10, 16, 2**28, 3), (2**30 - 1, 4, 4, 512, 128, 64, 10, 16, 5, 3),
                 (2, 4, 4, 2, 256, 64, 10, 2**23, 5, 3)]:
        with pytest.raises(LaunchError):
            F.rotary_append_fp8(dt.bfloat16, *args, **ok)
    kw = dict(B=1, N=1, Hq=4, Hkv=2, D=128, q_str=(0, 512, 128), k_str=(0, 256, 128), v_str=(0, 256, 128), scale=1.0, tables=16,
              lens=16, ke=16, ve=16, page=16, pages=9, width=8, pitch=16)
    F.attend8(dt.bfloat16, 16, 16, 16, 16, **kw, ws=16)
    for change in [dict(B=0), dict(Hq=3), dict(D=257), dict(pitch=15), dict(pages=0), dict(width=2**27), dict(k_str=(0, 0, 128))]:
        with pytest.raises(LaunchError):
            F.attend8(dt.bfloat16, 16, 16, 16, 16, **{**kw, **change}, ws=16)
    with pytest.raises(LaunchError, match="workspace"):
        F.attend8(dt.bfloat16, 16, 16, 16, 16, **{**kw, "width": 2000})


def test_workgroups_of_an_append_cover_its_pages():
    """The tiles of a packed batch leave room for every page that a sequence
    may write (append8.hip: floor(start / page) + 2 b)."""
    rng = np.random.default_rng(8)
    for page in (1, 3, 16):
        new = rng.integers(0, 40, 30)
        starts = np.concatenate([[0], np.cumsum(new)])
        tiles = starts[:-1] // page + 2 * np.arange(30)
        for p0 in range(page):
            touched = np.where(new > 0, (p0 + new - 1) // page + 1, 0)
            assert (tiles[:-1] + touched[:-1] <= tiles[1:]).all()
            assert tiles[-1] + touched[-1] <= starts[-1] // page + 60
