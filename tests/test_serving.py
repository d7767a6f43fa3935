"""The serving operators on the CPU: their NumPy forms against plain 64-bit
ones, what they refuse, and what they lower to."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch import serving as S
from nkipy_amd.dispatch.launchers import LaunchError
from nkipy_amd.dispatch.lower import lower

import serving_plain as P


def draw(rng, shape, t, std=1.0):
    return P.cast(rng.standard_normal(shape) * std, t)


def close(got, want, tol):
    bad = ~(np.abs(P.up(got) - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(P.up(got) - want) - tol)}"


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
@pytest.mark.parametrize("packed", [True, False])
def test_paged_cpu(t, window, sinks, packed):
    rng = np.random.default_rng(3)
    lens, new = ([13, 0, 9, 21], [4, 0, 2, 21]) if packed else ([13, 0, 9, 21], None)
    tables, lens, starts, pages = P.batch(rng, lens, new, 4)
    n = int(starts[-1]) if packed else 4
    q, kc, vc = draw(rng, (n, 4, 16), t), draw(rng, (pages, 4, 2, 16), t), draw(rng, (pages, 4, 2, 16), t)
    tables[3, 2] = 1000  # a page that is none
    got = T.paged_attention(q, kc, vc, tables, lens, starts, window=window or None, sinks=sinks)
    assert got.dtype == q.dtype
    close(got, *P.paged(q, kc, vc, tables, lens, starts, window, sinks, t))


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_window_cpu(t):
    rng = np.random.default_rng(4)
    q, k, v = draw(rng, (3, 11, 4, 8), t), draw(rng, (3, 14, 2, 8), t), draw(rng, (3, 14, 2, 8), t)
    lengths, positions = np.array([14, 0, 6], np.int32), np.array([3, 0, -2], np.int32)
    for a, b, w, s in [(None, None, 0, 0), (lengths, positions, 0, 0), (lengths, None, 4, 1), (None, positions, 1, 3)]:
        close(T.window_attention(q, k, v, a, b, window=w or None, sinks=s), *P.dense(q, k, v, a, b, w, s, t))


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_append_cpu(t):
    rng = np.random.default_rng(5)
    tables, lens, starts, pages = P.batch(rng, [13, 2, 9], [4, 3, 9], 4)  # (a token before position 0)
    q, k, v = draw(rng, (17, 4, 16), t), draw(rng, (17, 2, 16), t), draw(rng, (17, 2, 16), t)
    kc, vc = draw(rng, (pages, 4, 2, 16), t), draw(rng, (pages, 4, 2, 16), t)
    tables[2, 1] = -1
    ang = rng.standard_normal((12, 6)).astype(np.float32)  # (positions 12 and up have no row)
    cos, sin = np.cos(ang), np.sin(ang)
    (rq, rk, rv), (tq, tk, tv) = P.append(q, k, v, cos, sin, kc, vc, tables, lens, starts, t)
    got = T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens, starts)
    close(got, rq, tq)
    close(kc, rk, tk)
    close(vc, rv, tv)


def test_sample_cpu():
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((40, 60)) * 3).astype(np.float32)
    x[:, ::7] = -np.inf
    x[3:6] = np.round(x[3:6])  # ties
    x[7] = -np.inf
    x[8, 5] = np.nan
    u = rng.random(40).astype(np.float32)
    for k, p, m in [(None, None, None), (5, None, None), (None, 0.8, None), (12, 0.7, 0.05), (1, None, None)]:
        got = T.sample(x, u, 0.7, k, p, m)
        assert got.dtype == np.int32 and got[7] == -1
        for r in range(40):
            if r == 7:
                continue
            ids, w = P.kept(x[r].astype(np.float64), 0.7, k, p, m)
            c = np.cumsum(w)
            assert got[r] == ids[int((c <= u[r] * c[-1]).sum())]
    assert (T.sample(x, u, 0.0)[:7] == np.argmax(x[:7], 1)).all()
    assert (T.sample(x[:4], u[:4], np.array([0, 1, 1, 0], "f4"), top_k=np.array([0, 1, 1, 3])) == np.argmax(x[:4], 1)).all()


# ---------------------------------------------------------------------------
def _call(f):
    """On the CPU and under trace."""
    yield f
    yield lambda *a, **k: NKIPyKernel.trace(f).specialize(*a, **k)


def _refused(f, error, text, *args, **kw):
    for call in _call(f):
        with pytest.raises(error, match=text):
            call(*args, **kw)


def test_append_refuses():
    z = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    i = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    ok = dict(q=z(3, 4, 8), k=z(3, 2, 8), v=z(3, 2, 8), cos=z(5, 4), sin=z(5, 4), key_cache=z(6, 2, 2, 8),
              value_cache=z(6, 2, 2, 8), block_tables=i(3, 2), context_lens=i(3))

    def f(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts=None):
        return T.rotary_append(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts)

    for call in _call(f):
        call(**ok)
    for error, text, change in [
            (ValueError, "k must have shape", dict(k=z(3, 2, 4))),
            (ValueError, "v must have shape", dict(v=z(2, 2, 8))),
            (ValueError, "3 dimensions", dict(q=z(3, 32))),
            (ValueError, "no multiple", dict(q=z(3, 3, 8))),
            (ValueError, "value_cache must have", dict(value_cache=z(6, 2, 2, 4))),
            (ValueError, "no page", dict(key_cache=z(0, 2, 2, 8), value_cache=z(0, 2, 2, 8))),
            (ValueError, "no page", dict(block_tables=i(3, 0))),
            (ValueError, "one new token", dict(context_lens=i(2), block_tables=i(2, 2))),
            (ValueError, "context_lens must have", dict(context_lens=i(2))),
            (ValueError, "query_starts must have", dict(query_starts=i(3))),
            (TypeError, "integers", dict(block_tables=z(3, 2))),
            (TypeError, "share one type", dict(q=z(3, 4, 8).astype(np.float16))),
            (TypeError, "must be of", dict(cos=z(5, 4).astype(np.float16))),
            (ValueError, "do not fit", dict(cos=z(5, 5), sin=z(5, 5))),
            (ValueError, "sin must have", dict(sin=z(4, 4)))]:
        _refused(f, error, text, **{**ok, **change})
    with pytest.raises(ValueError, match="same array"):
        T.rotary_append(ok["q"], ok["k"], ok["v"], ok["cos"], ok["sin"], ok["key_cache"], ok["key_cache"],
                        ok["block_tables"], ok["context_lens"])
    with pytest.raises(TypeError, match="written in place"):  # a constant cache
        NKIPyKernel.trace(lambda q: T.rotary_append(q, *list(ok.values())[1:])).specialize(ok["q"])


def test_attention_refuses():
    z = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    i = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    paged = dict(q=z(3, 4, 8), key_cache=z(6, 2, 2, 8), value_cache=z(6, 2, 2, 8), block_tables=i(3, 2), context_lens=i(3))

    def f(q, key_cache, value_cache, block_tables, context_lens, **kw):
        return T.paged_attention(q, key_cache, value_cache, block_tables, context_lens, **kw)

    for error, text, change in [
            (ValueError, "head_dim 4", dict(q=z(3, 4, 4))),
            (ValueError, "no multiple", dict(q=z(3, 5, 8))),
            (ValueError, "window", dict(window=0)),
            (ValueError, "window", dict(window=2.5)),
            (ValueError, "window", dict(window=True)),
            (ValueError, "sinks", dict(window=4, sinks=-1)),
            (ValueError, "give one", dict(sinks=2)),
            (ValueError, "scale", dict(scale=0.0)),
            (ValueError, "scale", dict(scale=float("nan"))),
            (TypeError, "share one type", dict(q=z(3, 4, 8).astype(np.float16))),
            (TypeError, "must be of", dict(q=i(3, 4, 8)))]:
        _refused(f, error, text, **{**paged, **change})
    _refused(f, ValueError, "1..256", z(3, 2, 264), z(6, 2, 2, 264), z(6, 2, 2, 264), i(3, 2), i(3))

    def g(q, k, v, **kw):
        return T.window_attention(q, k, v, **kw)

    dense = dict(q=z(2, 5, 4, 8), k=z(2, 6, 2, 8), v=z(2, 6, 2, 8))
    for error, text, change in [
            (ValueError, "does not fit", dict(k=z(3, 6, 2, 8))),
            (ValueError, "v must have", dict(v=z(2, 6, 1, 8))),
            (ValueError, "lengths must have", dict(lengths=i(3))),
            (TypeError, "integers", dict(positions=z(2)))]:
        _refused(g, error, text, **{**dense, **change})


def test_sample_refuses():
    x, u = np.zeros((3, 9), np.float32), np.zeros(3, np.float32)

    def f(logits, uniform, **kw):
        return T.sample(logits, uniform, **kw)

    for error, text, args, kw in [
            (ValueError, "uniform must have", (x, u[:2]), {}),
            (ValueError, "2 dimensions", (u, u), {}),
            (ValueError, "no token", (x[:, :0], u), {}),
            (TypeError, "must be of", (x.astype(np.int32), u), {}),
            (TypeError, "must be of", (x, u.astype(np.float16)), {}),
            (ValueError, "in 0..1", (x, u), dict(top_p=1.5)),
            (ValueError, "in 0..1", (x, u), dict(min_p=-0.1)),
            (ValueError, "at least 0", (x, u), dict(temperature=-1.0)),
            (ValueError, "at least 0", (x, u), dict(temperature=float("nan"))),
            (TypeError, "whole number", (x, u), dict(top_k=2.5)),
            (ValueError, "array of shape", (x, u), dict(top_k=np.zeros(2, np.int32))),
            (TypeError, "integers", (x, u), dict(top_k=np.zeros(3, np.float32)))]:
        _refused(f, error, text, *args, **kw)


def test_launch_helpers_refuse():
    with pytest.raises(LaunchError, match="tokens"):
        S.rotary_append(dt.bfloat16, 1, 0, 4, 2, 64, 32, 8, 16, 4, 2)
    with pytest.raises(LaunchError, match="block table"):
        S.rotary_append(dt.bfloat16, 1, 1, 4, 2, 64, 32, 8, 16, 4, 2, k=256, ok=256)
    kw = dict(B=1, N=1, Hq=4, Hkv=2, D=64, q_str=(0, 256, 64), k_str=(0, 128, 64), v_str=(0, 128, 64), scale=1.0)
    with pytest.raises(LaunchError, match="heads"):
        S.attend(dt.bfloat16, 256, 256, 256, 256, **{**kw, "Hkv": 3})
    with pytest.raises(LaunchError, match="too large"):
        S.attend(dt.bfloat16, 256, 256, 256, 256, tables=256, lens=256, page=16, pages=2**28, width=4, pitch=16, **kw)
    with pytest.raises(LaunchError, match="too long"):
        S.attend(dt.bfloat16, 256, 256, 256, 256, S=2, T=4, **kw)
    with pytest.raises(LaunchError, match="rows"):
        S.sample(dt.float32, 256, 256, 256, 0, 5, 5, temperature=(0, 1.0), top_k=(0, 0), top_p=(0, 1.0), min_p=(0, 0.0))


# ---------------------------------------------------------------------------
def _plan(f, *args, **kw):
    return lower(NKIPyKernel.trace(f).specialize(*args, **kw))


def test_step_lowers_to_its_launches():
    """The projection's heads are read in place, one launch appends, the
    caches are the caller's own buffers."""

    def step(qkv, cos, sin, kc, vc, tables, lens, starts):
        x = qkv.reshape(qkv.shape[0], 8, 64)
        q = T.rotary_append(x[:, :4], x[:, 4:6], x[:, 6:], cos, sin, kc, vc, tables, lens, starts)
        return T.paged_attention(q, kc, vc, tables, lens, starts, window=16, sinks=2)

    bf = lambda *s: np.zeros(s, dt.bfloat16)  # noqa: E731
    i = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    p = _plan(step, bf(10, 512), f(50, 32), f(50, 32), bf(9, 4, 2, 64), bf(9, 4, 2, 64), i(2, 4), i(2), i(3))
    assert p.kernel_kinds == ["rotary_append", "attend"]
    assert p.alias_outputs == {"kc": "kc.must_alias_input", "vc": "vc.must_alias_input"}

    def late(q, k, v, cos, sin, kc, vc, tables, lens):
        old = kc * 2.0  # the cache before the call is still read after it
        r = T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens)
        return r, kc + old

    p = _plan(late, f(2, 2, 8), f(2, 2, 8), f(2, 2, 8), f(5, 4), f(5, 4), f(3, 2, 2, 8), f(3, 2, 2, 8), i(2, 2), i(2))
    assert "rotary_append" in p.kernel_kinds and len(p.kernel_kinds) > 2


def test_empty_batches_launch_nothing():
    f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    i = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    assert not _plan(lambda x, u: T.sample(x, u), f(0, 9), f(0)).steps
    assert not _plan(lambda q, k, v: T.window_attention(q, k, v), f(2, 0, 2, 8), f(2, 3, 2, 8), f(2, 3, 2, 8)).steps
    assert not _plan(lambda q, k, v, t, n, s: T.paged_attention(q, k, v, t, n, s), f(0, 2, 8), f(3, 4, 2, 8), f(3, 4, 2, 8),
                     i(2, 2), i(2), i(3)).steps
    assert T.paged_attention(f(0, 2, 8), f(3, 4, 2, 8), f(3, 4, 2, 8), i(2, 2), i(2), i(3)).shape == (0, 2, 8)
    assert T.sample(f(0, 9), f(0)).shape == (0,)


def test_two_appends_keep_their_own_tables():
    """A call whose rotated q nobody reads, then one with other tables: the second's
    q is not turned by the first's."""

    def two(q, k, v, cos, sin, cos2, sin2, kc, vc, kc2, vc2, tables, lens):
        T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens)
        return T.rotary_append(q, k, v, cos2, sin2, kc2, vc2, tables, lens)

    f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    i = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    p = _plan(two, f(2, 2, 8), f(2, 2, 8), f(2, 2, 8), f(5, 4), f(5, 4), f(5, 2), f(5, 2), f(3, 2, 2, 8), f(3, 2, 2, 8),
              f(4, 2, 2, 8), f(4, 2, 2, 8), i(2, 2), i(2))
    assert p.kernel_kinds == ["rotary_append", "rotary_append"]
    assert [sorted(s.desc.split(": ")[1].split(", ")) for s in p.steps] == [["k", "v"], ["k", "q", "v"]]


def test_attention_refuses_scales_outside_32_bits():
    q, k = np.zeros((1, 2, 2, 8), np.float32), np.zeros((1, 3, 2, 8), np.float32)
    for scale in (2.0**65, 1e300, 2.0**-65, -1.0):
        with pytest.raises(ValueError, match="scale"):
            T.window_attention(q, k, k, scale=scale)
    assert (T.window_attention(q, k, k, scale=2.0**-64) == 0).all()
