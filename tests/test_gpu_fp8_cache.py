"""The 8-bit paged cache on the GPU against plain 64-bit forms."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T

import fp8_plain as Q
import serving_plain as P
from test_gpu_serving import draw, load, run

pytestmark = pytest.mark.gpu


def close(got, want, tol):
    got = P.up(got) if got.dtype != np.float64 else got
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}, worst by {np.nanmax(np.where(bad, np.abs(got - want), 0))}"


def f_append(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, tables, lens, starts=None):
    return T.rotary_append_fp8(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, tables, lens, starts)


def f_attend(q, key_cache, value_cache, key_exps, value_exps, tables, lens, starts=None, window=None, sinks=0, scale=None):
    return T.paged_attention_fp8(q, key_cache, value_cache, key_exps, value_exps, tables, lens, starts, window=window,
                                 sinks=sinks, scale=scale)


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def check_append(rng, t, hq, hkv, d, half, page, lens, new, positions=None, spoil=None, std=1.0, exps=(-14, 3)):
    tables, lens, starts, pages = P.batch(rng, lens, new, page)
    n = int(starts[-1]) if starts is not None else len(lens)
    q, k, v = draw(rng, (n, hq, d), t), draw(rng, (n, hkv, d), t, std), draw(rng, (n, hkv, d), t, std)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, page, hkv, d, *exps), Q.random_cache(rng, pages, page, hkv, d, *exps)
    ang = rng.standard_normal((positions or max(int(max(lens)), 1), half)).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    if spoil is not None:
        spoil(k, v, tables, lens, kc, vc, ke, ve)
    (rq, tq), parts = Q.append(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts, t)
    got = run(f_append, q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts)
    close(got["output0"], rq, tq)
    for name, (e, val, tol, wrote) in (("key", parts[0]), ("value", parts[1])):
        assert (got[name + "_exps"] == e).all()
        close(Q.values(got[name + "_cache"], got[name + "_exps"]), val, tol)
        # what nobody writes keeps its bits, NaN codes included
        same = ~wrote & (e == (ke if name == "key" else ve))[:, None, :, None]
        assert (Q.bits(got[name + "_cache"])[same] == Q.bits(kc if name == "key" else vc)[same]).all()
    return got


HEADS = [(4, 2, 128, 64), (3, 1, 64, 32), (16, 16, 64, 16), (32, 8, 128, 64), (4, 4, 80, 40), (2, 2, 20, 10), (3, 1, 5, 2), (2, 1, 256, 3)]


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,half", HEADS)
def test_append_single_tokens(t, hq, hkv, d, half):
    check_append(np.random.default_rng(21), t, hq, hkv, d, half, 16, [1, 300, 33, 17, 32, 129], None)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,half", HEADS)
def test_append_prompts(t, hq, hkv, d, half):
    check_append(np.random.default_rng(22), t, hq, hkv, d, half, 16, [70, 1, 5, 130, 129], [70, 1, 0, 65, 3])


@pytest.mark.parametrize("page", [1, 3, 24, 64, 200])
@pytest.mark.parametrize("new", [None, [5, 40, 1, 200]])
def test_append_page_sizes(page, new):
    check_append(np.random.default_rng(23), "bf16", 4, 2, 64, 32, page, [90, 40, 513, 260], new)


def test_append_many_sequences():
    rng = np.random.default_rng(24)
    new = [int(x) for x in rng.integers(0, 4, 200)]
    check_append(rng, "bf16", 4, 2, 64, 32, 16, [n + int(rng.integers(0, 90)) for n in new], new)


def test_append_drops_tokens_without_a_place():
    """Pages that are none, positions outside the tables, past the block table
    and before 0."""

    def spoil(k, v, tables, lens, kc, vc, ke, ve):
        tables[0, 1] = -1
        tables[1, 0] = 10**6
        lens[2] = 2
        lens[3] += 16 * tables.shape[1]

    check_append(np.random.default_rng(25), "bf16", 4, 2, 64, 32, 16, [40, 9, 30, 33], [20, 9, 5, 7], positions=45, spoil=spoil)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_append_grows_and_keeps_scales(t):
    """New rows larger and smaller than those there, zeros, and the largest
    and smallest exponents."""

    def spoil(k, v, tables, lens, kc, vc, ke, ve):
        ke[:] = np.array([-30, 10])[None]
        ve[tables[0, 0]] = [-500, 500]
        ve[tables[1, 0]] = [-120, 120]
        v[1] = P.cast(np.zeros(v[1].shape), t)

    check_append(np.random.default_rng(26), t, 4, 2, 64, 32, 16, [5, 9, 16, 17], None, spoil=spoil)
    check_append(np.random.default_rng(27), t, 4, 2, 64, 32, 16, [12, 15, 18, 40], [4, 9, 2, 7], std=1e-30)
    check_append(np.random.default_rng(28), t, 4, 2, 64, 32, 16, [12, 15, 18, 40], [4, 9, 2, 7], std=1e30)


def test_append_values_that_are_not_finite():
    def spoil(k, v, tables, lens, kc, vc, ke, ve):
        v[0, 0, 3], v[5, 1, 60], v[6] = P.cast(np.inf, "bf16"), P.cast(np.nan, "bf16"), P.cast(np.full(v[6].shape, -np.inf), "bf16")
        k[2, 1, 9] = P.cast(np.nan, "bf16")
        Q.bits(kc)[tables[1, 0], 0] = 0x7F
        vc.view(np.uint8)[tables[1, 0], 1] = 0xFF
        ke[:] = -40

    def check(rng):
        return check_append(rng, "bf16", 4, 2, 64, 32, 16, [9, 12, 40], [9, 7, 20], spoil=spoil)

    with np.errstate(invalid="ignore"):
        check(np.random.default_rng(29))


def test_append_strided_and_odd_addresses():
    """Heads sliced out of a projection, at addresses that fit 16 bytes and not."""
    rng = np.random.default_rng(30)
    for extra in (0, 3):
        tables, lens, starts, pages = P.batch(rng, [30, 20], [7, 20], 16)
        x = draw(rng, (27, 8 * 64 + extra), "bf16")
        (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 64), Q.random_cache(rng, pages, 16, 2, 64)
        ang = rng.standard_normal((30, 32)).astype(np.float32)
        cos, sin = np.cos(ang), np.sin(ang)

        def f(x, cos, sin, kc, vc, ke, ve, tables, lens, starts):
            y = x[:, extra:].reshape(27, 8, 64)
            return T.rotary_append_fp8(y[:, :4], y[:, 4:6], y[:, 6:], cos, sin, kc, vc, ke, ve, tables, lens, starts)

        y = x[:, extra:].reshape(27, 8, 64)
        (rq, tq), parts = Q.append(y[:, :4], y[:, 4:6], y[:, 6:], cos, sin, kc, vc, ke, ve, tables, lens, starts, "bf16")
        got = run(f, x, cos, sin, kc, vc, ke, ve, tables, lens, starts)
        close(got["output0"], rq, tq)
        for c, s, (e, val, tol, _) in (("kc", "ke", parts[0]), ("vc", "ve", parts[1])):
            assert (got[s] == e).all()
            close(Q.values(got[c], got[s]), val, tol)


def test_append_rows_outside_every_sequence():
    rng = np.random.default_rng(31)
    tables, lens, _, pages = P.batch(rng, [50, 20], [3, 4], 16)
    starts = np.array([5, 8, 12], np.int32)  # rows 0-4 and 12-19 belong to none
    q, k, v = draw(rng, (20, 4, 64), "bf16"), draw(rng, (20, 2, 64), "bf16"), draw(rng, (20, 2, 64), "bf16")
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 64), Q.random_cache(rng, pages, 16, 2, 64)
    ang = rng.standard_normal((50, 32)).astype(np.float32)
    (rq, tq), parts = Q.append(q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables, lens, starts, "bf16")
    got = run(f_append, q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables, lens, starts)
    close(got["output0"], rq, tq)
    assert (got["key_exps"] == parts[0][0]).all()
    close(Q.values(got["key_cache"], got["key_exps"]), parts[0][1], parts[0][2])


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def check_attend(rng, t, hq, hkv, d, page, lens, new, window, sinks, spoil=None, std=1.0, scale=None, exps=(-9, -4)):
    tables, lens, starts, pages = P.batch(rng, lens, new, page)
    n = int(starts[-1]) if starts is not None else len(lens)
    q = draw(rng, (n, hq, d), t, std)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, page, hkv, d, *exps), Q.random_cache(rng, pages, page, hkv, d, *exps)
    if spoil is not None:
        spoil(tables, lens, starts, kc, vc, ke, ve)
    got = run(f_attend, q, kc, vc, ke, ve, tables, lens, starts, window=window or None, sinks=sinks, scale=scale)["output0"]
    close(got, *Q.paged(q, kc, vc, ke, ve, tables, lens, starts, window, sinks, t, scale))


QUERY_HEADS = [(4, 2, 128), (5, 1, 128), (2, 2, 128), (16, 1, 128), (40, 2, 128), (8, 2, 64), (6, 2, 64), (3, 3, 64)]


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", QUERY_HEADS)
def test_attend_single_tokens(t, hq, hkv, d):
    check_attend(np.random.default_rng(41), t, hq, hkv, d, 16, [1, 300, 33, 0, 32, 129, 31, 700], None, 0, 0)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", QUERY_HEADS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5)])
def test_attend_prompts(t, hq, hkv, d, window, sinks):
    check_attend(np.random.default_rng(42), t, hq, hkv, d, 16, [70, 1, 0, 330, 129, 300], [70, 1, 0, 65, 128, 3], window, sinks)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 1000])
@pytest.mark.parametrize("new", [None, [5, 40, 1, 200]])
def test_attend_page_sizes(page, new):
    rng = np.random.default_rng(43)
    check_attend(rng, "bf16", 8, 2, 128, page, [90, 40, 513, 260], new, 0, 0)
    check_attend(rng, "bf16", 8, 2, 64, page, [90, 40, 513, 260], new, 70, 3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 32), (33, 40), (64, 1), (200, 63), (5000, 5000), (40, 600)])
@pytest.mark.parametrize("new", [None, [1, 1, 150, 333]])
def test_attend_windows(window, sinks, new):
    check_attend(np.random.default_rng(44), "bf16", 4, 1, 128, 16, [1, 65, 450, 1333], new, window, sinks)


@pytest.mark.parametrize("t,hq,hkv,d", [("f32", 4, 2, 128), ("f32", 3, 1, 64), ("bf16", 4, 2, 80), ("f16", 2, 1, 256),
                                        ("bf16", 6, 3, 5), ("f32", 2, 2, 1), ("bf16", 8, 2, 96)])
def test_attend_other_heads(t, hq, hkv, d):
    rng = np.random.default_rng(45)
    check_attend(rng, t, hq, hkv, d, 16, [70, 0, 150], [10, 0, 33], 50, 4)
    check_attend(rng, t, hq, hkv, d, 5, [70, 1, 150], None, 0, 0)


@pytest.mark.parametrize("new", [None, [300, 1, 40]])
def test_attend_long_contexts(new):
    """Keys split over workgroups and joined."""
    check_attend(np.random.default_rng(46), "bf16", 8, 2, 128, 16, [5000, 3000, 1], None if new is None else [300, 1, 1], 0, 0)
    check_attend(np.random.default_rng(47), "f16", 4, 1, 64, 16, [4111, 2, 900], None if new is None else [17, 2, 9], 0, 0)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("new", [None, [60, 1, 40]])
def test_attend_scales_far_apart(t, new):
    """Exponents that differ from page to page by more than a type's range, and
    outside their own."""

    def spoil(tables, lens, starts, kc, vc, ke, ve):
        ve[tables[0, :3]] = [[-40], [20], [-9]]
        ve[tables[2, 1]] = -700

    check_attend(np.random.default_rng(48), t, 4, 2, 128, 16, [77, 50, 290], new, 0, 0, spoil)
    check_attend(np.random.default_rng(48), t, 4, 2, 64, 16, [77, 50, 290], new, 0, 0, exps=(-14, 1), scale=0.002)


@pytest.mark.parametrize("new", [None, [40, 1, 130]])
@pytest.mark.parametrize("bad", [-1, -7, 10**6])
def test_attend_missing_pages(new, bad):
    def spoil(tables, lens, starts, kc, vc, ke, ve):
        tables[0, 0] = bad
        tables[2, 2:5] = bad
        tables[1] = bad
        lens[2] += 16 * tables.shape[1]

    check_attend(np.random.default_rng(49), "bf16", 4, 2, 128, 16, [77, 50, 290], new, 0, 0, spoil)

    def early(tables, lens, starts, kc, vc, ke, ve):
        lens[:] = [-5, 0, 100]

    check_attend(np.random.default_rng(50), "bf16", 4, 2, 128, 16, [77, 50, 290], new, 0, 0, early)


@pytest.mark.parametrize("t,d", [("bf16", 128), ("f16", 64), ("f32", 64)])
@pytest.mark.parametrize("new", [None, [40, 1, 130]])
def test_attend_nan_codes(t, d, new):
    """NaN where nobody looks enters nothing; where some queries look, it
    reaches those and no others."""
    rng = np.random.default_rng(51)
    tables, lens, starts, pages = P.batch(rng, [77, 50, 290], new, 16)
    n = int(starts[-1]) if new else 3
    q = draw(rng, (n, 4, d), t)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, d), Q.random_cache(rng, pages, 16, 2, d)
    kb, vb = kc.view(np.uint8), vc.view(np.uint8)
    free = np.setdiff1d(np.arange(pages), tables[tables >= 0])
    kb[free], vb[free] = 0x7F, 0xFF
    for b in range(3):  # behind the last token
        last = tables[b, (lens[b] - 1) // 16]
        kb[last, (lens[b] - 1) % 16 + 1:], vb[last, (lens[b] - 1) % 16 + 1:] = 0xFF, 0x7F
    vb[tables[2, 10], 3, 1, 5] = 0x7F   # key 163 of the third: only its head 1
    kb[tables[0, 3], 7, 0, 9] = 0x7F    # key 55 of the first
    want = P.up(f_attend(q, kc, vc, ke, ve, tables, lens, starts))
    got = run(f_attend, q, kc, vc, ke, ve, tables, lens, starts)["output0"]
    assert (np.isnan(P.up(got)) == np.isnan(want)).all()
    assert np.isnan(want).any() and not np.isnan(want).all()
    fine = np.where(np.isnan(want), 0, want)
    _, tol = Q.paged(q, np.where(np.isnan(Q.TABLE[kb]), 0, kb).astype(np.uint8).view(kc.dtype),
                     np.where(np.isnan(Q.TABLE[vb]), 0, vb).astype(np.uint8).view(vc.dtype), ke, ve, tables, lens, starts, 0, 0, t)
    # (the CPU form's own rounding: half a step)
    close(np.where(np.isnan(P.up(got)), 0, P.up(got)), fine, tol + P.HALF_STEP[t] * np.abs(fine))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("new", [None, [40, 1, 130]])
def test_attend_large_scores(t, new):
    """One key far ahead of the others, and offsets that grow along the keys."""
    rng = np.random.default_rng(52)
    tables, lens, starts, pages = P.batch(rng, [77, 50, 290], new, 16)
    n = int(starts[-1]) if new else 3
    q = P.cast(np.sign(rng.standard_normal((n, 4, 64))), t)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 64), Q.random_cache(rng, pages, 16, 2, 64)
    kc = (rng.integers(0x30, 0x38, kc.shape).astype(np.uint8) | (rng.integers(0, 2, kc.shape) << 7).astype(np.uint8)).view(kc.dtype)
    ke = rng.integers(0, 5, ke.shape).astype(np.int32)
    got = run(f_attend, q, kc, vc, ke, ve, tables, lens, starts)["output0"]
    close(got, *Q.paged(q, kc, vc, ke, ve, tables, lens, starts, 0, 0, t))


def test_attend_rows_outside_every_sequence():
    rng = np.random.default_rng(53)
    tables, lens, _, pages = P.batch(rng, [50, 20], [3, 4], 16)
    starts = np.array([5, 8, 12], np.int32)  # rows 0-4 and 12-19 belong to none
    for d in (128, 80):
        q = draw(rng, (20, 4, d), "bf16")
        (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, d), Q.random_cache(rng, pages, 16, 2, d)
        got = run(f_attend, q, kc, vc, ke, ve, tables, lens, starts)["output0"]
        assert (P.up(got)[:5] == 0).all() and (P.up(got)[12:] == 0).all()
        close(got, *Q.paged(q, kc, vc, ke, ve, tables, lens, starts, 0, 0, "bf16"))


def test_attend_many_sequences():
    rng = np.random.default_rng(54)
    new = [int(x) for x in rng.integers(0, 4, 200)]
    lens = [n + int(rng.integers(0, 90)) for n in new]
    check_attend(rng, "bf16", 4, 2, 64, 16, lens, new, 0, 0)
    check_attend(rng, "bf16", 4, 2, 64, 16, [max(x, 1) for x in lens], None, 40, 2)


@pytest.mark.parametrize("n", [256, 257, 700])
def test_attend_sequences_in_order_of_length_and_not(n):
    """As many sequences as a workgroup sorts, and more."""
    rng = np.random.default_rng(57)
    new = [int(x) for x in rng.integers(0, 3, n)]
    check_attend(rng, "bf16", 4, 2, 128, 16, [x + int(rng.integers(0, 60)) for x in new], new, 0, 0)


def test_attend_layouts():
    """A layer of one big cache, heads before rows, queries out of a projection."""
    rng = np.random.default_rng(55)
    tables, lens, starts, pages = P.batch(rng, [50, 70], [3, 70], 16)
    for new in (True, False):
        n = 73 if new else 2
        x = draw(rng, (n, 6, 64), "bf16")
        kb = np.stack([Q.random_cache(rng, pages, 16, 2, 64)[0] for _ in range(2)])
        vb = np.stack([Q.random_cache(rng, pages, 16, 2, 64)[0] for _ in range(2)])
        ke, ve = (rng.integers(-9, -4, (2, pages, 2)).astype(np.int32) for _ in range(2))
        kt = np.ascontiguousarray(kb.view(np.uint8)[1].transpose(0, 2, 1, 3)).view(kb.dtype)

        def f(x, kb, vb, ke, ve, tables, lens, starts=None):
            return T.paged_attention_fp8(x[:, :4], kb[1], vb[1], ke[1], ve[1], tables, lens, starts)

        def g(x, kt, vb, ke, ve, tables, lens, starts=None):
            return T.paged_attention_fp8(x[:, :4], kt.transpose(0, 2, 1, 3), vb[1], ke[1], ve[1], tables, lens, starts)

        s = starts if new else None
        want = Q.paged(x[:, :4], kb[1], vb[1], ke[1], ve[1], tables, lens, s, 0, 0, "bf16")
        close(run(f, x, kb, vb, ke, ve, tables, lens, s)["output0"], *want)
        close(run(g, x, kt, vb, ke, ve, tables, lens, s)["output0"], *want)


def test_steps_queue_and_repeat():
    """An append and the attention behind it in one kernel, replayed as a graph
    and queued, give what they give once."""
    rng = np.random.default_rng(56)
    tables, lens, _, pages = P.batch(rng, [50, 70, 1], None, 16)
    q, k, v = draw(rng, (3, 4, 128), "bf16"), draw(rng, (3, 2, 128), "bf16"), draw(rng, (3, 2, 128), "bf16")
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 128), Q.random_cache(rng, pages, 16, 2, 128)
    ang = rng.standard_normal((70, 64)).astype(np.float32)

    def f(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens):
        y = T.rotary_append_fp8(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens)
        return T.paged_attention_fp8(y, kc, vc, ke, ve, tables, lens)

    args = (q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables, lens)
    first = run(f, *args)
    dk, ins, outs = load(f, *args)
    for graph in (True, True, False, True):
        dk(ins, outs, graph=graph)
        for n, x in first.items():
            assert outs[n].numpy().tobytes() == x.tobytes()


@pytest.mark.parametrize("new", [None, [3, 60]])
def test_attend_heads_at_odd_addresses(new):
    """Caches whose heads are parts of longer ones: rows that fit no 16 bytes."""
    rng = np.random.default_rng(58)
    tables, lens, starts, pages = P.batch(rng, [50, 70], new, 16)
    q = draw(rng, (63 if new else 2, 4, 64), "bf16")
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 72), Q.random_cache(rng, pages, 16, 2, 72)

    def f(q, kc, vc, ke, ve, tables, lens, starts=None):
        return T.paged_attention_fp8(q, kc[:, :, :, 8:], vc[:, :, :, :64], ke, ve, tables, lens, starts)

    got = run(f, q, kc, vc, ke, ve, tables, lens, starts)["output0"]
    close(got, *Q.paged(q, kc[..., 8:], vc[..., :64], ke, ve, tables, lens, starts, 0, 0, "bf16"))


@pytest.mark.parametrize("half", [64, 32])
def test_append_behind_2_31_codes_of_a_page(half):
    """Rows of a page whose places pass 32 bits."""
    rng = np.random.default_rng(59)
    hkv, d, page = 128, 128, 2**17 + 24
    row = page - 9  # (131087 rows of 16384 codes before it)
    k, v = draw(rng, (1, hkv, d), "bf16"), draw(rng, (1, hkv, d), "bf16")
    kc, vc = (np.zeros((1, page, hkv, d), dt.float8_e4m3fn) for _ in range(2))
    ke, ve = (np.full((1, hkv), -5, np.int32) for _ in range(2))
    cos, sin = np.ones((page, half), np.float32), np.zeros((page, half), np.float32)
    dk, ins, outs = load(f_append, k, k, v, cos, sin, kc, vc, ke, ve, np.zeros((1, 1), np.int32),
                         np.array([row + 1], np.int32))
    dk(ins, outs)
    for name, x in (("key", k), ("value", v)):
        assert (outs[name + "_exps"].numpy() == -5).all()  # (up to 14 in magnitude)
        got = outs[name + "_cache"].numpy()
        y = P.up(x)[0]
        close(Q.values(got[:, row:row + 1], np.full((1, hkv), -5))[0, 0], y, np.maximum(np.abs(y) * 2.0**-4, 2.0**-15))
        z = Q.bits(got)
        assert z[0, row].any()
        z[0, row] = 0
        assert not z.any()


def test_caches_past_2_31_bytes():
    """Pages whose places pass 32 bits: appended to, then read by single tokens
    and by a prompt."""
    rng = np.random.default_rng(60)
    hkv, d, page, few = 8, 128, 16, 64
    pages = 2**17 + few
    small = [Q.random_cache(rng, few, page, hkv, d) for _ in range(2)]
    caches, exps = [], []
    for codes, e in small:
        big = np.zeros((pages, page, hkv, d), codes.dtype)
        big[-few:] = codes
        caches.append(big)
        exps.append(np.concatenate([np.full((pages - few, hkv), 9, np.int32), e]))
    ang = rng.standard_normal((600, 64)).astype(np.float32)

    def f(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, tables, lens, starts=None):
        y = T.rotary_append_fp8(q, k, v, cos, sin, key_cache, value_cache, key_exps, value_exps, tables, lens, starts)
        return y, T.paged_attention_fp8(y, key_cache, value_cache, key_exps, value_exps, tables, lens, starts)

    for new in (None, [140, 3]):
        tables, lens, starts, n = P.batch(rng, [500, 200], new, page)
        assert n <= few
        t = 143 if new else 2
        q, k, v = draw(rng, (t, 16, d), "bf16"), draw(rng, (t, hkv, d), "bf16"), draw(rng, (t, hkv, d), "bf16")
        (kc, ke), (vc, ve) = small
        (rq, tq), parts = Q.append(q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables, lens, starts, "bf16")
        got = run(f, q, k, v, np.cos(ang), np.sin(ang), *caches, *exps, np.where(tables < 0, -1, tables + pages - few).astype(np.int32),
                  lens, starts)
        close(got["output0"], rq, tq)
        for name, (e, val, tol, _) in (("key", parts[0]), ("value", parts[1])):
            assert (got[name + "_exps"][-few:] == e).all() and (got[name + "_exps"][:-few] == 9).all()
            close(Q.values(got[name + "_cache"][-few:], got[name + "_exps"][-few:]), val, tol)
            assert not Q.bits(got[name + "_cache"][:-few]).any()
        close(got["output1"], *Q.paged(got["output0"], got["key_cache"][-few:], got["value_cache"][-few:],
                                       got["key_exps"][-few:], got["value_exps"][-few:], tables, lens, starts, 0, 0, "bf16"))


def test_starts_in_no_order():
    """Query starts that decrease or lie outside the tokens change nothing else:
    the call behind gives what it always does."""
    rng = np.random.default_rng(61)
    tables, lens, starts, pages = P.batch(rng, [50, 70, 20], [3, 4, 5], 16)
    q, k, v = (draw(rng, (12, h, 64), "bf16") for h in (4, 2, 2))
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 64), Q.random_cache(rng, pages, 16, 2, 64)
    ang = rng.standard_normal((100, 32)).astype(np.float32)

    def f(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts):
        y = T.rotary_append_fp8(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts)
        return T.paged_attention_fp8(y, kc, vc, ke, ve, tables, lens, starts)

    args = (q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables)
    first = run(f, *args, lens, starts)
    far = [2**31 - 1, -2**31]
    for s in ([0, 9, 3, 12], [-5, far[0], 0, far[0]], [7, 7, 7, 7], [12, 0, 0, 0], [far[0], far[1], far[0], 3]):
        for n in (lens, np.array([far[0], far[1], 7], np.int32)):
            got = run(f, *args, n, np.array(s, np.int32))
            held = np.unique(tables[tables >= 0])
            others = np.setdiff1d(np.arange(pages), held)
            for name, x in (("kc", kc), ("vc", vc)):  # (pages of nobody)
                assert (Q.bits(got[name])[others] == Q.bits(x)[others]).all()
    again = run(f, *args, lens, starts)
    assert all(again[n].tobytes() == first[n].tobytes() for n in first)


def test_two_sets_of_tensors_replayed_in_turns():
    """Two graphs of one kernel share its workspace (the splits of a step)."""
    rng = np.random.default_rng(62)
    sets = []
    dk = None
    for _ in range(2):
        tables, lens, _, pages = P.batch(rng, [700, 90, 1500], None, 16)
        q = draw(rng, (3, 8, 128), "bf16")
        (kc, ke), (vc, ve) = Q.random_cache(rng, 160, 16, 2, 128), Q.random_cache(rng, 160, 16, 2, 128)
        tables = np.pad(tables, ((0, 0), (0, 100 - tables.shape[1])), constant_values=-1)
        one, ins, outs = load(f_attend, q, kc, vc, ke, ve, tables, lens)
        dk = dk or one
        sets.append((ins, outs, Q.paged(q, kc, vc, ke, ve, tables, lens, None, 0, 0, "bf16")))
    for _ in range(3):
        for ins, outs, want in sets:
            dk(ins, outs, graph=True, sync=False)
        for ins, outs, want in sets:
            close(outs["output0"].numpy(), *want)


def test_exponents_overwritten_behind_an_append():
    """An array that the kernel writes again: the append updates a copy of it."""
    rng = np.random.default_rng(63)
    tables, lens, starts, pages = P.batch(rng, [30, 20], [7, 20], 16)
    q, k, v = (draw(rng, (27, h, 64), "bf16") for h in (4, 2, 2))
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, 2, 64), Q.random_cache(rng, pages, 16, 2, 64)
    ang = rng.standard_normal((30, 32)).astype(np.float32)

    def f(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts):
        T.rotary_append_fp8(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, starts)
        seen = ke + 1
        ke[:] = 7
        return seen

    _, parts = Q.append(q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables, lens, starts, "bf16")
    got = run(f, q, k, v, np.cos(ang), np.sin(ang), kc, vc, ke, ve, tables, lens, starts)
    assert (got["output0"] == parts[0][0] + 1).all() and (got["ke"] == 7).all() and (got["ve"] == parts[1][0]).all()
    close(Q.values(got["kc"], parts[0][0]), parts[0][1], parts[0][2])
