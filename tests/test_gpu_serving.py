"""The serving operators on the GPU against plain 64-bit forms."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.runtime import DeviceKernel, DeviceTensor

import serving_plain as P

pytestmark = pytest.mark.gpu


def load(f, *args, **kw):
    """(kernel, inputs, outputs) of ``f`` on device copies of the arrays."""
    import inspect

    dk = DeviceKernel.compile_and_load(f, *args, use_cached_if_exists=False, **kw)
    bound = inspect.signature(f).bind(*args, **kw).arguments
    dev = {n: x if isinstance(x, DeviceTensor) else DeviceTensor.from_numpy(x, name=n) for n, x in bound.items()
           if hasattr(x, "shape")}
    ins = {n: dev[n.split(".must_alias_input")[0]] for n in dk.input_tensors_info}
    outs = {n: dev[n] if n in dev else DeviceTensor.empty(tuple(m.shape), m.dtype, name=n)
            for n, m in dk.output_tensors_info.items()}
    return dk, ins, outs


def run(f, *args, **kw):
    dk, ins, outs = load(f, *args, **kw)
    dk(ins, outs)
    return {n: x.numpy() for n, x in outs.items()}


def draw(rng, shape, t, std=1.0):
    return P.cast(rng.standard_normal(shape).astype(np.float32) * np.float32(std), t)


def close(got, want, tol):
    e = np.abs(P.up(got) - want)
    bad = ~(e <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}, worst by {np.max(np.where(bad, e, 0))}"


def f_paged(q, kc, vc, tables, lens, starts=None, window=None, sinks=0, scale=None):
    return T.paged_attention(q, kc, vc, tables, lens, starts, window=window, sinks=sinks, scale=scale)


def check_paged(rng, t, hq, hkv, d, page, lens, new, window, sinks, spoil=None, std=1.0):
    tables, lens, starts, pages = P.batch(rng, lens, new, page)
    n = int(starts[-1]) if starts is not None else len(lens)
    q = draw(rng, (n, hq, d), t, std)
    kc, vc = draw(rng, (pages, page, hkv, d), t), draw(rng, (pages, page, hkv, d), t)
    if spoil is not None:
        spoil(tables, lens, starts, kc, vc)
    got = run(f_paged, q, kc, vc, tables, lens, starts, window=window or None, sinks=sinks)["output0"]
    close(got, *P.paged(q, kc, vc, tables, lens, starts, window, sinks, t))


# ---------------------------------------------------------------------------
# Paged attention
# ---------------------------------------------------------------------------
HEADS = [(4, 2, 128), (5, 1, 128), (2, 2, 128), (16, 1, 128), (40, 8, 128), (8, 2, 64), (6, 2, 64), (3, 3, 64)]


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_paged_single_tokens(t, hq, hkv, d):
    rng = np.random.default_rng(11)
    check_paged(rng, t, hq, hkv, d, 16, [1, 300, 33, 0, 32, 129, 31, 700], None, 0, 0)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5)])
def test_paged_prompts(t, hq, hkv, d, window, sinks):
    rng = np.random.default_rng(12)
    check_paged(rng, t, hq, hkv, d, 16, [70, 1, 0, 330, 129, 300], [70, 1, 0, 65, 128, 3], window, sinks)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 1000])
@pytest.mark.parametrize("new", [None, [5, 40, 1, 200]])
def test_paged_page_sizes(page, new):
    rng = np.random.default_rng(13)
    check_paged(rng, "bf16", 8, 2, 128, page, [90, 40, 513, 260], new, 0, 0)
    check_paged(rng, "bf16", 8, 2, 64, page, [90, 40, 513, 260], new, 70, 3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 32), (33, 40), (64, 1), (200, 63), (5000, 5000), (40, 600)])
@pytest.mark.parametrize("new", [None, [1, 1, 150, 333]])
def test_paged_windows(window, sinks, new):
    rng = np.random.default_rng(14)
    check_paged(rng, "bf16", 4, 1, 128, 16, [1, 65, 450, 1333], new, window, sinks)


@pytest.mark.parametrize("t,hq,hkv,d", [("f32", 4, 2, 128), ("f32", 3, 1, 64), ("bf16", 4, 2, 80), ("f16", 2, 1, 256),
                                        ("bf16", 6, 3, 5), ("f32", 2, 2, 1), ("bf16", 8, 2, 96)])
def test_paged_other_heads(t, hq, hkv, d):
    rng = np.random.default_rng(15)
    check_paged(rng, t, hq, hkv, d, 16, [70, 0, 150], [10, 0, 33], 50, 4)
    check_paged(rng, t, hq, hkv, d, 5, [70, 1, 150], None, 0, 0)


def test_paged_many_sequences():
    """More sequences than lanes look for theirs at once."""
    rng = np.random.default_rng(16)
    new = [int(x) for x in rng.integers(0, 4, 200)]
    lens = [n + int(rng.integers(0, 90)) for n in new]
    check_paged(rng, "bf16", 4, 2, 64, 16, lens, new, 0, 0)
    check_paged(rng, "bf16", 4, 2, 64, 16, [max(x, 1) for x in lens], None, 40, 2)


def test_paged_rows_outside_every_sequence():
    rng = np.random.default_rng(17)
    tables, lens, _, pages = P.batch(rng, [50, 20], [3, 4], 16)
    starts = np.array([5, 8, 12], np.int32)  # rows 0-4 and 12-19 belong to none
    q, kc, vc = draw(rng, (20, 4, 128), "bf16"), draw(rng, (pages, 16, 2, 128), "bf16"), draw(rng, (pages, 16, 2, 128), "bf16")
    got = P.up(run(f_paged, q, kc, vc, tables, lens, starts)["output0"])
    assert (got[:5] == 0).all() and (got[12:] == 0).all()
    close(P.cast(got, "f32"), *P.paged(q, kc, vc, tables, lens, starts, 0, 0, "bf16"))


@pytest.mark.parametrize("new", [None, [40, 1, 130]])
@pytest.mark.parametrize("bad", [-1, -7, 10**6])
def test_paged_missing_pages(new, bad):
    """Pages that are none, at the start, in the middle and as a whole
    sequence; lengths past the table; queries before position 0."""
    rng = np.random.default_rng(18)

    def spoil(tables, lens, starts, kc, vc):
        tables[0, 0] = bad
        tables[2, 2:5] = bad
        tables[1] = bad
        lens[2] += 16 * tables.shape[1]

    check_paged(rng, "bf16", 4, 2, 128, 16, [77, 50, 290], new, 0, 0, spoil)

    def early(tables, lens, starts, kc, vc):
        lens[:] = [-5, 0, 100]

    check_paged(rng, "bf16", 4, 2, 64, 16, [77, 50, 290], new, 30, 2, early)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [None, [9, 300]])
def test_paged_spoiled_rows_unseen(new, d):
    """NaN and infinities where no query looks: cache rows past the lengths,
    behind the window, pages of others."""
    rng = np.random.default_rng(19)

    def spoil(tables, lens, starts, kc, vc):
        page, width = kc.shape[1], tables.shape[1]
        used = np.zeros(kc.shape[:2], bool)
        for b in range(len(lens)):
            n = 1 if starts is None else starts[b + 1] - starts[b]
            for j in range(lens[b]):
                if j < 3 or j > lens[b] - n - 50:
                    used[tables[b, j // page], j % page] = True
        junk = P.cast(np.array([np.nan, np.inf, -np.inf], np.float32), "bf16")
        for x in (kc, vc):
            x[~used] = junk[rng.integers(0, 3, x[~used].shape)]

    check_paged(rng, "bf16", 4, 2, d, 16, [200, 411], new, 50, 3, spoil)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_paged_spoiled_value_seen_by_some(value, d):
    """A value that is not finite reaches the queries that see its key and no
    other of their tile."""
    rng = np.random.default_rng(20)
    t = "bf16"
    tables, lens, starts, pages = P.batch(rng, [150, 90], [150, 20], 16)
    q, kc, vc = draw(rng, (170, 4, d), t), draw(rng, (pages, 16, 2, d), t), draw(rng, (pages, 16, 2, d), t)
    at = tables[0, 100 // 16], 100 % 16
    vc[at][1, 7] = P.cast(np.float32(value), t)
    clean = vc.copy()
    clean[at][1, 7] = P.cast(np.float32(0), t)
    got = P.up(run(f_paged, q, kc, vc, tables, lens, starts, window=30)["output0"])
    want, tol = P.paged(q, kc, clean, tables, lens, starts, 30, 0, t)
    hit = np.zeros(got.shape, bool)
    hit[100:130, 2:, 7] = True
    assert (np.isnan(got[hit]).all() if np.isnan(value) else (got[hit] == value).all())
    assert (np.abs(got - want)[~hit] <= tol[~hit]).all()


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_paged_wide_scores(t):
    """Scores far apart: weights that all but vanish, a maximum that comes
    late, one that comes first."""
    rng = np.random.default_rng(21)
    for sign in (1, -1):
        def slope(tables, lens, starts, kc, vc):
            page = kc.shape[1]
            for b in range(len(lens)):
                for j in range(lens[b]):
                    i = tables[b, j // page], j % page
                    kc[i] = P.cast(P.up(kc[i]) * 0.2 + sign * 3.0 * (j / lens[b] - 0.5), t)

        check_paged(rng, t, 4, 1, 64, 16, [500, 900], [40, 200], 0, 0, slope, 4.0)
        check_paged(rng, t, 4, 1, 64, 16, [500, 900], None, 0, 0, slope, 4.0)


@pytest.mark.parametrize("layout", ["pairs", "heads_first", "layers"])
def test_paged_strided_caches(layout):
    """Caches that are views: keys and values of a page side by side, heads
    before rows, one layer of several."""
    rng = np.random.default_rng(22)
    tables, lens, starts, pages = P.batch(rng, [90, 40], [7, 40], 16)
    q = draw(rng, (47, 4, 128), "bf16")
    if layout == "pairs":
        kv = draw(rng, (pages, 2, 16, 2, 128), "bf16")
        f = lambda q, kv, t, n, s: T.paged_attention(q, kv[:, 0], kv[:, 1], t, n, s)  # noqa: E731
        kc, vc = kv[:, 0], kv[:, 1]
    elif layout == "heads_first":
        kv = draw(rng, (2, pages, 2, 16, 128), "bf16")
        f = lambda q, kv, t, n, s: T.paged_attention(q, kv[0].transpose(0, 2, 1, 3), kv[1].transpose(0, 2, 1, 3), t, n, s)  # noqa: E731
        kc, vc = kv[0].transpose(0, 2, 1, 3), kv[1].transpose(0, 2, 1, 3)
    else:
        kv = draw(rng, (3, 2, pages, 16, 2, 128), "bf16")
        f = lambda q, kv, t, n, s: T.paged_attention(q, kv[1, 0], kv[1, 1], t, n, s)  # noqa: E731
        kc, vc = kv[1, 0], kv[1, 1]
    got = run(f, q, kv, tables, lens, starts)["output0"]
    close(got, *P.paged(q, kc, vc, tables, lens, starts, 0, 0, "bf16"))


def test_paged_far_pages():
    """Pages whose rows lie past 2^32 bytes and elements of the cache."""
    rng = np.random.default_rng(23)
    pages, page, hkv, d = 2**21 + 40, 16, 1, 128  # 8.6 GB, 4.3e9 elements
    t = "bf16"
    kd, vd = (DeviceTensor.empty((pages, page, hkv, d), dt.bfloat16, name=n) for n in ("kc", "vc"))
    tables = np.array([[pages - 1, 3, pages - 9], [2**20 + 5, pages - 4, -1]], np.int32)
    lens = np.array([45, 32], np.int32)
    small, stables, at = [np.zeros((6, page, hkv, d), dt.bfloat16) for _ in range(2)], np.full((2, 3), -1, np.int32), 0
    for b in range(2):
        for i in range(3):
            if tables[b, i] < 0:
                continue
            for x, dev in zip(small, (kd, vd)):
                x[at] = draw(rng, (page, hkv, d), t)
                raw = np.ascontiguousarray(x[at].view(np.uint16))
                dev.tensor_ref.write(raw.ctypes.data, raw.nbytes, int(tables[b, i]) * raw.nbytes)
            stables[b, i] = at
            at += 1
    for starts, n in ((None, 2), (np.array([0, 12, 20], np.int32), 20)):
        q = draw(rng, (n, 4, d), t)
        got = run(f_paged, q, kd, vd, tables, lens, starts)["output0"]
        close(got, *P.paged(q, small[0], small[1], stables, lens, starts, 0, 0, t))

    def f(q, k, v, cos, sin, kc, vc, tables, lens):
        return T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens)

    cos, sin = np.ones((64, 64), np.float32), np.zeros((64, 64), np.float32)
    k, v = draw(rng, (2, hkv, d), t), draw(rng, (2, hkv, d), t)
    dk, ins, outs = load(f, draw(rng, (2, 4, d), t), k, v, cos, sin, kd, vd, tables, lens)
    dk(ins, outs)
    for x, dev in ((k, kd), (v, vd)):
        for b, p in ((0, 44), (1, 31)):
            raw = np.zeros((1, hkv, d), np.uint16)
            dev.tensor_ref.read(raw.ctypes.data, raw.nbytes, int(tables[b, p // page]) * page * hkv * d * 2 + p % page * hkv * d * 2)
            assert (raw[0] == x[b].view(np.uint16)).all()


@pytest.mark.parametrize("hq,hkv,d", [(40, 2, 64), (17, 1, 128), (160, 1, 64), (256, 2, 128)])
@pytest.mark.parametrize("new", [None, [1, 9, 2]])
def test_paged_large_groups(hq, hkv, d, new):
    """More heads of a group than a step's workgroup takes, and than a tile has rows."""
    rng = np.random.default_rng(24)
    check_paged(rng, "bf16", hq, hkv, d, 16, [70, 9, 300], new, 0, 0)
    check_paged(rng, "f16", hq, hkv, d, 16, [70, 9, 300], new, 33, 2)


@pytest.mark.parametrize("seqs,hq,hkv,length", [(1, 4, 2, 9000), (40, 32, 1, 2100), (3, 8, 1, 6000)])
def test_paged_split_keys(seqs, hq, hkv, length):
    """Splits joined by a workgroup for each row, and by a wave where rows are many;
    short sequences beside the long one, which have no part in most splits."""
    rng = np.random.default_rng(25)
    lens = [length] + [int(x) for x in rng.integers(0, 400, seqs - 1)]
    check_paged(rng, "bf16", hq, hkv, 64, 32, lens, None, 0, 0)
    check_paged(rng, "bf16", hq, hkv, 64, 32, lens, [min(9, x) for x in lens], 0, 0)


def test_paged_unordered_starts_stay_inside():
    """Starts and lengths that make no sense read and write nothing outside
    the tensors (the results are of no use)."""
    rng = np.random.default_rng(24)
    tables, lens, _, pages = P.batch(rng, [50, 20, 90], [3, 4, 5], 16)
    q, kc, vc = draw(rng, (12, 4, 128), "bf16"), draw(rng, (pages, 16, 2, 128), "bf16"), draw(rng, (pages, 16, 2, 128), "bf16")
    for starts in ([0, 9, 3, 12], [-5, 2**31 - 1, 0, 2**31 - 1], [7, 7, 7, 7], [12, 0, 0, 0]):
        for ls in (lens, np.array([2**31 - 1, -2**31, 7], np.int32)):
            run(f_paged, q, kc, vc, tables, ls, np.array(starts, np.int64).astype(np.int32), window=20, sinks=1)


# ---------------------------------------------------------------------------
# Window attention
# ---------------------------------------------------------------------------
def f_window(q, k, v, lengths=None, positions=None, window=None, sinks=0, scale=None):
    return T.window_attention(q, k, v, lengths, positions, window=window, sinks=sinks, scale=scale)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (5, 1, 128), (8, 8, 64), (6, 2, 64)])
@pytest.mark.parametrize("B,S,K", [(1, 1, 1), (2, 1, 300), (3, 37, 37), (2, 128, 128), (1, 333, 400), (2, 5, 2), (1, 700, 700)])
def test_window(t, hq, hkv, d, B, S, K):
    rng = np.random.default_rng(31)
    q, k, v = draw(rng, (B, S, hq, d), t), draw(rng, (B, K, hkv, d), t), draw(rng, (B, K, hkv, d), t)
    for window, sinks in ((0, 0), (50, 3)):
        got = run(f_window, q, k, v, window=window or None, sinks=sinks)["output0"]
        close(got, *P.dense(q, k, v, None, None, window, sinks, t))


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 9), (33, 400)])
def test_window_lengths_and_positions(window, sinks):
    """Padded batches, generation into a plain cache, lengths and positions
    outside the tensors."""
    rng = np.random.default_rng(32)
    q, k, v = (draw(rng, (5, s, h, 128), "bf16") for s, h in ((90, 4), (350, 2), (350, 2)))
    lengths = np.array([350, 0, 61, 400, -3], np.int32)
    positions = np.array([0, 5, -40, 300, 2**31 - 1], np.int32)
    for a, b in ((lengths, None), (None, positions), (lengths, positions)):
        got = run(f_window, q, k, v, a, b, window=window or None, sinks=sinks)["output0"]
        close(got, *P.dense(q, k, v, a, None if b is None else b.astype(np.int64), window, sinks, "bf16"))


def test_window_strides():
    """Heads sliced out of a projection, heads before rows, and rows that lie
    where no 16-byte access can."""
    rng = np.random.default_rng(33)
    x = draw(rng, (2, 150, 8, 64), "bf16")
    want = P.dense(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], None, None, 40, 2, "bf16")
    f = lambda x: T.window_attention(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], window=40, sinks=2)  # noqa: E731
    close(run(f, x)["output0"], *want)
    f = lambda x: T.window_attention(*(x.transpose(0, 2, 1, 3)[:, :, a:b] for a, b in ((0, 4), (4, 6), (6, 8))), window=40, sinks=2)  # noqa: E731
    close(run(f, np.ascontiguousarray(x.transpose(0, 2, 1, 3)))["output0"], *want)
    y = np.zeros((2, 150, 8 * 64 + 3), dt.bfloat16)
    y[:, :, 3:] = x.reshape(2, 150, -1)
    def g(y):
        z = y[:, :, 3:].reshape(2, 150, 8, 64)
        return T.window_attention(z[:, :, :4], z[:, :, 4:6], z[:, :, 6:], window=40, sinks=2)
    close(run(g, y)["output0"], *want)


def test_window_scale_and_long():
    rng = np.random.default_rng(34)
    q, k, v = (draw(rng, (1, 2500, h, 64), "bf16") for h in (2, 1, 1))
    got = run(f_window, q, k, v, window=700, sinks=40, scale=0.3)["output0"]
    close(got, *P.dense(q, k, v, None, None, 700, 40, "bf16", 0.3))


def test_window_spoiled_keys_unseen():
    rng = np.random.default_rng(35)
    q, k, v = (draw(rng, (2, 200, h, 128), "f16") for h in (4, 2, 2))
    lengths = np.array([200, 77], np.int32)
    want = P.dense(q, k, v, lengths, None, 64, 0, "f16")
    k[1, 77:], v[1, 77:] = np.float16(np.nan), np.float16(np.inf)
    close(run(f_window, q, k, v, lengths, window=64)["output0"], *want)


@pytest.mark.parametrize("t,d", [("bf16", 64), ("f16", 128), ("f32", 32)])
def test_window_without_keys(t, d):
    rng = np.random.default_rng(39)
    for S in (1, 5, 200):
        f = lambda q, k, v: T.window_attention(q, k[:, 3:3], v[:, 3:3])  # noqa: E731
        q, k = draw(rng, (2, S, 4, d), t), draw(rng, (2, 7, 2, d), t)
        assert (P.up(run(f, q, k, k)["output0"]) == 0).all()


@pytest.mark.parametrize("t,d", [("bf16", 64), ("f16", 128), ("bf16", 128)])
def test_window_single_tokens(t, d):
    """One query of each sequence over plain keys of their own lengths."""
    rng = np.random.default_rng(36)
    q, k, v = (draw(rng, (4, s, h, d), t) for s, h in ((1, 6), (777, 2), (777, 2)))
    lengths, positions = np.array([777, 0, 300, 5], np.int32), np.array([776, 3, 299, 900], np.int32)
    for a, b in ((None, None), (lengths, positions), (None, positions), (lengths, None)):
        for window, sinks in ((0, 0), (130, 7)):
            got = run(f_window, q, k, v, a, b, window=window or None, sinks=sinks)["output0"]
            close(got, *P.dense(q, k, v, a, None if b is None else b.astype(np.int64), window, sinks, t))


@pytest.mark.parametrize("t,d,big", [("bf16", 64, 1e12), ("bf16", 128, 1e17), ("f16", 64, 6e4), ("f16", 128, 3e4), ("f32", 48, 1e15)])
@pytest.mark.parametrize("S", [1, 40, 130])
@pytest.mark.parametrize("K", [130, 3000])
def test_window_huge_scores(t, d, big, S, K):
    """Scores far past where 32 bits hold their differences: the largest alone has
    weight, equal ones share it."""
    rng = np.random.default_rng(40)
    v = P.cast(rng.integers(-8, 8, (2, K, 2, d)).astype(np.float32), t)
    q, k = np.full((2, S, 4, d), big, np.float32), np.ones((2, K, 2, d), np.float32)
    k[0, 70] = 2.0  # (every query sees it where S < 60)
    q[:, :, 1] *= -1
    k[1, :, 1] *= -1
    want, tol = P.dense(*(P.cast(x, t) for x in (q, k)), v, None, None, 0, 0, t)
    # among equal scores: at most 8, by the roundings of weights, sums and result
    close(run(f_window, P.cast(q, t), P.cast(k, t), v)["output0"], want, np.minimum(tol, 8 * 4 * 2.0**-8))


@pytest.mark.parametrize("S", [1, 50])
def test_window_broadcast_keys(S):
    """Keys and values that all sequences share, and one row that is every key."""
    rng = np.random.default_rng(37)
    q, k, v, one = (draw(rng, (b, s, h, 64), "bf16") for b, s, h in ((3, S, 4), (1, 90, 2), (1, 90, 2), (1, 1, 2)))
    f = lambda q, k, v: T.window_attention(q, np.broadcast_to(k, (3, 90, 2, 64)), np.broadcast_to(v, (3, 90, 2, 64)))  # noqa: E731
    for a in (k, one):
        keys, vals = (np.ascontiguousarray(np.broadcast_to(x, (3, 90, 2, 64))) for x in (a, v))
        close(run(f, q, a, v)["output0"], *P.dense(q, keys, vals, None, None, 0, 0, "bf16"))
        close(run(f, q, v, a)["output0"], *P.dense(q, vals, keys, None, None, 0, 0, "bf16"))


@pytest.mark.parametrize("d", [64, 128])
def test_window_far_rows(d):
    """Keys 16 MB apart, so that the last lie past 2^32 bytes."""
    rng = np.random.default_rng(38)
    wide = 2**23 // d
    kd, vd = (DeviceTensor.empty((1, 300, wide, d), dt.bfloat16, name=n) for n in ("k", "v"))
    k, v = draw(rng, (1, 300, 2, d), "bf16"), draw(rng, (1, 300, 2, d), "bf16")
    for x, dev in ((k, kd), (v, vd)):
        for j in range(300):
            raw = np.ascontiguousarray(x[0, j].view(np.uint16))
            dev.tensor_ref.write(raw.ctypes.data, raw.nbytes, j * 2**24)
    f = lambda q, k, v: T.window_attention(q, k[:, :, :2], v[:, :, :2], window=200, sinks=3)  # noqa: E731
    for S in (1, 280):
        q = draw(rng, (1, S, 4, d), "bf16")
        close(run(f, q, kd, vd)["output0"], *P.dense(q, k, v, None, None, 200, 3, "bf16"))


# ---------------------------------------------------------------------------
# Rotation and append
# ---------------------------------------------------------------------------
def f_append(q, k, v, cos, sin, kc, vc, tables, lens, starts=None):
    return T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens, starts)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,half", [(4, 2, 128, 64), (8, 1, 64, 16), (3, 3, 40, 20), (2, 1, 6, 2), (5, 5, 256, 128), (1, 1, 2, 1)])
@pytest.mark.parametrize("new", [None, [40, 0, 1, 77]])
def test_append(t, hq, hkv, d, half, new):
    rng = np.random.default_rng(41)
    tables, lens, starts, pages = P.batch(rng, [60, 3, 1, 100], new, 16 if hq != 3 else 7)
    n, page = (4 if new is None else sum(new)), 16 if hq != 3 else 7
    q, k, v = (draw(rng, (n, h, d), t) for h in (hq, hkv, hkv))
    kc, vc = (draw(rng, (pages, page, hkv, d), t) for _ in range(2))
    ang = (rng.random((100, half)) * 7).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    want, tol = P.append(q, k, v, cos, sin, kc, vc, tables, lens, starts, t)
    got = run(f_append, q, k, v, cos, sin, kc, vc, tables, lens, starts)
    for name, w, e in zip(("output0", "kc", "vc"), want, tol):
        close(got[name], w, e)


def test_append_dropped_tokens():
    """Positions outside the tables, pages that are none, rows outside every
    sequence: nothing is written for them; NaN of other tokens stays there."""
    rng = np.random.default_rng(42)
    t = "bf16"
    tables, lens, _, pages = P.batch(rng, [60, 30, 50], [6, 30, 4], 16)
    starts = np.array([2, 8, 38, 42], np.int32)
    tables[1, 1] = -1
    tables[0, 3] = pages
    lens[2] = 2  # its first tokens would sit before position 0
    q, k, v = (draw(rng, (45, h, 64), t) for h in (4, 2, 2))
    for x in (q, k, v):
        x[[0, 1, 42, 43, 44]] = P.cast(np.float32(np.nan), t)
    kc, vc = (draw(rng, (pages, 16, 2, 64), t) for _ in range(2))
    ang = (rng.random((58, 32)) * 7).astype(np.float32)  # positions 58, 59 have no row
    cos, sin = np.cos(ang), np.sin(ang)
    want, tol = P.append(q, k, v, cos, sin, kc, vc, tables, lens, starts, t)
    got = run(f_append, q, k, v, cos, sin, kc, vc, tables, lens, starts)
    for name, w, e in zip(("output0", "kc", "vc"), want, tol):
        close(got[name], w, e)


def test_append_twice():
    """Two calls of one kernel, other tables for the second: into caches of their
    own, and into the same ones."""
    rng = np.random.default_rng(46)
    t, n = "f32", 6
    tables, lens, starts, pages = P.batch(rng, [9, 30], [2, 4], 8)
    x = [draw(rng, (n, h, 64), t) for h in (4, 2, 2, 4, 2, 2)]
    ang = [np.outer(np.arange(40), b ** np.arange(m)).astype(np.float32) for b, m in ((0.6, 32), (0.3, 16))]
    trig = [f(a) for a in ang for f in (np.cos, np.sin)]
    caches = [draw(rng, (pages, 8, 2, 64), t) for _ in range(4)]

    def apart(q, k, v, q2, k2, v2, cos, sin, cos2, sin2, kc, vc, kc2, vc2, tables, lens, starts):
        T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens, starts)
        return T.rotary_append(q2, k2, v2, cos2, sin2, kc2, vc2, tables, lens, starts)

    got = run(apart, *x, *trig, *caches, tables, lens, starts)
    one = P.append(*x[:3], *trig[:2], *caches[:2], tables, lens, starts, t)
    two = P.append(*x[3:], *trig[2:], *caches[2:], tables, lens, starts, t)
    for g, w, e in zip((got[k] for k in ("output0", "kc", "vc", "kc2", "vc2")), (two[0][0], *one[0][1:], *two[0][1:]),
                       (two[1][0], *one[1][1:], *two[1][1:])):
        close(g, w, e)

    def same(q, k, v, q2, k2, v2, cos, sin, cos2, sin2, kc, vc, tables, lens, later, starts):
        a = T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens, starts)
        old = kc + 0.0
        return a, T.rotary_append(q2, k2, v2, cos2, sin2, kc, vc, tables, later, starts), old

    later = lens + np.array([2, 1], np.int32)  # (the second over part of the first's rows)
    wide = P.batch(rng, [11, 31], [2, 4], 8)[0]
    tables = np.arange(wide.size, dtype=np.int32).reshape(wide.shape)
    caches = [draw(rng, (wide.size, 8, 2, 64), t) for _ in range(2)]
    got = run(same, *x, *trig, *caches, tables, lens, later, starts)
    one = P.append(*x[:3], *trig[:2], *caches, tables, lens, starts, t)
    mid = [P.cast(a, t) for a in one[0][1:]]
    two = P.append(*x[3:], *trig[2:], *mid, tables, later, starts, t)
    for name, w, e in (("output0", one[0][0], one[1][0]), ("output1", two[0][0], two[1][0]), ("output2", one[0][1], one[1][1])):
        close(got[name], w, e)
    # (rows of the first call that stay are rounded already)
    close(got["kc"], two[0][1], two[1][1] + one[1][1] * 2)
    close(got["vc"], two[0][2], two[1][2])


def test_append_many_sequences_strided():
    rng = np.random.default_rng(43)
    new = [int(x) for x in rng.integers(0, 5, 150)]
    lens = [n + int(rng.integers(0, 60)) for n in new]
    tables, lens, starts, pages = P.batch(rng, lens, new, 16)
    x = draw(rng, (int(starts[-1]), 8, 64), "bf16")
    kc, vc = (draw(rng, (pages, 16, 2, 64), "bf16") for _ in range(2))
    ang = (rng.random((100, 32)) * 7).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    f = lambda x, cos, sin, kc, vc, tables, lens, starts: T.rotary_append(  # noqa: E731
        x[:, 2:6], x[:, 6:], x[:, :2], cos, sin, kc, vc, tables, lens, starts)
    want, tol = P.append(x[:, 2:6], x[:, 6:], x[:, :2], cos, sin, kc, vc, tables, lens, starts, "bf16")
    got = run(f, x, cos, sin, kc, vc, tables, lens, starts)
    for name, w, e in zip(("output0", "kc", "vc"), want, tol):
        close(got[name], w, e)


def test_append_cache_still_read():
    """A cache whose old contents are read after the call is updated in a copy
    first."""
    rng = np.random.default_rng(44)
    tables, lens, starts, pages = P.batch(rng, [20, 9], None, 4)
    q, k, v = (draw(rng, (2, h, 8), "f32") for h in (2, 1, 1))
    kc, vc = (draw(rng, (pages, 4, 1, 8), "f32") for _ in range(2))
    cos, sin = np.ones((20, 4), np.float32), np.zeros((20, 4), np.float32)

    def f(q, k, v, cos, sin, kc, vc, tables, lens):
        old = kc * np.float32(2)
        r = T.rotary_append(q, k, v, cos, sin, kc, vc, tables, lens)
        return r, kc + old

    want, _ = P.append(q, k, v, cos, sin, kc, vc, tables, lens, starts, "f32")
    got = run(f, q, k, v, cos, sin, kc, vc, tables, lens)
    assert (got["kc"] == want[1]).all() and (got["vc"] == want[2]).all()
    assert np.allclose(got["output1"], want[1] + 2 * kc.astype(np.float64), rtol=2**-23)


# ---------------------------------------------------------------------------
# Sampling
# ---------------------------------------------------------------------------
def f_sample(x, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    return T.sample(x, u, temperature, top_k, top_p, min_p)


def check_sample(rng, x, t, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """Draws in the middle of kept tokens' shares, away from their borders."""
    x = P.cast(x, t)
    u, want = [], []
    for r in range(len(x)):
        ids, w = P.kept(P.up(x[r:r + 1])[0], temperature, top_k, top_p, min_p)
        c, total = np.cumsum(w), w.sum()
        ok = np.nonzero(w > 2e-5 * total)[0]
        i = int(rng.choice(ok))
        u.append((c[i] - w[i] / 2) / total)
        want.append(ids[i])
    u = np.array(u, np.float32)
    got = run(f_sample, x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)["output0"]
    assert got.dtype == np.int32 and (got == np.array(want)).all(), (got, want)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 257, 5000, 33333])
def test_sample_sizes(t, vocab):
    rng = np.random.default_rng(51)
    x = rng.standard_normal((5, vocab)) * 3
    check_sample(rng, x, t, 0.8)
    check_sample(rng, x, t, 0.8, top_k=7)
    check_sample(rng, x, t, 1.3, top_p=0.777)
    check_sample(rng, x, t, 0.8, top_k=40, top_p=0.83, min_p=0.031)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("top_k,top_p", [(300, None), (None, 0.613), (4321, 0.613), (4999, None)])
def test_sample_ties(t, top_k, top_p):
    """Borders inside runs of equal logits, few and whole rows long."""
    rng = np.random.default_rng(52)
    check_sample(rng, np.round(rng.standard_normal((4, 5000)) * 2), t, 1.0, top_k, top_p)
    check_sample(rng, np.zeros((2, 5000)), t, 1.0, top_k, top_p)
    check_sample(rng, np.repeat([[1.0, 3.0]], 2500, 1).reshape(1, -1), t, 1.0, top_k, top_p)


def test_sample_narrow_and_wide_rows():
    """All values in one bin of the first histogram but no ties, and values
    far apart."""
    rng = np.random.default_rng(53)
    for std in (1e-4, 1e-2, 300.0):
        x = rng.standard_normal((3, 20000)) * std + 5
        check_sample(rng, x, "f32", 1.0, top_k=900)
        check_sample(rng, x, "f32", 1.0, top_p=0.4321)
    check_sample(rng, rng.standard_normal((3, 20000)), "f32", 50.0, top_k=9000, top_p=0.7)
    check_sample(rng, rng.standard_normal((3, 20000)), "f32", 0.01, top_p=0.99)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_sample_masked(t):
    """-inf and the type's lowest value as masks, NaN, infinities, rows with
    nothing to draw."""
    rng = np.random.default_rng(54)
    low = {"bf16": -3.3895314e38, "f16": -65504.0, "f32": np.finfo(np.float32).min}[t]
    x = rng.standard_normal((6, 3000)).astype(np.float32)
    x[:, rng.permutation(3000)[:2900]] = -np.inf
    x[3:, 5] = low
    check_sample(rng, x, t, top_k=30)
    check_sample(rng, x, t, top_p=0.9)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 1:] = np.nan
    x[2, 0] = -1.0
    x[3] = low
    x[4, [9, 40]] = np.inf
    x[5, 100:] = np.nan
    u = np.array([0.3, 0.3, 0.9, 0.5001, 0.7, 0.999], np.float32)
    for kw in ({}, dict(top_k=3000), dict(top_p=1.0), dict(min_p=0.0)):
        got = run(f_sample, P.cast(x, t), u, **kw)["output0"]
        assert list(got[:3]) == [-1, -1, 0] and got[3] == 1500 and got[4] == 40 and (got[5] == -1 or got[5] < 100)
    assert list(run(f_sample, P.cast(x, t), u, temperature=0.0)["output0"][:5]) == [-1, -1, 0, 0, 9]


def test_sample_rows_of_parameters():
    """Filters and temperatures per row, out of range ones among them."""
    rng = np.random.default_rng(55)
    x = (rng.standard_normal((8, 4000)) * 3).astype(np.float32)
    temp = np.array([1, 0, 0.5, np.inf, 1, 2, np.nan, 1e-30], np.float32)
    k = np.array([10, 5, 0, -3, 1, 4001, 7, 9], np.int32)
    p = np.array([0.9, 0.5, 2.0, 1.0, 0.1, 0.0, 0.3, np.nan], np.float32)
    m = np.array([0.1, 0, -1, 0, 0, 7.0, np.nan, np.nan], np.float32)
    u = np.full(8, 0.4, np.float32)
    got = run(f_sample, x, u, temp, k, p, m)["output0"]
    assert (got == f_sample(x, u, temp, k, p, m)).all()
    assert got[1] == got[1] and got[3] == int(0.4 * 4000)


def test_sample_uniform_ends():
    x = np.zeros((6, 1000), np.float32)
    x[:, :3] = -np.inf
    x[:, 900:] = -np.inf
    u = np.array([0.0, 1.0 - 2.0**-24, 1.0, 2.0, -1.0, np.nan], np.float32)
    assert list(run(f_sample, x, u)["output0"]) == [3, 899, 899, 899, 3, 899]


def test_sample_strided_rows():
    """The real part of a padded vocabulary, one position of several."""
    rng = np.random.default_rng(56)
    x = P.cast(rng.standard_normal((5, 3, 1003)) * 3, "bf16")
    u = rng.random(5).astype(np.float32)
    f = lambda x, u: T.sample(x[:, -1, :999], u, top_k=50)  # noqa: E731
    assert (run(f, x, u)["output0"] == T.sample(np.ascontiguousarray(x[:, -1, :999]), u, top_k=50)).all()


def test_sample_large_vocabulary():
    rng = np.random.default_rng(57)
    x = rng.standard_normal((2, 262144)) * 2
    check_sample(rng, x, "bf16", 1.0, 1000, 0.9)
    check_sample(rng, x, "f32", 1.0)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [8193, 40001, 131080])
def test_sample_long_rows(t, vocab):
    """Rows of several segments: few and many kept, past what the segments' lists
    and the row's hold."""
    rng = np.random.default_rng(58)
    x = rng.standard_normal((3 if vocab < 100000 else 1, vocab)) * 3
    for k in (1, 50, 257, 700, 6000, vocab - 1):
        check_sample(rng, x, t, 0.8, top_k=k)
    check_sample(rng, x, t, 0.8, top_k=300, top_p=0.9)
    check_sample(rng, x, t, 0.8, top_k=300, min_p=0.05)
    check_sample(rng, x, t, 0.8, min_p=0.01)
    check_sample(rng, x, t, 0.8, top_k=5000, top_p=0.95, min_p=1e-6)
    for p in (0.0, 0.3, 0.9, 0.999):
        check_sample(rng, x, t, 1.0, top_p=p)
        check_sample(rng, x, t, 6.0, top_p=p)
    check_sample(rng, x, t, 0.05, top_k=200)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("top_k,top_p", [(1, None), (5, 0.5), (300, None), (600, 0.613), (None, 0.613), (9000, 0.9)])
def test_sample_long_ties(t, top_k, top_p):
    """Whole rows of one value, of few, of two; all large values in one segment."""
    rng = np.random.default_rng(59)
    check_sample(rng, np.zeros((2, 20011)), t, 1.0, top_k, top_p)
    check_sample(rng, np.round(rng.standard_normal((3, 20011)) * 2), t, 1.0, top_k, top_p)
    check_sample(rng, np.repeat([[1.0, 9.0]], 10001, 1).reshape(1, -1), t, 1.0, top_k, top_p)
    check_sample(rng, np.linspace(8, -8, 20011).reshape(1, -1), t, 1.0, top_k, top_p)
    check_sample(rng, np.linspace(-8, 8, 20011).reshape(1, -1), t, 0.1, top_k, top_p)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_sample_long_masked(t):
    """A few tokens left of a long row, fewer than top_k; infinities and NaN."""
    rng = np.random.default_rng(60)
    low = {"bf16": -3.3895314e38, "f16": -65504.0, "f32": np.finfo(np.float32).min}[t]
    for mask in (-np.inf, low, np.nan):
        x = np.full((4, 30000), mask, np.float32)
        for r, m in enumerate((1, 10, 60, 3000)):
            x[r, rng.permutation(30000)[:m]] = rng.standard_normal(m) * 2
        for k in (3, 40, 900):
            check_sample(rng, x, t, top_k=k)
            check_sample(rng, x, t, top_k=k, top_p=0.8, min_p=0.01)
        check_sample(rng, x, t, top_p=0.9)
    x = np.full((4, 30000), -np.inf, np.float32)
    x[1] = np.nan
    x[2, [777, 29999]] = np.inf
    x[3] = low
    u = np.array([0.3, 0.3, 0.7, 0.5], np.float32)
    for kw in (dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1)):
        got = run(f_sample, P.cast(x, t), u, **kw)["output0"]
        assert list(got[:3]) == [-1, -1, 29999]
        assert got[3] == {"top_k": 25, "top_p": 13500, "min_p": 15000}[list(kw)[0]]


def test_sample_long_rows_of_parameters():
    rng = np.random.default_rng(62)
    x = (rng.standard_normal((9, 17001)) * 3).astype(np.float32)
    temp = np.array([1, 0, 0.5, np.inf, 1, 2, np.nan, 1e-30, 1], np.float32)
    k = np.array([10, 5, 0, -3, 1, 17002, 7, 9, 500], np.int32)
    p = np.array([0.9, 0.5, 2.0, 1.0, 0.1, 0.0, 0.3, np.nan, 0.99], np.float32)
    m = np.array([0.1, 0, -1, 0, 0, 7.0, np.nan, np.nan, 1e-3], np.float32)
    u = np.full(9, 0.4, np.float32)
    got = run(f_sample, x, u, temp, k, p, m)["output0"]
    assert (got == f_sample(x, u, temp, k, p, m)).all()
    assert got[3] == int(0.4 * 17001)


def test_sample_long_strided_rows():
    """Odd rows that start off any alignment, drawn again and again from one load."""
    rng = np.random.default_rng(63)
    x = P.cast(rng.standard_normal((5, 2, 20003)) * 3, "bf16")
    u = rng.random(5).astype(np.float32)
    f = lambda x, u: T.sample(x[:, -1, 1:20000], u, top_k=50, top_p=0.9)  # noqa: E731
    dk, ins, outs = load(f, x, u)
    want = T.sample(np.ascontiguousarray(x[:, -1, 1:20000]), u, top_k=50, top_p=0.9)
    for graph in (False, True, False, True):
        for _ in range(3):
            dk(ins, outs, sync=False, graph=graph)
        dk(ins, outs, sync=True, graph=graph)
        assert (outs["output0"].numpy() == want).all()


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
def _step(heads, kv):
    def step(qkv, cos, sin, kc, vc, tables, lens, starts, head, u):
        x = qkv.reshape(qkv.shape[0], heads + 2 * kv, -1)
        q = T.rotary_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], cos, sin, kc, vc, tables, lens, starts)
        o = T.paged_attention(q, kc, vc, tables, lens, starts, window=48, sinks=3)
        logits = o.reshape(o.shape[0], -1) @ head
        return o, logits, T.sample(logits, u, temperature=0.9, top_k=20, top_p=0.95), q

    return step


def test_calls_queued_by_turns():
    """Kernels with workspaces of their own, queued by turns without a wait, eager and
    replayed."""
    rng = np.random.default_rng(64)
    tables, lens, _, pages = P.batch(rng, [5000, 40], None, 16)
    kc, vc = draw(rng, (pages, 16, 2, 64), "bf16"), draw(rng, (pages, 16, 2, 64), "bf16")
    x = P.cast(rng.standard_normal((2, 30000)) * 3, "f32")
    work = []
    for i in range(3):
        q, u = draw(rng, (2, 4, 64), "bf16"), rng.random(2).astype(np.float32)
        f = lambda q, kc, vc, tables, lens: T.paged_attention(q, kc, vc, tables, lens)  # noqa: E731
        work.append((load(f, q, kc, vc, tables, lens), None if i else P.paged(q, kc, vc, tables, lens, None, 0, 0, "bf16")))
        f = lambda x, u: T.sample(x, u, 0.9, 100, 0.9)  # noqa: E731
        work.append((load(f, x, u), T.sample(x, u, 0.9, 100, 0.9)))
    alone = []
    for (dk, ins, outs), _ in work:
        dk(ins, outs)
        alone.append(outs["output0"].numpy())
    for graph in (False, True, True):
        for turn in range(4):
            for (dk, ins, outs), _ in work:
                dk(ins, outs, sync=False, graph=graph)
        for (dk, ins, outs), _ in work:
            dk(ins, outs, sync=True, graph=graph)
        for (call, want), first in zip(work, alone):
            got = call[2]["output0"].numpy()
            assert (got == first).all()
            if isinstance(want, tuple):
                close(got, *want)
            elif want is not None:
                assert (got == want).all()


def test_serving_step_together():
    """A prompt step, then steps of one token, each replayed as a graph and
    queued without a wait between."""
    rng = np.random.default_rng(61)
    t, heads, kv, d, page = "bf16", 8, 2, 64, 16
    lens, new = [70, 5, 33], [70, 5, 33]
    tables, _, _, pages = P.batch(rng, [90, 30, 60], new, page)
    ang = np.outer(np.arange(100), 0.5 ** np.arange(d // 2)).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    head = draw(rng, (heads * d, 512), t, 0.2)
    kc, vc = np.zeros((pages, page, kv, d), dt.bfloat16), np.zeros((pages, page, kv, d), dt.bfloat16)
    kd, vd = DeviceTensor.from_numpy(kc, name="kc"), DeviceTensor.from_numpy(vc, name="vc")
    for step in range(5):
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if step == 0 else np.arange(4, dtype=np.int32)
        n = int(starts[-1])
        ln = np.array(lens, np.int32) + step
        qkv, u = draw(rng, (n, (heads + 2 * kv) * d), t), rng.random(n).astype(np.float32)
        dk, ins, outs = load(_step(heads, kv), qkv, cos, sin, kd, vd, tables, ln, starts, head, u)
        for graph in (False, True, True):
            dk(ins, outs, sync=graph, graph=graph)
        got = {k: v.numpy() for k, v in outs.items()}
        x = qkv.reshape(n, heads + 2 * kv, d)
        want, tol = P.append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], cos, sin, kc, vc, tables, ln, starts, t)
        close(got["kc"], want[1], tol[1])
        close(got["vc"], want[2], tol[2])
        kc, vc = got["kc"], got["vc"]
        close(got["output3"], want[0], tol[0])
        close(got["output0"], *P.paged(got["output3"], kc, vc, tables, ln, starts, 48, 3, t))
        assert (got["output2"] == T.sample(got["output1"], u, temperature=0.9, top_k=20, top_p=0.95)).all()
