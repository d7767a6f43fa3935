"""Appends into the same caches one after the other on the GPU."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T

import serving_plain as P
from test_gpu_serving import close, draw, load

pytestmark = pytest.mark.gpu


def test_appends_in_turn_with_attention_between():
    """Prompts, then a token each behind them, in one kernel: each attention sees the
    caches as they stand then; eager and replayed."""
    rng = np.random.default_rng(95)
    t, heads, kv, d, page = "bf16", 4, 2, 64, 16
    new = [40, 3, 130]
    tables, lens, starts, pages = P.batch(rng, [61, 9, 140], new, page)
    lens, later = lens - 1, lens
    n = sum(new)
    x, y = draw(rng, (n, heads + 2 * kv, d), t), draw(rng, (3, heads + 2 * kv, d), t)
    ang = np.outer(np.arange(150), 0.5 ** np.arange(d // 2)).astype(np.float32)
    cos, sin = np.cos(ang), np.sin(ang)
    kc, vc = draw(rng, (pages, page, kv, d), t), draw(rng, (pages, page, kv, d), t)

    def step(x, y, cos, sin, kc, vc, tables, lens, later, starts):
        q = T.rotary_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], cos, sin, kc, vc, tables, lens, starts)
        a = T.paged_attention(q, kc, vc, tables, lens, starts)
        old = kc[:2] * np.float32(1)
        r = T.rotary_append(y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], cos, sin, kc, vc, tables, later)
        return a, T.paged_attention(r, kc, vc, tables, later), q, r, old

    dk, ins, outs = load(step, x, y, cos, sin, kc, vc, tables, lens, later, starts)
    assert dk.plan.kernel_kinds.count("rotary_append") == 2
    one, tol1 = P.append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], cos, sin, kc, vc, tables, lens, starts, t)
    for graph in (False, True, False, True):
        dk(ins, outs, sync=True, graph=graph)
        got = {k: v.numpy() for k, v in outs.items()}
        two, tol2 = P.append(y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], cos, sin, got["kc"], got["vc"], tables, later,
                             None, t)
        close(got["output2"], one[0], tol1[0])
        close(got["output3"], two[0], tol2[0])
        rows = tables[np.arange(3), (later - 1) // page], (later - 1) % page  # (of the second call)
        mid = np.ones(kc.shape[:2], bool)
        mid[rows] = False
        for name, i in (("kc", 1), ("vc", 2)):
            close(got[name][mid], one[i][mid], tol1[i][mid])
            close(got[name][rows], two[i][rows], tol2[i][rows])
        close(got["output0"], *P.paged(got["output2"], got["kc"], got["vc"], tables, lens, starts, 0, 0, t))
        close(got["output1"], *P.paged(got["output3"], got["kc"], got["vc"], tables, later, None, 0, 0, t))
        close(got["output4"][mid[:2]], one[1][:2][mid[:2]], tol1[1][:2][mid[:2]])
