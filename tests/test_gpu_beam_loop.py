"""A beam search over an 8-bit paged cache on the GPU, all five operators in one
kernel, against the same search on the CPU."""

import numpy as np
import pytest

from nkipy_amd.kernels import qwen3
from nkipy_amd.kernels.rmsnorm import rmsnorm_kernel

import beam_loop as L
import beams_plain as B
import fp8_plain as Q
import layer_plain
import serving_plain as P
from test_gpu_beams import select_tolerance
from test_gpu_serving import load, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("graph", [False, True])
def test_search(t, graph):
    """Step by step over the same device arrays: tables, tokens and parents are
    the CPU's; the cache its values but for neighbouring codes; attention is that
    over the cache as it stands on the GPU before the beams change places."""
    rng = np.random.default_rng(21)
    state = L.begin(rng)
    cpu = {n: state[n].copy() for n in L.ARRAYS}
    scores = np.full((L.GROUPS, L.BEAMS), -np.inf, np.float32)
    scores[:, 0] = 0
    ended = np.zeros((L.GROUPS, L.BEAMS), np.int32)
    dk = None
    for i in range(20):
        x = L.token(rng, i, t, scores, ended)
        if dk is None:
            dk, ins, outs = load(L.step, **state, **x)
            assert dk.plan.kernel_kinds == ["assign_pages", "rotary_append_fp8", "attend8", "beam_select", "beam_reorder"]
        for n, a in x.items():
            ins[n].write_from_numpy(a)
        dk(ins, outs, graph=graph)
        got = {n: y.numpy() for n, y in outs.items()}
        want = L.step(cos=state["cos"], sin=state["sin"], **cpu, **x)
        assert (got["tables"] == cpu["tables"]).all()
        for n, y in (("output1", want[1]), ("output2", want[2]), ("output3", want[3]), ("output4", want[4]), ("output6", want[6])):
            assert (got[n] == y).all(), n
        near = np.abs(got["output5"] - want[5]) <= select_tolerance(x["logits"], L.VOCAB) + 2.0**-24 * np.abs(want[5])
        assert (near | (got["output5"] == want[5])).all()
        for c, e in (("kc", "ke"), ("vc", "ve")):
            assert (got[e] == cpu[e]).all()
            u, w = Q.values(got[c], got[e]), Q.values(cpu[c], cpu[e])
            # neighbouring codes are a step apart, 2^-3 of the larger or 2^-9 of the scale
            tol = np.maximum(np.maximum(np.abs(u), np.abs(w)) * 2.0**-3, 2.0 ** (cpu[e][:, None, :, None] - 9.0))
            assert (np.abs(u - w) <= tol).all()
            assert (u != w).mean() < 1e-3
        scores, ended = got["output5"], got["output6"]


def test_layer_over_codes(gpu):
    """The layer's own kernel: its attention is that of the codes it wrote."""
    rng = np.random.default_rng(22)
    for t, dim, new in (("f32", 48, [20, 3, 9]), ("bf16", 64, None), ("bf16", 128, [20, 3, 9])):
        c = layer_plain.case(rng, t, [33, 71, 10], new, 96, 6, 2, dim, 16)
        ke, ve = (rng.integers(-9, -4, (c["kc"].shape[0], 2)).astype(np.int32) for _ in range(2))
        kc, vc = Q.random_cache(rng, *c["kc"].shape)[0], Q.random_cache(rng, *c["kc"].shape)[0]
        n = len(c["x"])

        def layer(x, w, qn, kn, kc, vc, ke, ve, tables, lens, wo, starts=None):
            out = qwen3.qwen3_paged_attention_kernel(x, w, qn, kn, 1e-6, 6, dim, 2, kc, vc, tables, lens, starts, wo, key_exps=ke,
                                                     value_exps=ve)
            q = rmsnorm_kernel((x @ w)[:, :6 * dim].reshape(n, 6, dim), qn, 1e-6)
            return out, q

        rest = {} if new is None else dict(starts=c["starts"])
        got = run(layer, c["x"], c["w"], c["qn"], c["kn"], kc, vc, ke, ve, c["tables"], c["lens"], c["wo"], **rest)
        cos, sin = qwen3.compute_cos_sin_cache(dim, c["tables"].shape[1] * 16, base=1000000)
        zeros = P.cast(np.zeros((n, 2, dim)), t)
        (rq, tq), _ = Q.append(got["output1"], zeros, zeros, cos, sin, kc, vc, ke, ve, c["tables"], c["lens"], c["starts"], t)
        q = P.cast(rq, t)  # (the layer's own is a rounding away)
        o, tol = Q.paged(q, got["kc"], got["vc"], got["ke"], got["ve"], c["tables"], c["lens"], c["starts"], 0, 0, t)
        # a query off by e moves its scores by up to e sum |k| / sqrt(dim), twice over
        # (its own and the largest), and its values' mean by that share of the largest
        h = P.HALF_STEP[t]
        share = np.zeros(n)
        for b, lo, m, length in P.sequences(c["tables"], c["lens"], c["starts"], n):
            keys = np.arange(length)
            pg = c["tables"][b][keys // 16]
            k = np.abs(Q.values(got["kc"][pg, keys % 16], got["ke"][pg])).max()
            v = np.abs(Q.values(got["vc"][pg, keys % 16], got["ve"][pg])).max()
            for i in range(lo, lo + m):
                e = (2 * h * np.abs(rq[i]) + tq[i]).sum(-1).max() * k / np.sqrt(dim)
                share[i] = np.expm1(2 * e) * v
        tol = tol + share[:, None, None]
        wo = P.up(c["wo"])
        want = o.reshape(n, -1) @ wo
        bound = (tol + h * np.abs(o)).reshape(n, -1) @ np.abs(wo) + 2.0**-24 * (len(wo) + 2) * (np.abs(o).reshape(n, -1) @ np.abs(wo))
        bound += h * (np.abs(want) + bound)
        assert (np.abs(P.up(got["output0"]) - want) <= bound).all()


def test_beam_step():
    rng = np.random.default_rng(23)
    for vocab in (1000, 20000):
        h, w, lm = rng.standard_normal((6, 2, 128)), rng.uniform(0.5, 1.5, 128), rng.standard_normal((128, vocab)) * 0.3
        h, w, lm = (P.cast(a, "bf16") for a in (h, w, lm))
        scores, ended = -rng.random((2, 3)).astype(np.float32), np.array([[0, 1, 0], [0, 0, 0]], np.int32)

        def f(h, w, lm, scores, ended):
            return qwen3.beam_step(h, w, lm, 1e-6, scores, ended, 3) + (rmsnorm_kernel(h, w, 1e-6)[:, -1, :] @ lm,)

        got = run(f, h, w, lm, scores, ended)
        B.check_select([got[f"output{i}"] for i in range(4)], got["output4"], scores, ended, 3, select_tolerance(h, vocab))
