"""A beam search over an 8-bit paged cache on the CPU: every beam attends to the
tokens of its own past."""

import numpy as np

from nkipy_amd.core import tensor_apis as T
from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch.lower import lower
from nkipy_amd.kernels import qwen3

import beam_loop as L
import fp8_plain as Q
import layer_plain
import serving_plain as P


def test_beams_attend_to_their_own_past():
    """The caches of a search with shared and copied pages hold, for each beam,
    the values of the tokens that its parents appended."""
    rng = np.random.default_rng(11)
    state = L.begin(rng)
    scores = np.full((L.GROUPS, L.BEAMS), -np.inf, np.float32)
    scores[:, 0] = 0
    ended = np.zeros((L.GROUPS, L.BEAMS), np.int32)
    past = [[] for _ in range(L.ROWS)]  # the values appended for each row
    for i in range(21):
        x = L.token(rng, i, "f32", scores, ended)
        arrays = {n: state[n] for n in L.ARRAYS}
        out, slots, free, _, parents, scores, ended = L.step(cos=state["cos"], sin=state["sin"], **arrays, **x)
        past = [p + [P.up(x["v"][r])] for r, p in enumerate(past)]
        assert len(set(slots.tolist())) == L.ROWS and (slots >= 0).all()
        assert free[0] >= 0
        past = [past[g * L.BEAMS + parents[g, b]] for g in range(L.GROUPS) for b in range(L.BEAMS)]
        keys = np.arange(i + 1)
        for r in range(L.ROWS):
            pg = state["tables"][r][keys // L.PAGE]
            v = Q.values(state["vc"][pg, keys % L.PAGE], state["ve"][pg])
            # half a step of a code, and half a step of the least ones (2^-10 of the
            # scale) for each time that the scale grew under it: at most once a row
            tol = 2.0**-4 * np.abs(past[r]) + 2.0 ** (state["ve"][pg][..., None] - 10.0) * L.PAGE
            assert (np.abs(v - past[r]) <= tol).all()
    # rows of one group share their full pages, and no page of two groups
    owner = {}
    for r in range(L.ROWS):
        for pg in state["tables"][r][:2]:
            assert owner.setdefault(int(pg), r // L.BEAMS) == r // L.BEAMS
    assert len(owner) < 2 * L.ROWS


def test_step_lowers_without_copies():
    rng = np.random.default_rng(12)
    x = L.token(rng, 0, "bf16", np.zeros((L.GROUPS, L.BEAMS), np.float32), np.zeros((L.GROUPS, L.BEAMS), np.int32))
    plan = lower(NKIPyKernel.trace(L.step).specialize(**L.begin(rng), **x))
    assert plan.kernel_kinds == ["assign_pages", "rotary_append_fp8", "attend8", "beam_select", "beam_reorder"]
    assert set(plan.alias_outputs) == set(L.ARRAYS)


def test_layer_over_codes():
    """The paged attention layer with 8-bit caches: its bounds, and those of the
    codes of what it appends."""
    rng = np.random.default_rng(13)
    c = layer_plain.case(rng, "f32", [9, 3, 11], [5, 3, 11], 24, 4, 2, 8, 4)
    ke, ve = (np.zeros((c["kc"].shape[0], 2), np.int32) for _ in range(2))
    kc, vc = (np.zeros(c["kc"].shape, Q.random_cache(rng, 1, 1, 1, 1)[0].dtype) for _ in range(2))
    args = (c["x"], c["w"], c["qn"], c["kn"], 1e-6, 4, 8, 2)
    where = (c["tables"], c["lens"], c["starts"], c["wo"])
    got = qwen3.qwen3_paged_attention_kernel(*args, kc, vc, *where, key_exps=ke, value_exps=ve)
    # the same layer in pieces, from the operators
    cos, sin = qwen3.compute_cos_sin_cache(8, c["tables"].shape[1] * 4, base=1000000)
    xq, xk, xv = np.split(c["x"] @ c["w"], [32, 48], axis=1)
    xq = qwen3.rmsnorm_kernel(xq.reshape(19, 4, 8), c["qn"], 1e-6)
    xk = qwen3.rmsnorm_kernel(xk.reshape(19, 2, 8), c["kn"], 1e-6)
    kd, vd, kf, vf = np.zeros_like(kc), np.zeros_like(vc), np.zeros_like(ke), np.zeros_like(ve)
    q = T.rotary_append_fp8(xq, xk, xv.reshape(19, 2, 8), cos, sin, kd, vd, kf, vf, *where[:3])
    out = T.paged_attention_fp8(q, kd, vd, kf, vf, *where[:3])
    assert (got == out.reshape(19, 32) @ c["wo"]).all()
    assert (kc.tobytes(), vc.tobytes()) == (kd.tobytes(), vd.tobytes()) and (ke == kf).all() and (ve == vf).all()


def test_beam_step_is_select_of_the_logits():
    rng = np.random.default_rng(14)
    h, w, lm = rng.standard_normal((6, 2, 16)), rng.uniform(0.5, 1.5, 16), rng.standard_normal((16, 50))
    h, w, lm = (a.astype(np.float32) for a in (h, w, lm))
    scores, ended = -rng.random((2, 3)).astype(np.float32), np.array([[0, 1, 0], [0, 0, 0]], np.int32)
    got = qwen3.beam_step(h, w, lm, 1e-6, scores, ended, 3)
    want = T.beam_select(qwen3.rmsnorm_kernel(h, w, 1e-6)[:, -1, :] @ lm, scores, ended, end_token=3)
    assert all((a == b).all() for a, b in zip(got, want))
