"""The paged attention layer and the drawn token on the CPU."""

import numpy as np
import pytest

from nkipy_amd.core import tensor_apis as T
from nkipy_amd.kernels import qwen3 as Q

import layer_plain as L

HALF = 2.0**-24


@pytest.mark.parametrize("new", [None, [5, 0, 11]])
@pytest.mark.parametrize("window,sinks", [(None, 0), (4, 1)])
def test_paged_layer(new, window, sinks):
    rng = np.random.default_rng(5)
    c = L.case(rng, "f32", [9, 3, 11], new, 24, 4, 2, 8, 4)
    if new:
        c["lens"] = np.array([9, 0, 11], np.int32)
    cos, sin = Q.compute_cos_sin_cache(8, c["tables"].shape[1] * 4, base=1000000)
    want, tol = L.layer(c["x"], c["w"], c["qn"], c["kn"], 1e-6, 4, 2, 8, cos, sin, c["kc"], c["vc"], c["tables"], c["lens"],
                        c["starts"], c["wo"], window, sinks, HALF)
    got = Q.qwen3_paged_attention_kernel(c["x"], c["w"], c["qn"], c["kn"], 1e-6, 4, 8, 2, c["kc"], c["vc"], c["tables"],
                                         c["lens"], c["starts"], c["wo"], window=window, sinks=sinks)
    for g, x, e in zip((got, c["kc"], c["vc"]), want, tol):
        assert (np.abs(g - x) <= e).all()


def test_paged_layer_agrees_with_the_dense_cache():
    """One prompt and the token behind it, over pages out of order and over one
    dense cache: both within the layer's bounds, so twice those apart."""
    rng = np.random.default_rng(6)
    c = L.case(rng, "f32", [12], [12], 24, 4, 2, 8, 5)
    weights = c["w"], c["qn"], c["kn"], 1e-6
    cos, sin = Q.compute_cos_sin_cache(8, c["tables"].shape[1] * 5, base=1000000)
    dense_k, dense_v = (np.zeros((1, c["tables"].shape[1] * 5, 2, 8), np.float32) for _ in range(2))
    for length, new in ((11, 11), (12, 1)):
        x = rng.standard_normal((new, 24)).astype(np.float32)
        lens, starts = np.array([length], np.int32), np.array([0, new], np.int32)
        _, tol = L.layer(x, *weights, 4, 2, 8, cos, sin, c["kc"], c["vc"], c["tables"], lens, starts, c["wo"], None, 0, HALF)
        got = Q.qwen3_paged_attention_kernel(x, *weights, 4, 8, 2, c["kc"], c["vc"], c["tables"], lens, starts, c["wo"])
        want = Q.qwen3_attention_kernel(x[None], *weights, 4, 8, 2, dense_k, dense_v,
                                        None if new > 1 else np.array([11], np.int32), c["wo"])
        assert (np.abs(got - want[0]) <= 2 * tol[0]).all()


def test_sampling_without_randomness_is_greedy():
    rng = np.random.default_rng(7)
    h, w, lm = rng.standard_normal((3, 2, 16)), rng.uniform(0.5, 1.5, 16), rng.standard_normal((16, 50))
    h, w, lm = (a.astype(np.float32) for a in (h, w, lm))
    u = np.array([0.2, 0.5, 0.99], np.float32)
    greedy = Q.greedy_sampling(h, w, lm, 1e-6).reshape(-1)
    assert (Q.sampling(h, w, lm, 1e-6, u, temperature=0.0) == greedy).all()
    assert (Q.sampling(h, w, lm, 1e-6, u, top_k=1) == greedy).all()
    assert (Q.sampling(h, w, lm, 1e-6, u, top_p=0.0) == greedy).all()
    x = h[:, -1].astype(np.float64)
    logits = (x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w) @ lm
    assert (Q.sampling(h, w, lm, 1e-6, u, 0.7, 20, 0.9) == T.sample(logits.astype(np.float32), u, 0.7, 20, 0.9)).all()
