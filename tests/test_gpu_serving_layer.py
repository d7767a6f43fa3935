"""The paged attention layer and the drawn token on the GPU."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core import tensor_apis as T
from nkipy_amd.kernels import qwen3 as Q
from nkipy_amd.kernels.rmsnorm import rmsnorm_kernel
from nkipy_amd.runtime import DeviceKernel, DeviceTensor

import layer_plain as L
import serving_plain as P

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}


@pytest.mark.parametrize("t,dim", [("f32", 48), ("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("lens,new", [([33, 70, 9], [20, 3, 9]), ([33, 71, 10], None)])
def test_paged_layer(gpu, t, dim, lens, new):
    """A step over caches with random beginnings, eager and replayed: the same
    tokens at the same places give the same result each time."""
    rng = np.random.default_rng(8)
    hq, hkv, page = 6, 2, 16
    c = L.case(rng, t, lens, new, 96, hq, hkv, dim, page, 1.0 if t == "f32" else 2.0**-6)

    def layer(x, w, qn, kn, kc, vc, tables, lens, starts, wo):
        return Q.qwen3_paged_attention_kernel(x, w, qn, kn, 1e-6, hq, dim, hkv, kc, vc, tables, lens, starts, wo,
                                              window=40, sinks=2)

    def one_each(x, w, qn, kn, kc, vc, tables, lens, wo):
        return layer(x, w, qn, kn, kc, vc, tables, lens, None, wo)

    args = {k: x for k, x in c.items() if x is not None}
    f = layer if new else one_each
    dk = DeviceKernel.compile_and_load(f, **args, use_cached_if_exists=False)
    assert {"rotary_append", "attend"} <= set(dk.plan.kernel_kinds)
    dev = {k: DeviceTensor.from_numpy(x, name=k) for k, x in args.items()}
    ins = {k: dev[k.split(".must_alias_input")[0]] for k in dk.input_tensors_info}
    outs = {k: dev[k] if k in dev else DeviceTensor.empty(tuple(m.shape), m.dtype, name=k)
            for k, m in dk.output_tensors_info.items()}
    cos, sin = Q.compute_cos_sin_cache(dim, c["tables"].shape[1] * page, base=1000000)
    want, tol = L.layer(c["x"], c["w"], c["qn"], c["kn"], 1e-6, hq, hkv, dim, cos, sin, c["kc"], c["vc"], c["tables"], c["lens"],
                        c["starts"], c["wo"], 40, 2, HALF[t])
    first = None
    for graph in (False, True, False, True):
        dk(ins, outs, graph=graph)
        got = [P.up(outs[k].numpy()) for k in ("output0", "kc", "vc")]
        for g, x, e in zip(got, want, tol):
            assert (np.abs(g - x) <= e).all()
        first = first or got
        assert all((a == b).all() for a, b in zip(got, first))


def test_sampling(gpu):
    """Tokens drawn in the layer's kernel are those of its own logits."""
    rng = np.random.default_rng(9)
    for vocab in (1000, 20000):
        h, w, lm = rng.standard_normal((5, 2, 128)), rng.uniform(0.5, 1.5, 128), rng.standard_normal((128, vocab)) * 0.3
        h, w, lm = (dt.to_bf16(a.astype(np.float32)) for a in (h, w, lm))
        u = rng.random(5).astype(np.float32)

        def draws(h, w, lm, u):
            return (Q.sampling(h, w, lm, 1e-6, u, 0.8, 40, 0.9), Q.sampling(h, w, lm, 1e-6, u, 0.0),
                    rmsnorm_kernel(h, w, 1e-6)[:, -1, :] @ lm)

        dk = DeviceKernel.compile_and_load(draws, h, w, lm, u, use_cached_if_exists=False)
        dev = dict(h=h, w=w, lm=lm, u=u)
        ins = {k: DeviceTensor.from_numpy(dev[k], name=k) for k in dk.input_tensors_info}
        outs = {k: DeviceTensor.empty(tuple(m.shape), m.dtype, name=k) for k, m in dk.output_tensors_info.items()}
        dk(ins, outs)
        token, best, logits = (outs[f"output{i}"].numpy() for i in range(3))
        assert (token == T.sample(logits, u, 0.8, 40, 0.9)).all()
        assert (best == P.up(logits).argmax(1)).all()
