"""The paged attention layer with the rotary tables as its arguments."""

import numpy as np
import pytest

from nkipy_amd.core.trace import NKIPyKernel
from nkipy_amd.dispatch.lower import lower
from nkipy_amd.kernels import qwen3 as Q

import layer_plain as L


@pytest.mark.parametrize("new", [None, [5, 0, 11]])
def test_paged_layer_with_tables_given(new):
    """The cos / sin tables as arguments: the same result, and no table among the
    kernel's constants."""
    rng = np.random.default_rng(8)
    c = L.case(rng, "f32", [9, 3, 11], new, 24, 4, 2, 8, 4)
    if new:
        c["lens"] = np.array([9, 0, 11], np.int32)
    cos, sin = Q.compute_cos_sin_cache(8, 50, base=1000000)

    def layer(x, w, qn, kn, kc, vc, tables, lens, starts, wo, cos=None, sin=None):
        return Q.qwen3_paged_attention_kernel(x, w, qn, kn, 1e-6, 4, 8, 2, kc, vc, tables, lens, starts, wo, cos=cos, sin=sin)

    got = []
    for tables in ({}, dict(cos=cos, sin=sin)):
        a = {k: None if x is None else x.copy() for k, x in c.items()}
        got.append([layer(**a, **tables), a["kc"], a["vc"]])
    assert all((x == y).all() for x, y in zip(*got))
    sizes = []
    for tables in ({}, dict(cos=cos, sin=sin)):
        p = lower(NKIPyKernel.trace(layer).specialize(**c, **tables))
        sizes.append(sum(b.nbytes for b in p.buffers if b.kind == "const"))
    assert sizes[0] - sizes[1] == 2 * 4 * 4 * c["tables"].shape[1] * 4
    for one in (dict(cos=cos), dict(sin=sin)):
        with pytest.raises(ValueError, match="both"):
            layer(**c, **one)
