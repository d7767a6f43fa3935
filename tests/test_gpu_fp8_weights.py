"""The weights of the attention over 8-bit codes: what their rounding may cost."""

import numpy as np
import pytest

from nkipy_amd.core import dtypes as dt

import fp8_plain as Q
import serving_plain as P
from test_gpu_fp8_cache import f_attend
from test_gpu_serving import close, draw, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("lens,new", [([1, 31, 65, 400], None), ([70, 130, 400], [70, 1, 140]), ([3000], None), ([3000, 40], [200, 3])])
def test_equal_values_come_back(t, d, lens, new):
    """A weighted mean of equal values is that value.

    Key 0 of every 32 has score 0, the others -y with e^-y = 0.5018, which as a
    bf16 weight is 0.5 (a step there is 2^-8): (1 + 31 * 0.5) / (1 + 31 * 0.5018)
    = 0.9966.  Where weights keep 2^-16 of themselves, that and the 32-bit
    roundings of up to 3000 keys (2^-24 each) are below 2^-12, half a step of fp16
    below 1 and far below one of bf16, so the result is 1.  fp32: as many steps
    of 2^-24 as there are keys.  Packed queries of bf16 on matrix instructions
    have weights rounded to bf16: 2^-8 and a step of the result's."""
    rng = np.random.default_rng(71)
    tables, lens, starts, pages = P.batch(rng, lens, new, 16)
    n = int(starts[-1]) if new else len(lens)
    q = np.zeros((n, 4, d), np.float32)
    q[:, :, 0] = 1
    kb, vb = np.zeros((pages, 16, 2, d), np.uint8), np.full((pages, 16, 2, d), 0x38, np.uint8)  # 0 and 1.0
    for row in tables:
        for i, pg in enumerate(row):
            if pg >= 0:
                kb[pg, :, :, 0] = 0xB8  # -1.0
                if i % 2 == 0:
                    kb[pg, 0, :, 0] = 0
    zero = np.zeros((pages, 2), np.int32)
    assert (Q.TABLE[[0x38, 0xB8]] == [1, -1]).all()
    got = P.up(run(f_attend, P.cast(q, t), kb.view(dt.float8_e4m3fn), vb.view(dt.float8_e4m3fn), zero, zero, tables, lens, starts,
                   scale=float(-np.log(0.5018)))["output0"])
    if t == "bf16" and new and d != 80:
        assert np.abs(got - 1).max() <= 2.0**-8 + 2.0**-8
    elif t == "f32":
        assert np.abs(got - 1).max() <= max(lens) * 2.0**-24
    else:
        assert (got == 1).all(), (got.min(), got.max())


def near(q, kc, vc, ke, ve, tables, lens, starts, t, weight):
    """(result, tolerance) where a weight keeps ``weight`` of itself: of the plain
    form's tolerance, the share of the weights' own rounding replaced."""
    out, tol = Q.paged(q, kc, vc, ke, ve, tables, lens, starts, 0, 0, t)
    vb = np.ascontiguousarray(vc).view(np.uint8) & 0x7F  # the mean |v| is the result over |v|
    mag, _ = Q.paged(q, kc, vb.view(vc.dtype), ke, ve, tables, lens, starts, 0, 0, t)
    return out, tol - mag * P.HALF_STEP[t] + mag * weight


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (5, 1, 64), (40, 2, 128)])
def test_weights_of_single_tokens(t, hq, hkv, d):
    """Kept to 2^-16 of themselves: results within a rounding of their own and
    that."""
    rng = np.random.default_rng(72)
    tables, lens, _, pages = P.batch(rng, [1, 40, 129, 700, 3000], None, 16)
    q = draw(rng, (5, hq, d), t)
    (kc, ke), (vc, ve) = Q.random_cache(rng, pages, 16, hkv, d), Q.random_cache(rng, pages, 16, hkv, d)
    got = run(f_attend, q, kc, vc, ke, ve, tables, lens)["output0"]
    close(got, *near(q, kc, vc, ke, ve, tables, lens, None, t, 2.0**-16))
