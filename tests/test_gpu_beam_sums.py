"""The sums under the chosen continuations' scores, on the GPU: large logits and
logits close to each other."""

import numpy as np
import pytest

import beams_plain as B
import serving_plain as P
from test_gpu_beams import f_select
from test_gpu_serving import run

pytestmark = pytest.mark.gpu

# exact in bf16 up to 2^40; the first two times log2(e), rounded to 32 bits, are off by
# 124 and 126, their negatives by -124 and -126
LARGE = [1509949440.0, 3439329280.0, -1509949440.0, -3439329280.0, 2.0**40, -(2.0**40), 1e30, -1e30, 2.0**126, 3e38, -3e38]


def select(x, scores, ended, end):
    got = run(f_select, x, scores, ended, end_token=end)
    return [got[f"output{j}"] for j in range(4)]


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 20, 9000, 20000])
def test_equal_large_logits(t, vocab):
    """Each continuation has its share of 1: score - log(vocab), which is the sum
    of that many ones, exact in 32 bits, and a rounding of the score."""
    value = P.up(P.cast(np.array(LARGE), t))
    k = 3
    x = P.cast(np.repeat(value, k)[:, None] * np.ones((1, vocab)), t)
    scores = np.tile(np.array([-1, -50, -100], np.float32), (len(LARGE), 1))
    tokens, parents, new, _ = select(x, scores, np.zeros_like(scores, dtype=np.int32), -1)
    for j in range(k):
        b, i = (0, j) if vocab >= k else (j, 0)
        assert (parents[:, j] == b).all() and (tokens[:, j] == i).all()
        want = scores[0, b] - np.log(vocab)
        assert np.abs(new[:, j] - want).max() <= 2.0**-23 * np.abs(want), (j, new[:, j], want)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_one_large_logit(t):
    """One far ahead has all the weight, whatever lies below."""
    x = np.random.default_rng(92).standard_normal((len(LARGE), 9000))
    x[:, 4321] = 0
    x = P.cast(np.abs(np.array(LARGE))[:, None] * np.where(np.arange(9000) == 4321, 1.0, 2.0**-2) * (1 - 0.1 * np.abs(x)), t)
    scores = np.full((len(LARGE), 1), -2, np.float32)
    tokens, _, new, _ = select(x, scores, np.zeros_like(scores, dtype=np.int32), -1)
    assert (tokens == 4321).all() and (new == -2).all()


@pytest.mark.parametrize("t", ["f16", "f32"])
@pytest.mark.parametrize("g,k,vocab", [(2, 4, 1000), (1, 3, 8000), (2, 2, 50257)])
@pytest.mark.parametrize("mean", [0, 700, 1500, 3000, -3000])
def test_logits_close_to_each_other(t, g, k, vocab, mean):
    """Terms 2^t, t = (x - m) log2(e) of -11.6 to 0 for logits within 8 of the
    largest: in steps of 2^-24 of the sum, t's rounding 8 and the constant's 1, the
    power's ulp 2, additions of 32 and of 64 lanes 37, what m log2(e) was rounded
    by (a power, its argument and a product) 4, and a factor of a power and its
    argument with three additions for the waves' sums and for the segments' 2 x
    16: up to 84; then the score's own rounding."""
    rng = np.random.default_rng(abs(vocab + mean))
    x = P.cast(mean - 8 * rng.random((g * k, vocab)), t)
    scores = -3 * rng.random((g, k)).astype(np.float32)
    ended = np.zeros((g, k), np.int32)
    B.check_select(select(x, scores, ended, 0), x, scores, ended, 0, 84 * 2.0**-24)
