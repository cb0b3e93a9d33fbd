"""xpu_sample on gfx950 where its launches meet: bins whose weight rounds to
nothing, temperatures at which neighbouring floats are further apart than the
histogram is long."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import Buffers
from test_gpu_sample import Rows

pytestmark = pytest.mark.gpu
NEAR_ONE = np.float32(1 - 2.0 ** -24)


def call(rt, r):
    """The tokens and probabilities of Rows r."""
    with Buffers(rt) as b:
        s, ptr, workspace, size = r.device(b)
        tokens, probability = b.alloc(4 * r.rows), b.alloc(4 * r.rows)
        rt.sample(s, ptr, tokens, workspace, size, probability)
        rt.synchronize()
        return rt.download(tokens, r.rows, np.uint32), rt.download(probability, r.rows, np.float32)


@pytest.mark.parametrize("vocab", [16384, 40000])
@pytest.mark.parametrize("p", [1.0, 0.9999999])
def test_a_last_token_that_weighs_nothing(rt, vocab, p):
    """The 260th token's weight, 2^-46.3, rounds to no unit of 2^-44. Those of
    the 259 before it are 2^44 units for the first and 2^44 - 1 for the others
    (each bin's sum rounded; y is 2^0, 2^(-28 log2 e) 255 times, ...), so u = 1 / 2
    asks for the place half a unit before the end of the first token. By the
    exact weights, which are up to half a unit per token off, it is the first's
    or the second's; the last one's chance is 2^-47."""
    x = np.full((1, vocab), -np.inf)
    values = [0.0] + [-28.0] * 255 + [-0.5, -0.93275213, -20.780386, -46.3 * np.log(2)]
    at = np.random.RandomState(3).permutation(vocab)[: len(values)]
    x[0, at] = np.float32(values)
    token, probability = call(rt, Rows(x, xpu.FP32, t=1.0, k=260, p=p, u=0.5))
    share = np.exp(np.float32([0.0, -0.5])) / 2  # of a sum of 2, to 2^-44
    i = [at[0], at[256]].index(token[0])
    assert abs(probability[0] - share[i]) <= 2.0 ** -22 * share[i]


@pytest.mark.parametrize("top,t", [(2.0 ** 24, 0.0185), (30.0, 3.5e-8), (-1e6, 1.2e-3), (1e30, 1.36e21)])
@pytest.mark.parametrize("vocab", [500, 20000])
def test_neighbouring_floats_far_apart(rt, top, t, vocab):
    """The next float below the largest logit is 78 powers of two less in weight:
    nothing, of however many tokens."""
    top = np.float32(top)
    x = np.full((3, vocab), np.nextafter(top, np.float32(-np.inf)))
    x[0, 77] = x[1, vocab - 1] = x[2, 0] = x[2, 300] = top
    gap = (float(top) - float(x[0, 0])) / t * 1.4427 * 32
    assert 2048 < gap < 3198  # in bins: past the slots, nearer to the last bin than the largest is
    for numbers in (dict(), dict(k=300), dict(p=0.99999), dict(k=40)):
        got = Rows(x, xpu.FP32, t=t, u=NEAR_ONE, **numbers).verify(rt)
        assert list(got) == [77, vocab - 1, 300]
