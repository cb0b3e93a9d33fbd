"""xpu_sample on gfx950 where its launches meet: bins whose weight rounds to
nothing."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import Buffers
from test_gpu_sample import Rows

pytestmark = pytest.mark.gpu


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
