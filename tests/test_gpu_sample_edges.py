"""xpu_sample on gfx950 where its launches meet: bins whose weight rounds to
nothing, temperatures at which neighbouring floats are further apart than the
histogram is long, rows cut into one and two parts, and the three launches
captured and over rows at any element. The definition in 64 bits and its
tolerances are those of test_gpu_sample.py."""
import ctypes

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import Buffers
from test_gpu_sample import TYPES, Rows, logits, stored

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


def mixed(rows, vocab, seed, dtype, ties):
    r = np.random.RandomState(seed)
    x = logits(rows, vocab, seed)
    if ties:  # most tokens alike: lists that are not whole, bins that are divided down to the ids
        x[::3] = np.where(r.rand(len(x[::3]), vocab) < 0.6, 1.5, x[::3] * 0.25)
        x[1::7] = -2.25
    k = np.array([0, 20, 1000, 256, 257, 5, 60000])[np.arange(rows) % 7]
    return Rows(x, dtype, t=r.choice([0.4, 0.8, 1.0, 1.6], rows), k=k, p=r.choice([0.6, 0.95, 1.0], rows),
                m=r.choice([0.0, 0.0, 0.01, 0.3], rows), seed=seed)


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("rows,vocab,dtype", [(70, 16384, xpu.BF16), (70, 20011, xpu.FP32), (130, 32003, xpu.FP16),
                                              (130, 16384, xpu.FP32), (260, 17001, xpu.BF16), (33, 32003, xpu.BF16)])
def test_rows_of_few_parts(rt, rows, vocab, dtype, ties):
    """Rows in four, two and one parts on 256 compute units, and more rows than
    those."""
    mixed(rows, vocab, rows + vocab, dtype, ties).verify(rt)


@pytest.mark.parametrize("ties", [False, True])
def test_a_row_alone_and_among_others(rt, ties):
    """However a row is cut, it draws the same token, with its share to one
    rounding; alike rows of a batch have the same bits."""
    base = mixed(7, 32003, 5, xpu.BF16, ties)
    numbers = {n: getattr(base, n) for n in "tkpmu"}
    whole = call(rt, Rows(np.tile(base.x, (20, 1)), base.dtype, **{n: np.tile(v, 20) for n, v in numbers.items()}))
    for i in range(7):
        token, probability = call(rt, Rows(base.x[i: i + 1], base.dtype, **{n: v[i: i + 1] for n, v in numbers.items()}))
        assert (whole[0][i::7] == token[0]).all()
        assert len(np.unique(whole[1][i::7])) == 1
        assert abs(whole[1][i] - probability[0]) <= 2.0 ** -23 * probability[0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,stride,shift", [(16385, 16385, 1), (20011, 20013, 3), (32003, 32768, 5)])
def test_rows_anywhere_in_parts(rt, dtype, vocab, stride, shift):
    for numbers in (dict(k=30), dict(p=0.9), dict(k=700, m=0.01)):
        Rows(logits(5, vocab, 10), dtype, t=0.9, stride=stride, shift=shift, **numbers).verify(rt)


@pytest.mark.parametrize("n", [5, 70])
def test_captured_in_parts(rt, n):
    """The three launches in a graph, over other logits and numbers with eager
    calls between."""
    vocab = 17001
    first = Rows(logits(n, vocab, 20), xpu.BF16, t=0.8, k=40, p=0.9, m=0.01)
    with Buffers(rt) as b:
        s, ptr, workspace, size = first.device(b)
        tokens, eager = b.alloc(4 * n), b.alloc(4 * n)
        rt.sample(s, ptr, tokens, workspace, size)
        rt.synchronize()
        xpu.check(rt.lib.xpu_rt_capture_begin(rt.handle))
        rt.sample(s, ptr, tokens, workspace, size)
        graph = ctypes.c_void_p()
        xpu.check(rt.lib.xpu_rt_capture_end(rt.handle, ctypes.byref(graph)))
        for i in range(4):
            r = Rows(logits(n, vocab, 21 + i), xpu.BF16, t=0.7 + 0.2 * i, k=[40, 0, 500, 3][i], p=0.9, m=0.01, seed=i)
            raw, r.values = stored(r.x, r.dtype)
            for at, v in ((ptr, raw), (s.random, r.u), (s.temperature, r.t), (s.top_k, r.k)):
                rt.copy_to(at, v)
            xpu.check(rt.lib.xpu_rt_graph_launch(rt.handle, graph))
            rt.sample(s, ptr, eager, workspace, size)
            rt.synchronize()
            got = rt.download(tokens, n, np.uint32)
            assert np.array_equal(got, r.want()[0]) and np.array_equal(rt.download(eager, n, np.uint32), got)
        rt.lib.xpu_rt_graph_destroy(graph)
