"""xpu_sample on gfx950 against the definition in 64 bits: the tokens exactly
(a random number would have to lie within 2^-28 of a token's share to be drawn
otherwise), the probabilities to 2^-23 of themselves (one rounding to FP32,
2^-24, and sums that are exact to 2^-28)."""
import ctypes

import numpy as np
import pytest
import torch

import xpu_playground_amd as xpu
from cache_util import Buffers

pytestmark = pytest.mark.gpu
TYPES = [xpu.BF16, xpu.FP16, xpu.FP32]
TORCH = {xpu.BF16: torch.bfloat16, xpu.FP16: torch.float16, xpu.FP32: torch.float32}
NONE = xpu.SAMPLE_NONE


def stored(x, dtype):
    """float array -> (raw array, values as float64)."""
    t = torch.from_numpy(np.asarray(x, np.float32)).to(TORCH[dtype])
    raw = t.view(torch.int32 if dtype == xpu.FP32 else torch.int16).numpy()
    return raw, t.double().numpy()


def expected(x, t=1.0, k=0, p=1.0, m=0.0, u=0.0):
    """One row: (token, probability)."""
    t, p, m, u = (np.float64(np.float32(v)) for v in (t, p, m, u))
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return NONE, np.nan
    if not (0 <= t < np.inf and p >= 0 and 0 <= m <= 1 and 0 <= u < 1):
        return NONE, np.nan
    order = np.lexsort((np.arange(len(x)), -(x + 0.0)))
    if t == 0:
        return int(order[0]), 1.0
    if k:
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / t)
    if p < 1:
        n = 1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))
        order, w = order[:n], w[:n]
    order, w = order[w >= m], w[w >= m]
    at = min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), len(w) - 1)
    return int(order[at]), w[at] / w.sum()


class Rows:
    """Logits of a batch with their numbers; None: not given."""

    def __init__(self, x, dtype, t=None, k=None, p=None, m=None, u=None, stride=None, shift=0, seed=1):
        self.x, self.dtype, (self.rows, self.vocab) = np.asarray(x, np.float32), dtype, np.shape(x)
        self.stride, self.shift = stride or self.vocab, shift
        of = lambda v, kind: None if v is None else np.broadcast_to(np.asarray(v, kind), (self.rows,)).copy()  # noqa: E731
        self.t, self.p, self.m, self.k = of(t, np.float32), of(p, np.float32), of(m, np.float32), of(k, np.uint32)
        self.u = of(np.random.RandomState(seed).rand(self.rows) if u is None else u, np.float32)
        self.u = np.where(self.u == 1, np.float32(1 - 2.0 ** -24), self.u) if u is None else self.u

    def device(self, b):
        raw, self.values = stored(self.x, self.dtype)
        full = np.full(self.shift + (self.rows - 1) * self.stride + self.vocab, -1, raw.dtype)  # NaN between the rows
        for i in range(self.rows):
            full[self.shift + i * self.stride: self.shift + i * self.stride + self.vocab] = raw[i]
        up = lambda v: None if v is None else b.up(v)  # noqa: E731
        s = xpu.Sampling(self.dtype, self.rows, self.vocab, b.up(self.u), up(self.t), up(self.k), up(self.p), up(self.m),
                         self.stride)
        size = b.rt.sample_workspace(s)
        return s, b.up(full) + self.shift * raw.itemsize, b.alloc(size), size

    def want(self):
        got = [expected(self.values[i], *(d if v is None else v[i] for d, v in ((1.0, self.t), (0, self.k), (1.0, self.p), (0.0, self.m))),
                        self.u[i]) for i in range(self.rows)]
        return np.array([g[0] for g in got], np.uint32), np.array([g[1] for g in got])

    def verify(self, rt):
        print(f"sample {self.rows} x {self.vocab} dtype {self.dtype} stride {self.stride} shift {self.shift} t {self.t} k {self.k} "
              f"p {self.p} m {self.m}"[:300], flush=True)
        with Buffers(rt) as b:
            s, logits, workspace, size = self.device(b)
            tokens, probability = b.up(np.full(self.rows + 1, 77, np.uint32)), b.up(np.full(self.rows + 1, 7.5, np.float32))
            rt.sample(s, logits, tokens, workspace, size, probability)
            rt.synchronize()
            got, prob = rt.download(tokens, self.rows + 1, np.uint32), rt.download(probability, self.rows + 1, np.float32)
            rt.sample(s, logits, tokens, workspace, size)  # without probabilities, the same again
            rt.synchronize()
            assert np.array_equal(rt.download(tokens, self.rows + 1, np.uint32), got)
            assert got[-1] == 77 and prob[-1] == 7.5
            token, share = self.want()
            assert np.array_equal(got[:-1], token), (np.flatnonzero(got[:-1] != token)[:5], got[:-1][got[:-1] != token][:5],
                                                     token[got[:-1] != token][:5])
            odd = np.isnan(share)
            assert np.array_equal(np.isnan(prob[:-1]), odd)
            assert (np.abs(prob[:-1][~odd] - share[~odd]) <= 2.0 ** -23 * share[~odd] + 1e-45).all()
        return got[:-1]


def logits(rows, vocab, seed, spread=2.5, peaks=30):
    r = np.random.RandomState(seed)
    x = r.randn(rows, vocab) * spread
    for i in range(rows):
        at = r.randint(0, vocab, min(peaks, vocab))
        x[i, at] += r.rand(len(at)) * 12
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 63, 64, 100, 1000, 4096, 8191, 32003, 151936])
def test_vocabularies(rt, dtype, vocab):
    rows = 6 if vocab > 5000 else 12
    Rows(logits(rows, vocab, vocab), dtype).verify(rt)
    Rows(logits(rows, vocab, vocab + 1), dtype, t=0.7, k=20, p=0.95).verify(rt)
    Rows(logits(rows, vocab, vocab + 2), dtype, t=1.3, p=0.9, m=0.02).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 2, 50, 255, 256, 257, 1000, 4999, 5000, 5001, 0xFFFFFFFF])
@pytest.mark.parametrize("p,m", [(1.0, 0.0), (0.8, 0.0), (1.0, 0.1), (0.95, 0.001)])
def test_filters_together(rt, dtype, k, p, m):
    Rows(logits(9, 5000, 3), dtype, t=1.1, k=k, p=p, m=m).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
def test_each_row_has_its_own_numbers(rt, dtype):
    n = 40
    r = np.random.RandomState(5)
    Rows(logits(n, 20011, 4), dtype, t=r.choice([0.0, 0.3, 1.0, 1.7], n), k=r.choice([0, 1, 5, 300, 50000], n),
         p=r.choice([0.0, 0.5, 0.99, 1.0, 2.0], n), m=r.choice([0.0, 0.01, 0.5, 1.0], n)).verify(rt)


@pytest.mark.parametrize("vocab", [5, 300, 2048, 2049, 30000])
@pytest.mark.parametrize("k", [0, 3, 200, 1000])
def test_equal_logits(rt, vocab, k):
    """All alike, and two values alone: the lowest ids first."""
    u = np.array([0.0, 0.25, 0.5, 1 - 2.0 ** -24, 0.3], np.float32)
    for p in (1.0, 0.3, 0.0):
        Rows(np.full((5, vocab), -3.25), xpu.BF16, k=k, p=p, u=u).verify(rt)
        x = np.where(np.arange(vocab) % 3 == 1, 2.0, 1.0)
        Rows(np.tile(x, (5, 1)), xpu.FP32, t=0.9, k=k, p=p, u=u).verify(rt)


def test_the_largest_vocabulary_alike(rt):
    """2^20 equal tokens: a bin that is divided down to the ids."""
    u = np.array([0.0, 0.123456, 1 - 2.0 ** -24], np.float32)
    Rows(np.zeros((3, 1 << 20)), xpu.BF16, u=u).verify(rt)
    Rows(np.zeros((3, 1 << 20)), xpu.BF16, u=u, k=777777, p=0.77).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_tokens(rt, dtype):
    """-infinity is never drawn, also where top-k has to take it."""
    x = logits(8, 3000, 6)
    x[0, 1:] = x[1, :-1] = x[2, 2::2] = -np.inf
    x[3, np.random.RandomState(1).permutation(3000)[:2990]] = -np.inf
    x[4] = -np.inf
    x[5, 5] = np.nan
    x[6, 2999] = np.inf
    u = np.full(8, 1 - 2.0 ** -24, np.float32)
    for k in (0, 50, 700):
        for p in (1.0, 0.999):
            got = Rows(x, dtype, k=k, p=p, u=u).verify(rt)
            assert list(got[4:7]) == [NONE] * 3 and got[0] == 0 and got[1] == 2999


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [9000, 40000, 151936])
def test_few_tokens_that_are_not_masked(rt, dtype, vocab):
    """Whole parts of a row are -infinity or the type's lowest number, first,
    last or in between."""
    lowest = float(torch.finfo(TORCH[dtype]).min)
    x = logits(8, vocab, 13)
    for i, mask in enumerate((-np.inf, lowest)):
        x[4 * i, : vocab - 5] = mask
        x[4 * i + 1, 5:] = mask
        x[4 * i + 2, : vocab // 2] = x[4 * i + 2, vocab // 2 + 3000:] = mask
        x[4 * i + 3, np.random.RandomState(i).permutation(vocab)[: vocab - 40]] = mask
    for k in (0, 20, 300):
        for p in (1.0, 0.9):
            Rows(x, dtype, t=0.8, k=k, p=p, m=0.001).verify(rt)
            Rows(x, dtype, t=3e38, k=k, p=p).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
def test_logits_that_rise_and_fall(rt, dtype):
    """The largest so far changes all the way through a row, and by powers of
    two beyond those that the histogram holds at a time."""
    at = np.arange(50000)
    x = np.stack([at * 2e-4, 10 - at * 2e-4, at * 0.01 - 500, 500 - at * 0.01, np.sin(at / 3000) * 90, at // 1000 * 20.0 - 999])
    for numbers in (dict(), dict(p=0.95), dict(k=2000, p=0.9), dict(k=30), dict(m=0.2), dict(t=7.0, p=0.7)):
        Rows(x, dtype, **numbers).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
def test_numbers_out_of_range(rt, dtype):
    x = logits(1, 500, 7)
    bad = [dict(t=-1.0), dict(t=np.nan), dict(t=np.inf), dict(p=-0.1), dict(p=np.nan), dict(m=-0.1), dict(m=1.5),
           dict(m=np.nan), dict(u=-0.1), dict(u=1.0), dict(u=np.nan)]
    for numbers in bad:
        assert Rows(x, dtype, **numbers).verify(rt)[0] == NONE


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1e-45, 1e-30, 1e-3, 30.0, 1e30, 3e38])
def test_temperatures(rt, dtype, t):
    Rows(logits(6, 4001, 8), dtype, t=t).verify(rt)
    Rows(logits(6, 4001, 9), dtype, t=t, k=40, p=0.9).verify(rt)


def test_logits_far_apart(rt):
    """Differences that pass FP32's range, denormal logits, zeros of both signs."""
    r = np.random.RandomState(9)
    x = np.clip(r.randn(6, 3000) * 1e38, -3.4e38, 3.4e38).astype(np.float32)
    x[1] = np.float32(r.randn(3000)) * np.float32(1e-42)
    x[2] = np.where(r.rand(3000) < 0.5, 0.0, -0.0)
    x[3, :] = -3.4e38
    x[3, 17] = 3.4e38
    for t in (1.0, 1e38):
        for k in (0, 30, 500):
            Rows(x, xpu.FP32, t=t, k=k, p=0.9).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,stride,shift", [(1001, 1001, 0), (1001, 1003, 1), (4096, 4097, 3), (999, 1024, 5)])
def test_rows_anywhere(rt, dtype, vocab, stride, shift):
    """Rows at any element, NaN between them."""
    Rows(logits(7, vocab, 10), dtype, t=0.9, k=30, stride=stride, shift=shift).verify(rt)
    Rows(logits(7, vocab, 11), dtype, p=0.9, stride=stride, shift=shift).verify(rt)


def test_greedy_is_the_lowest_of_the_largest(rt):
    x = np.zeros((3, 5000))
    x[0, [4000, 17, 900]] = 5
    x[1, 4999] = 5
    for numbers in (dict(t=0.0), dict(k=1), dict(p=0.0), dict(m=1.0, u=0.0)):
        assert list(Rows(x, xpu.BF16, **numbers).verify(rt)) == [17, 4999, 0]


def test_no_numbers_at_all_and_no_rows(rt):
    Rows(logits(3, 700, 12), xpu.FP16).verify(rt)
    with Buffers(rt) as b:
        s = xpu.Sampling(xpu.BF16, 0, 100, None)
        assert rt.sample_workspace(s) == 0
        rt.sample(s, None, None)


def test_shares_of_many_draws(rt):
    """512 evenly spaced random numbers draw every token of a small row as often
    as its share says, to one draw at each end of its range."""
    x = np.tile([1.0, 0.0, 2.0, -1.0, 0.5], (512, 1))
    u = (np.arange(512) + 0.5) / 512
    got = Rows(x, xpu.FP32, u=u).verify(rt)
    w = np.exp(x[0]) / np.exp(x[0]).sum()
    assert (np.abs(np.bincount(got, minlength=5) - 512 * w) <= 1).all()


def test_captured(rt):
    """A graph of a call, replayed over other logits and numbers with eager calls
    between."""
    n, vocab = 5, 9001
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
