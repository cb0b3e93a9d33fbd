"""xpu_prompt_attention on gfx950 against attention in 64 bits (the bound is
derived in cache_util.py): packed sequences of ragged lengths, keys before the
queries, queries that see nothing, strides, in place, values that only unseen
keys hold, starts that do not fit, capture."""
import ctypes

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, INF, NAN, Buffers, attend, check, codes, normal, u32, values

pytestmark = pytest.mark.gpu

TYPES = [xpu.BF16, xpu.FP16]


def sums(lengths, first=0):
    return u32(np.cumsum([first] + list(lengths)))


def expected(q, k, v, q_starts, k_starts, scale, dtype, out):
    """out (codes before the call) with the sequences' rows computed, and the bound."""
    heads, kv = q.shape[1], k.shape[1]
    want, tol = values(out, dtype).copy(), np.zeros(out.shape)
    qf, kf, vf = values(q, dtype), values(k, dtype), values(v, dtype)
    for s in range(len(q_starts) - 1):
        a, b, c, d = (int(x) for x in (q_starts[s], q_starts[s + 1], k_starts[s], k_starts[s + 1]))
        n, m = b - a, d - c
        seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + m - n
        for h in range(heads):
            g = h // (heads // kv)
            want[a:b, h], tol[a:b, h] = attend(qf[a:b, h], kf[c:d, g], vf[c:d, g], seen, scale, dtype)
    return want, tol


def launch(rt, q, k, v, q_starts, k_starts, dtype, scale=None, out=None, shared=False):
    heads, d = q.shape[1:]
    out = np.full(q.shape, GUARD, np.uint16) if out is None else out
    with Buffers(rt) as b:
        dq, dk, dv, do = b.up(q), b.up(k), b.up(v), b.up(out)
        p = xpu.Packed(dtype, heads, k.shape[1], d, len(q_starts) - 1, len(q), b.up(q_starts), len(k),
                       None if shared else b.up(k_starts), scale)
        rt.prompt_attention(p, dq, dk, dv, do)
        rt.synchronize()
        return rt.download(do, out.size, np.uint16).reshape(out.shape)


def run(rt, lengths, priors, heads, kv, d, dtype, seed, scale=None, gain=1.0):
    q_starts, k_starts = sums(lengths), sums([n + p for n, p in zip(lengths, priors)])
    q = normal((max(int(q_starts[-1]), 1), heads, d), seed, dtype, gain)
    k = normal((max(int(k_starts[-1]), 1), kv, d), seed + 1, dtype, gain)
    v = normal((max(int(k_starts[-1]), 1), kv, d), seed + 2, dtype)
    print(f"prompt attention {lengths} priors {priors} heads {heads}/{kv} d {d} dtype {dtype}", flush=True)
    out = np.full(q.shape, GUARD, np.uint16)
    got = launch(rt, q, k, v, q_starts, k_starts, dtype, scale, out, shared=not any(priors))
    want, tol = expected(q, k, v, q_starts, k_starts, d ** -0.5 if scale is None else scale, dtype, out)
    check(values(got, dtype), want, tol)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,heads,kv", [
    ([1], 1, 1), ([2], 2, 1), ([31], 4, 2), ([32], 3, 3), ([33], 4, 2), ([64], 2, 2), ([65], 6, 2), ([127], 2, 1),
    ([128], 8, 8), ([129], 4, 1), ([257], 2, 1), ([512], 1, 1), ([0, 1, 0, 0, 63, 128, 0], 4, 2),
    ([5, 200, 1, 129, 64, 31], 4, 2), ([1] * 70, 8, 8), ([3, 0, 300, 17] * 20, 2, 1)])
def test_packed_lengths(rt, dtype, d, lengths, heads, kv):
    run(rt, lengths, [0] * len(lengths), heads, kv, d, dtype, 100 + len(lengths))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,priors", [
    ([1], [1]), ([1], [500]), ([70], [63]), ([128, 3], [129, 1000]), ([200, 1, 40], [0, 64, 777]),
    # fewer keys than queries: the first queries see nothing
    ([10], [-3]), ([200], [-70]), ([129, 64, 5], [-129, -64, -1]), ([300, 20], [-200, 5])])
def test_keys_before_the_queries_and_queries_without_keys(rt, dtype, d, lengths, priors):
    run(rt, lengths, priors, 4, 2, d, dtype, 300 + len(lengths))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,gain", [(0.02, 1.0), (1.0, 1.0), (0.125, 6.0)])
def test_scales_and_rising_scores(rt, dtype, scale, gain):
    """Scores far apart: the reference maximum moves many times, and most
    probabilities vanish."""
    run(rt, [300, 90], [0, 20], 2, 1, 128, dtype, 400, scale, gain)


@pytest.mark.parametrize("dtype", TYPES)
def test_ascending_scores(rt, dtype):
    """Every key's score passes all before it, by more than a rescale's threshold."""
    n, d = 200, 64
    q = codes(np.ones((n, 1, d)), dtype)
    k = codes(np.repeat(np.arange(n)[:, None, None] / 8.0, d, 2), dtype)
    v = normal((n, 1, d), 5, dtype)
    starts = sums([n])
    got = launch(rt, q, k, v, starts, starts, dtype, 1.0, shared=True)
    want, tol = expected(q, k, v, starts, starts, 1.0, dtype, np.zeros(q.shape, np.uint16))
    check(values(got, dtype), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [6.0, 10.4, 11.1, 13.9, 16.0])
def test_many_small_probabilities(rt, dtype, shift):
    """One key far above thousands of others, whose probabilities are in or
    below the subnormal range of fp16 and together make a good part of the sum."""
    n, d = 4000, 64
    q, k = codes(np.ones((1, 1, d)), dtype), np.full((n, 1, d), -shift / d, np.float32)
    k[1234] = 0
    v = np.ones((n, 1, d), np.float32)
    v[1234] = 0
    k, v = codes(k, dtype), codes(v, dtype)
    got = launch(rt, q, k, v, u32([0, 1]), u32([0, n]), dtype, 1.0)
    want, tol = expected(q, k, v, u32([0, 1]), u32([0, n]), 1.0, dtype, np.zeros(q.shape, np.uint16))
    check(values(got, dtype), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("at", [5, 40, 63, 64, 131, 199])
def test_unseen_keys_take_no_part(rt, dtype, d, bad, at):
    """A non-finite key and value late in the prompt: the queries before it
    give exactly what they give without it, those after it the formula's."""
    n, code = 200, (NAN if bad == "nan" else INF)[dtype]
    q, k, v = normal((n, 2, d), 1, dtype), normal((n, 2, d), 2, dtype), normal((n, 2, d), 3, dtype)
    starts = sums([n])
    clean = launch(rt, q, k, v, starts, starts, dtype, shared=True)
    k2, v2 = k.copy(), v.copy()
    k2[at, 0, 3] = code
    v2[at, 1, d - 1] = code
    got = launch(rt, q, k2, v2, starts, starts, dtype, shared=True)
    want, tol = expected(q, k, v, starts, starts, d ** -0.5, dtype, np.zeros(q.shape, np.uint16))
    check(values(got[:at], dtype), want[:at], tol[:at], "before")
    check(values(got[at:, 1, : d - 1], dtype), want[at:, 1, : d - 1], tol[at:, 1, : d - 1], "other dims")
    later = values(got[at:], dtype)
    if bad == "nan":
        assert np.isnan(later[:, 0]).all() and np.isnan(later[:, 1, d - 1]).all()
    else:
        assert not np.isfinite(later[:, 1, d - 1]).any()
    assert np.array_equal(got[: at // 64 * 64 // 128 * 128], clean[: at // 64 * 64 // 128 * 128])


@pytest.mark.parametrize("dtype", TYPES)
def test_later_sequences_values_do_not_reach_earlier_ones(rt, dtype):
    lengths, d = [70, 33, 129], 128
    starts = sums(lengths)
    q, k, v = (normal((int(starts[-1]), 2, d), s, dtype) for s in (1, 2, 3))
    k[starts[1]:starts[2]] = NAN[dtype]
    v[starts[1]:starts[2]] = INF[dtype]
    got = values(launch(rt, q, k, v, starts, starts, dtype, shared=True), dtype)
    want, tol = expected(q, k, v, starts, starts, d ** -0.5, dtype, np.zeros(q.shape, np.uint16))
    for s in (0, 2):
        check(got[starts[s]:starts[s + 1]], want[starts[s]:starts[s + 1]], tol[starts[s]:starts[s + 1]])
    assert np.isnan(got[starts[1]:starts[2]]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_one_interleaved_buffer_in_place(rt, dtype, d):
    """q, k and v as columns of one row (the output of one projection), the
    result over q; rows of no sequence and the columns behind stay."""
    heads, kv, lengths, first = 4, 2, [100, 31], 3
    starts = sums(lengths, first)
    rows, width = int(starts[-1]) + 5, (heads + 2 * kv) * d + 8
    x = normal((rows, width), 9, dtype)
    q = x[:, : heads * d].reshape(rows, heads, d)
    k = x[:, heads * d: (heads + kv) * d].reshape(rows, kv, d)
    v = x[:, (heads + kv) * d: (heads + 2 * kv) * d].reshape(rows, kv, d)
    want, tol = expected(q, k, v, starts, starts, d ** -0.5, dtype, q)
    with Buffers(rt) as b:
        at = b.up(x, pad=16)
        p = xpu.Packed(dtype, heads, kv, d, len(lengths), rows, b.up(starts), q_stride=width, k_stride=width,
                       v_stride=width, out_stride=width)
        rt.prompt_attention(p, at, at + heads * d * 2, at + (heads + kv) * d * 2, at)
        rt.synchronize()
        y = rt.download(at, x.size, np.uint16).reshape(x.shape)
    assert np.array_equal(y[:, heads * d:], x[:, heads * d:])
    assert np.array_equal(y[:first], x[:first]) and np.array_equal(y[starts[-1]:], x[starts[-1]:])
    check(values(y[:, : heads * d].reshape(q.shape), dtype), want, tol)


def test_starts_that_do_not_fit_touch_nothing(rt):
    """Descending starts, starts past the rows: the kernel leaves those
    sequences' rows and serves the others."""
    dtype, d, rows = xpu.BF16, 64, 100
    q, k, v = (normal((rows, 2, d), s, dtype) for s in (1, 2, 3))
    for q_starts, k_starts, served in [([0, 40, 30, 30], [0, 40, 40, 40], [0]), ([0, 20, 200], [0, 20, 100], [0]),
                                       ([0, 20, 60], [0, 300, 60], []), ([50, 20], [0, 20], [])]:
        got = launch(rt, q, k, v, u32(q_starts), u32(k_starts), dtype)
        want, tol = values(np.full(q.shape, GUARD, np.uint16), dtype), np.zeros(q.shape)
        for s in served:
            a, b = q_starts[s], q_starts[s + 1]
            w, t = expected(q, k, v, u32([a, b]), u32(k_starts[s:s + 2]), d ** -0.5, dtype,
                            np.full(q.shape, GUARD, np.uint16))
            want[a:b], tol[a:b] = w[a:b], t[a:b]
        check(values(got, dtype), want, tol, f"{q_starts} {k_starts}")


def test_no_key_rows_at_all(rt):
    q = normal((40, 2, 64), 1, xpu.BF16)
    with Buffers(rt) as b:
        do = b.up(np.full(q.shape, GUARD, np.uint16))
        p = xpu.Packed(xpu.BF16, 2, 2, 64, 1, 40, b.up(u32([0, 40])), 0, b.up(u32([0, 0])))
        rt.prompt_attention(p, b.up(q), 0, 0, do)
        rt.synchronize()
        assert not rt.download(do, q.size, np.uint16).any()


def test_nothing_to_do(rt):
    rt.prompt_attention(xpu.Packed(xpu.BF16, 2, 2, 64, 0, 0, None), 0, 0, 0, 0)
    rt.prompt_attention(xpu.Packed(xpu.BF16, 2, 2, 64, 3, 0, None), 0, 0, 0, 0)


def test_same_bits_every_time_and_captured(rt):
    """Two shapes captured in two graphs, replayed with eager calls between."""
    cases = []
    with Buffers(rt) as b:
        for lengths, seed in (([300, 40, 1], 1), ([64, 500], 5)):
            starts = sums(lengths)
            q, k, v = (normal((int(starts[-1]), 4, 128), seed + i, xpu.BF16) for i in range(3))
            k, v = k[:, :2].copy(), v[:, :2].copy()
            do = b.up(np.zeros(q.shape, np.uint16))
            args = (xpu.Packed(xpu.BF16, 4, 2, 128, len(lengths), len(q), b.up(starts)), b.up(q), b.up(k), b.up(v), do)
            rt.prompt_attention(*args)
            rt.synchronize()
            eager = rt.download(do, q.size, np.uint16)
            xpu.check(rt.lib.xpu_rt_capture_begin(rt.handle))
            rt.prompt_attention(*args)
            graph = ctypes.c_void_p()
            xpu.check(rt.lib.xpu_rt_capture_end(rt.handle, ctypes.byref(graph)))
            cases.append((args, eager, graph))
        for _ in range(3):
            for args, eager, graph in cases:
                rt.copy_to(args[4], np.zeros(eager.size, np.uint16))
                xpu.check(rt.lib.xpu_rt_graph_launch(rt.handle, graph))
                rt.synchronize()
                assert np.array_equal(rt.download(args[4], eager.size, np.uint16), eager)
                rt.prompt_attention(*args)
                rt.synchronize()
                assert np.array_equal(rt.download(args[4], eager.size, np.uint16), eager)
        for _, _, graph in cases:
            rt.lib.xpu_rt_graph_destroy(graph)
