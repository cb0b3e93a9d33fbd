"""xpu_prompt_attention at its edges: starts that do not fit among many
sequences, out beside q in one buffer, what unseen keys hold."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, INF, NAN, Buffers, attend, check, normal, u32, values
from test_gpu_prompt_attention import expected, launch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 2), (8, 2)])
@pytest.mark.parametrize("n", [60, 70, 130, 400])
@pytest.mark.parametrize("what", ["past the rows", "back", "another order", "keys"])
def test_starts_that_do_not_fit_among_many(rt, heads, kv, n, what):
    """However many sequences there are, those whose starts fit are served, and
    the rows of the others are left."""
    dtype, d = xpu.BF16, 64
    rng = np.random.RandomState(n)
    lengths = rng.choice([0, 1, 3, 40, 150 if n < 100 else 5], n)
    lengths[:5] = 33, 7, 65, 12, 40
    q_starts = np.concatenate([[2], 2 + np.cumsum(lengths)]).astype(np.int64)
    rows = int(q_starts[-1]) + 3
    k_starts = q_starts.copy()
    bad = rng.choice(np.arange(1, n - 1), 4, replace=False)
    bad[0] = 3
    if what == "past the rows":
        q_starts[bad] = rows + 1 + bad
    elif what == "back":
        q_starts[bad] = q_starts[bad - 1] - 1
    elif what == "another order":  # the first half of the sequences has the later rows
        half = n // 2
        q_starts = np.concatenate([q_starts[half:], q_starts[:half + 1]])
        k_starts = q_starts.copy()
    else:
        k_starts[bad] = rows + 7
    count = len(q_starts) - 1
    holders, served = np.zeros(rows, int), []
    for s in range(count):
        a, b, c, e = q_starts[s], q_starts[s + 1], k_starts[s], k_starts[s + 1]
        if a <= b <= rows and c <= e <= rows:
            served.append(s)
            holders[a:b] += 1
    q, k, v = normal((rows, heads, d), 1, dtype), normal((rows, kv, d), 2, dtype), normal((rows, kv, d), 3, dtype)
    print(f"prompt attention {count} sequences heads {heads}/{kv} starts {what}", flush=True)
    got = values(launch(rt, q, k, v, u32(q_starts), u32(k_starts), dtype), dtype)
    assert (got[holders == 0] == values(np.array([GUARD], np.uint16), dtype)[0]).all()
    qf, kf, vf = values(q, dtype), values(k, dtype), values(v, dtype)
    checked = 0
    for s in served:
        a, b, c, e = (int(x[i]) for x, i in ((q_starts, s), (q_starts, s + 1), (k_starts, s), (k_starts, s + 1)))
        one = holders[a:b] == 1  # rows that two sequences claim are either's
        seen = np.arange(e - c)[None, :] <= np.arange(b - a)[:, None] + (e - c) - (b - a)
        for h in range(heads):
            g = h // (heads // kv)
            want, tol = attend(qf[a:b, h], kf[c:e, g], vf[c:e, g], seen, d ** -0.5, dtype)
            check(got[a:b, h][one], want[one], tol[one], f"sequence {s} head {h}")
        checked += int(one.sum())
    assert checked > rows // 4


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
@pytest.mark.parametrize("before", [False, True])
def test_out_beside_q_in_one_buffer(rt, dtype, before):
    """q and out as columns of one buffer, in either order."""
    heads, d, n = 4, 64, 150
    x = np.full((n, 2 * heads * d + 8), GUARD, np.uint16)
    at_q, at_out = (heads * d + 8, 0) if before else (0, heads * d + 8)
    q, k, v = normal((n, heads, d), 1, dtype), normal((n, 2, d), 2, dtype), normal((n, 2, d), 3, dtype)
    x[:, at_q:at_q + heads * d] = q.reshape(n, -1)
    starts = u32([1, 100, 149])
    want, tol = expected(q, k, v, starts, starts, d ** -0.5, dtype, np.full(q.shape, GUARD, np.uint16))
    with Buffers(rt) as b:
        at = b.up(x)
        p = xpu.Packed(dtype, heads, 2, d, 2, n, b.up(starts), q_stride=x.shape[1], out_stride=x.shape[1])
        rt.prompt_attention(p, at + 2 * at_q, b.up(k), b.up(v), at + 2 * at_out)
        rt.synchronize()
        y = rt.download(at, x.size, np.uint16).reshape(x.shape)
    check(values(y[:, at_out:at_out + heads * d].reshape(q.shape), dtype), want, tol)
    y[:, at_out:at_out + heads * d] = GUARD
    assert np.array_equal(y, x)


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("at", [1, 5, 40, 63, 64, 131, 199])
def test_unseen_keys_change_no_bit(rt, dtype, d, bad, at):
    """Every query before a key gives the same bits whatever the key and its
    value are: also the queries of the tile that the key is in, whose scores of
    it are masked and whose part of its value is 0."""
    n, code = 200, (NAN if bad == "nan" else INF)[dtype]
    q, k, v = normal((n, 2, d), 1, dtype), normal((n, 2, d), 2, dtype), normal((n, 2, d), 3, dtype)
    starts = u32([0, n])
    clean = launch(rt, q, k, v, starts, starts, dtype, shared=True)
    k[at], v[at] = code, code
    got = launch(rt, q, k, v, starts, starts, dtype, shared=True)
    assert at and np.array_equal(got[:at], clean[:at])
    assert not np.isfinite(values(got[at:], dtype)).any()
