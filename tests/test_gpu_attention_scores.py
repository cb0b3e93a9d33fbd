"""Both attentions (xpu_prompt_attention, xpu_tree_attention) where the scores
are large numbers, against the softmax in 64 bits.

The scores of these tests are exact in FP32 whatever the order of the sum:
q = (A, 1, 0, ...) and k_j = (A', t_j, 0, ...) give A A' + t_j with A, A' powers
of two and t_j multiples of the spacing of the floats there. So nothing is lost
before the softmax, and of the bound of cache_util there remains, with u half a
step of the type: p's relative error e = |s_j - m| scale 2^-22 (the difference
is exact; scale log2 e and the product are rounded) and 2^-20 for exp2, twice;
p's rounding to the type (u, and in fp16 2^-25 below its normal range, relative
to the largest p); the FP32 sums (n 2^-22); the result's rounding."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, HALF_STEP, TINY, Buffers, check, codes, normal, u32, values

pytestmark = pytest.mark.gpu


def prompt(rt, q, k, v, dtype, scale):
    """Every query row sees all keys: it is a sequence's last one. One row per call."""
    out = np.empty_like(q)
    with Buffers(rt) as b:
        dk, dv, do = b.up(k), b.up(v), b.up(np.full(q[:1].shape, GUARD, np.uint16))
        for i in range(len(q)):
            p = xpu.Packed(dtype, q.shape[1], k.shape[1], q.shape[2], 1, 1, b.up(u32([0, 1])), len(k), b.up(u32([0, len(k)])),
                           scale)
            rt.prompt_attention(p, b.up(q[i:i + 1]), dk, dv, do)
            rt.synchronize()
            out[i] = rt.download(do, q[0].size, np.uint16).reshape(q[0].shape)
    return out


def tree(rt, q, k, v, dtype, scale):
    """The keys are a context, the queries nodes behind it that see nothing else."""
    n, heads, d = q.shape
    kv, page, keys = k.shape[1], 64, len(k)
    pages = (keys + n + page - 1) // page
    pools = [np.zeros((1, pages, kv, page, d), np.uint16) for _ in range(2)]
    for pool, rows in zip(pools, (k, v)):
        for i in range(keys):
            pool[0, i // page, :, i % page] = rows[i]
    with Buffers(rt) as b:
        cache = xpu.Cache(dtype, 1, kv, d, page, pages, b.up(pools[0]), b.up(pools[1]))
        batch = xpu.Batch(1, n, pages, b.up(u32(range(pages))), b.up(u32([0, n])), b.up(u32([keys])))
        size, do = rt.tree_attention_workspace(cache, batch, heads), b.up(np.full(q.shape, GUARD, np.uint16))
        rt.tree_attention(cache, batch, 0, heads, b.up(q), do, b.alloc(size), size, scale=scale,
                          visible=b.up(np.zeros(n, np.uint64)))
        rt.synchronize()
        return rt.download(do, q.size, np.uint16).reshape(q.shape)


def softmax(scores, v, scale, dtype):
    """scores [rows][keys] exact; (result, bound)."""
    out, tol = [], []
    u = HALF_STEP[dtype]
    for s in scores:
        w = np.exp((s - s.max()) * scale)
        w /= w.sum()
        o, size = w @ v, w @ np.abs(v)
        live = w > 2.0 ** -40  # the others weigh nothing, whatever their error
        e = np.abs(s[live] - s.max()).max() * scale * 2.0 ** -22 + 2.0 ** -19
        t = (u + 2 * e + len(s) * 2.0 ** -22) * size + 2 * u * np.abs(o) + TINY[dtype]
        t += 2.0 ** -25 * (np.abs(v).sum(0) + len(s) * np.abs(o)) if dtype == xpu.FP16 else len(s) * 2.0 ** -40
        out.append(o)
        tol.append(t * (1 + 3 * u))
    return np.array(out), np.array(tol)


LARGE = [  # type, log2 of A and A', spacing of the t_j, scales
    (xpu.FP16, 10, 10, 0.25, [0.3, 1.0, 5.0]), (xpu.FP16, 13, 13, 8, [0.05, 0.21, 1.0]),
    (xpu.FP16, 15, 15, 128, [0.011, 0.0127, 0.3, 0.77, 7.0, 1000.0]),
    (xpu.BF16, 10, 10, 0.25, [0.3, 1.0, 5.0]), (xpu.BF16, 15, 15, 128, [0.011, 0.0127, 0.3, 7.0]),
    (xpu.BF16, 18, 18, 8192, [0.0002, 0.9, 3.0, 77.0]), (xpu.BF16, 60, 50, 2.0 ** 87, [1e-26, 3e-20, 0.1]),
    (xpu.BF16, 60, 60, 2.0 ** 116, [1e6])]  # the differences times the scale pass the floats, too


@pytest.mark.parametrize("attention", [prompt, tree])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,a,b,step,scales", LARGE)
def test_large_scores(rt, attention, d, sign, dtype, a, b, step, scales):
    """Scores whose products with scale log2 e a float holds to many powers of
    two only: the softmax takes their differences, which are exact."""
    n, rng = 700, np.random.RandomState(a + 100 * d + sign)
    # the largest is no power of two, whose product with scale log2 e would be exact
    t = rng.choice([-7, -8, -9, -10, -12, -15], n) * float(step)
    t[:40] -= 8 * step  # rising scores: the reference moves
    t[400:] -= 8 * step  # and whole tiles far below it
    q, k = np.zeros((2, 2, d)), np.zeros((n, 2, d))
    q[:, :, 0], q[:, :, 1] = 2.0 ** a, 1
    q[1, 1, 0] *= 0.5  # rows of one tile with other references
    k[:, :, 0], k[:, :, 1] = sign * 2.0 ** b, t[:, None]
    q, k, v = codes(q, dtype), codes(k, dtype), normal((n, 2, d), 3, dtype)
    qf, kf, vf = (values(x, dtype) for x in (q, k, v))
    for scale in scales:
        print(f"large scores {attention.__name__} d {d} dtype {dtype} 2^{a + b} scale {scale} sign {sign}", flush=True)
        got = values(attention(rt, q, k, v, dtype, scale), dtype)
        for h in range(2):
            scores = qf[:, h, :2] @ kf[:, h, :2].T
            assert np.array_equal(scores, scores.astype(np.float32))
            want, tol = softmax(scores, vf[:, h], float(np.float32(scale)), dtype)
            check(got[:, h], want, tol, f"scale {scale} head {h}")


def far_below(shift, d, n, every):
    """Keys whose score is `shift` below that of one key in `every`, which has the value 0."""
    k, v = np.zeros((n, 1, d)), np.full((n, 1, d), 1024.0)
    top = np.arange(n) % every == 5 % every
    k[~top, 0, 1], v[top] = -shift, 0
    return k, v, top


@pytest.mark.parametrize("attention", [prompt, tree])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shift", [9.0, 10.4, 13.0, 16.0, 17.25, 18.0])
@pytest.mark.parametrize("n,every", [(700, 32), (100000, 100000)])
def test_many_keys_far_below_the_largest_in_fp16(rt, attention, d, shift, n, every):
    """The probabilities e^-9 .. e^-18 of most keys are 2^-13 .. 2^-26, around
    the end of fp16's normal range and far into the range below it. The result
    is their part of the sum, which is all that the bound goes by. p is scaled by
    2^7 before it is rounded, so its absolute rounding below the normal range is
    2^-25 / 2^7 = 2^-32 of the largest."""
    dtype = xpu.FP16
    k, v, top = far_below(shift, d, n, every)
    q = np.zeros((1, 1, d))
    q[0, 0, 1] = 1
    q, k, v = codes(q, dtype), codes(k, dtype), codes(v, dtype)
    print(f"far below {attention.__name__} d {d} shift {shift} keys {n}", flush=True)
    got = values(attention(rt, q, k, v, dtype, 1.0), dtype)[0, 0]
    shift = -float(values(k, dtype).min())  # as the type holds it: 10.4 is 10.3984375
    low, high = (n - top.sum()) * np.exp(-shift), top.sum()
    o, u = 1024 * low / (low + high), HALF_STEP[dtype]
    # e: exp2 and its argument; each key's rounding (u, and 2^-32 where e^-shift 2^7
    # is below 2^-14); sums of n terms in FP32; the result's rounding
    e = shift * 2.0 ** -22 + 2.0 ** -19
    size = u + (2.0 ** -32 / np.exp(-shift) if np.exp(-shift) < 2.0 ** -21 else 0.0)
    tol = o * (size + 2 * e + n * 2.0 ** -24 * 2 + u) * (1 + 4 * u) + TINY[dtype]
    assert (np.abs(got - o) <= tol).all(), (got[0], o, tol)
