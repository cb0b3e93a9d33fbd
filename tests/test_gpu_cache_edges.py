"""The paged cache's row operations on numbers that do not fit: what they
leave, what they serve all the same, and what the status says."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, Buffers, attend, check, normal, u32, values
from test_gpu_cache import Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,kv", [(64, 1), (128, 3)])
@pytest.mark.parametrize("what", ["past the pool", "past the table"])
@pytest.mark.parametrize("count", [5, 20])
def test_keep_reports_missing_pages_of_nodes_that_stay(rt, d, kv, what, count):
    """Kept nodes that are in their place already need no copy, but a page of
    theirs that does not exist sets the status as for any other row. A missing
    page of nodes that are not kept, or behind the sequence, does not."""
    page, rows, context = 16, count + 20, 14
    with Buffers(rt) as b:
        pool = Pool(rt, b, 5, kv, d, page)
        missing = [0, pool.n_pages, 2, 3]
        pitch = 4 if what == "past the pool" else 1
        tables = u32([missing[:pitch]])
        batch = xpu.Batch(1, rows, pitch, b.up(tables), b.up(u32([0, rows])), b.up(u32([context])))
        kept = b.up(u32(range(rows)))
        print(f"keep d {d} kv {kv} {what} count {count}", flush=True)
        for n, status in ((0, 0), (2, 0), (count, 1)):
            new = b.up(u32([GUARD]))
            rt.cache_keep(pool.cache, batch, kept, b.up(u32([n])), new)
            pool.verify(status=status)
            assert list(rt.download(new, 1, np.uint32)) == [context + n]


BAD_STARTS = [  # starts, rows, the sequences that have rows
    ([0, 50, 10, 20], 20, [2]),               # passes the rows; back; fine
    ([0, 0xFFFFFFFF, 10, 20], 20, [2]),
    ([4, 2, 8, 99, 8, 12], 14, [1, 4]),
    ([0, 3, 200, 300, 3, 9], 9, [0, 4]),
    ([12, 16, 0, 5], 16, [0, 2]),             # in another order than the rows
    ([0, 2] + [1000] * 70 + [2, 7], 9, [0, 72])]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("starts,rows,served", BAD_STARTS)
def test_append_serves_the_sequences_whose_starts_fit(rt, d, starts, rows, served):
    """A sequence whose starts descend or pass the rows has none; rows that one
    other sequence has are that one's all the same, for the attention too."""
    kv, page, n = 2, 16, len(starts) - 1
    with Buffers(rt) as b:
        pool = Pool(rt, b, 2 * n, kv, d, page, 1)
        tables = u32([[2 * s, 2 * s + 1] for s in range(n)])
        contexts = [14 + s % 3 for s in range(n)]
        k, v = normal((rows, kv, d), 5, pool.dtype), normal((rows, kv, d), 6, pool.dtype)
        batch = xpu.Batch(n, rows, 2, b.up(tables), b.up(u32(starts)), b.up(u32(contexts)))
        print(f"append d {d} starts {starts[:8]}", flush=True)
        rt.cache_append(pool.cache, batch, 0, b.up(k), b.up(v))
        seen = np.full(rows, -1)
        for s in served:
            for i in range(starts[s], starts[s + 1]):
                p, slot = pool.place(tables[s], contexts[s] + i - starts[s])
                pool.k[0, p, :, slot], pool.v[0, p, :, slot] = k[i], v[i]
                seen[i] = s
        pool.verify()
        # the attention serves the same rows: each is the value that its sequence's own scores give
        q, out = normal((rows, kv, d), 7, pool.dtype), b.up(np.full((rows, kv, d), GUARD, np.uint16))
        size = rt.tree_attention_workspace(pool.cache, batch, kv)
        rt.tree_attention(pool.cache, batch, 0, kv, b.up(q), out, b.alloc(size), size)
        rt.synchronize()
        got = rt.download(out, q.size, np.uint16).reshape(q.shape)
        for i, s in enumerate(seen):
            if s < 0:
                assert (got[i] == GUARD).all()
                continue
            at = [pool.place(tables[s], p) for p in range(contexts[s] + i - starts[s] + 1)]
            for h in range(kv):
                keys, vals = (np.array([x[0, p, h, slot] for p, slot in at]) for x in (pool.k, pool.v))
                want, tol = attend(values(q[i:i + 1, h], pool.dtype), values(keys, pool.dtype),
                                   values(vals, pool.dtype), np.ones((1, len(at)), bool), d ** -0.5, pool.dtype)
                check(values(got[i:i + 1, h], pool.dtype), want, tol, f"row {i} head {h}")


def test_append_finds_rows_among_thousands_of_sequences(rt):
    """Sequences of no row or some, a start that passes the rows now and then."""
    rng, d, page = np.random.RandomState(3), 64, 16
    lengths = rng.choice([0, 0, 1, 2, 3], 2500)
    starts = np.concatenate([[5], 5 + np.cumsum(lengths)])
    rows, n = int(starts[-1]) + 2, len(lengths)
    served = np.ones(n, bool)
    for s in rng.choice(np.arange(1, n), 40, replace=False):
        starts[s] = rows + s
        served[[s - 1, s]] = False
    with Buffers(rt) as b:
        pool = Pool(rt, b, n, 1, d, page, 1)
        contexts = rng.randint(0, 14, n)
        k, v = normal((rows, 1, d), 5, pool.dtype), normal((rows, 1, d), 6, pool.dtype)
        order = rng.permutation(n)
        batch = xpu.Batch(n, rows, 1, b.up(u32(order)), b.up(u32(starts)), b.up(u32(contexts)))
        rt.cache_append(pool.cache, batch, 0, b.up(k), b.up(v))
        for s in np.flatnonzero(served):
            for i in range(int(starts[s]), int(starts[s + 1])):
                slot = contexts[s] + i - int(starts[s])
                pool.k[0, order[s], :, slot], pool.v[0, order[s], :, slot] = k[i], v[i]
        pool.verify()


@pytest.mark.parametrize("starts,rows,counts", [
    ([0, 3, 99, 5, 5, 8], 8, [2, 0, 0, 0, 1]), ([4, 2, 6, 6], 6, [0, 3, 0]), ([4, 2, 6, 6], 6, [1, 3, 1]),
    ([0, 0xFFFFFFFF, 0, 2], 2, [0, 0, 2])])
def test_keep_of_sequences_whose_starts_do_not_fit(rt, starts, rows, counts):
    """They have no rows: a count of 0 gives their context as that of a sequence
    whose starts are equal, any other is one that does not fit."""
    n = len(counts)
    with Buffers(rt) as b:
        pool = Pool(rt, b, n, 2, 64, 16, 2)
        contexts = [3 + s for s in range(n)]
        batch = xpu.Batch(n, rows, 1, b.up(u32([[s] for s in range(n)])), b.up(u32(starts)), b.up(u32(contexts)))
        kept = np.zeros(rows, np.uint32)
        want, status = [], 0
        for s, (lo, hi, count) in enumerate(zip(starts, starts[1:], counts)):
            held = hi - lo if lo <= hi <= rows else 0
            if count > held:
                want.append(GUARD)
                status = 1
                continue
            want.append(contexts[s] + count)
            kept[lo:lo + count] = range(held - count, held)
            for pools in (pool.k, pool.v):
                old = pools.copy()
                for j in range(count):
                    pools[:, s, :, contexts[s] + j] = old[:, s, :, contexts[s] + held - count + j]
        new = b.up(u32([GUARD] * n))
        print(f"keep starts {starts} counts {counts}", flush=True)
        rt.cache_keep(pool.cache, batch, b.up(kept), b.up(u32(counts)), new)
        pool.verify(status=status)
        assert list(rt.download(new, n, np.uint32)) == want
