"""Calls of the 8-bit cache and of the rotated appends that are more work than
the GPU has wavefronts for at once: in one call as in several."""
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache8_util import Pool8
from cache_util import Buffers, u32
from rotary_util import tables
from test_gpu_cache import tables_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
def test_keep_of_many_drafts(rt, d):
    """Drafts of few and of many kept nodes, one after another."""
    rng = random.Random(4)
    rows = [rng.choice([1, 9, 16, 17, 40, 64]) for _ in range(230)]
    contexts = [rng.randrange(70) for _ in rows]
    kept = [[rng.randrange(n) for _ in range(rng.choice([0, 1, n // 2, n]))] for n in rows]
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool8(rt, b, sum(-(-s // 32) for s in sizes) + 1, 3, d, 32, 2)
        table, starts = tables_of(sizes, 32, pool.n_pages, rng), u32(np.cumsum([0] + rows))
        batch = xpu.Batch(len(rows), int(starts[-1]), table.shape[1], b.up(table), b.up(starts), b.up(u32(contexts)))
        flat = u32([i for r, ids in zip(rows, kept) for i in ids + [0xFFFFFFFF] * (r - len(ids))])
        new = b.up(u32([0] * len(rows)))
        print(f"keep8 of {len(rows)} drafts d {d}", flush=True)
        rt.cache8_keep(pool.cache, batch, b.up(flat), b.up(u32([len(ids) for ids in kept])), new)
        for s, ids in enumerate(kept):
            pool.keep(table[s], contexts[s], ids, rows[s])
        pool.verify()
        assert list(rt.download(new, len(rows), np.uint32)) == [c + len(ids) for c, ids in zip(contexts, kept)]


@pytest.mark.parametrize("eight", [False, True])
def test_a_long_prompt_in_pieces(rt, eight):
    n, piece, heads, kv, d, page, dtype = 70000, 8000, 1, 8, 64, 256, xpu.BF16
    pages = -(-n // page)
    rng = np.random.RandomState(6)

    def rows(width):  # exponents of 2^-3 .. 2^3, any sign and digits
        return (rng.randint(124, 130, (n, width)) << 7 | rng.randint(0, 128, (n, width)) |
                rng.randint(0, 2, (n, width)) << 15).astype(np.uint16)

    cos, sin = tables(n, d)
    with Buffers(rt) as b:
        k, v, q = b.up(rows(kv * d)), b.up(rows(kv * d)), b.up(rows(heads * d))
        table = b.up(u32(rng.permutation(pages)))
        rotary = xpu.Rotary(n, d, b.up(cos), b.up(sin))
        size = kv * page * d * 2
        if eight:
            size = -(-(kv * page * d + kv * page // 16) // 128) * 128
        got = []
        for pieces in ([n], [piece] * (n // piece) + [n % piece]):
            pool = [b.up(np.zeros(pages * size, np.uint8)) for _ in "kv"]
            out = b.up(np.zeros((n, heads * d), np.uint16))
            cache = (xpu.Cache8 if eight else xpu.Cache)(dtype, 1, kv, d, page, pages, *pool)
            at = 0
            for count in pieces:
                print(f"append eight {eight} rows {at} .. {at + count}", flush=True)
                batch = xpu.Batch(1, count, pages, table, b.up(u32([0, count])), b.up(u32([at])))
                (rt.cache8_append if eight else rt.cache_append_rotary)(
                    cache, batch, 0, k + at * kv * d * 2, v + at * kv * d * 2, rotary=rotary, heads=heads,
                    q=q + at * heads * d * 2, q_out=out + at * heads * d * 2)
                at += count
            rt.synchronize()
            got.append([rt.download(p, pages * size, np.uint8) for p in pool] + [rt.download(out, n * heads * d, np.uint16)])
        for one, several in zip(*got):
            assert one.any() and np.array_equal(one, several)
