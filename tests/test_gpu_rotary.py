"""xpu_cache_append_rotary on gfx950 against the rotation in 64 bits (the bound
is derived in rotary_util.py): where every row goes, V bit for bit, rotations in
halves and in adjacent pairs, of a part of a head, with and without gains, by
other positions than the cache's, strides, rows of no sequence, rows that have
no place or no position."""
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, Buffers, check, codes, normal, u32, values
from rotary_util import bound, tables, turned
from test_gpu_cache import Pool, tables_of

pytestmark = pytest.mark.gpu
TYPES = [xpu.BF16, xpu.FP16]


class Turn:
    """New rows of a batch over a Pool, and what they should become."""

    def __init__(self, rt, b, rows, contexts, heads, kv, d, page, dtype, dims, adjacent=False, gains=False, first=0,
                 at=None, pad=0, positions=None, in_place=False, seed=5, pool=None, strides=True):
        self.rt, self.rows, self.contexts, self.heads, self.d, self.dtype = rt, rows, contexts, heads, d, dtype
        sizes = [r + c for r, c in zip(rows, contexts)]
        self.pool = pool or Pool(rt, b, sum(-(-s // page) for s in sizes) + 2, kv, d, page, 2, dtype)
        self.tables = tables_of(sizes, page, self.pool.n_pages, random.Random(seed))
        self.starts = u32(np.cumsum([first] + list(rows)))
        self.total = int(self.starts[-1]) + pad
        more = (8, 24, 16, 40) if strides else (0, 0, 0, 0)
        self.strides = [w + m for w, m in zip((kv * d, kv * d, heads * d, heads * d), more)]
        self.k, self.v, self.q = (normal((self.total, s), seed + i, dtype, 1 + i) for i, s in enumerate(self.strides[:3]))
        self.at = [c + i for r, c in zip(rows, contexts) for i in range(r)]
        if at is not None:
            self.at = list(at)
        self.positions = positions or max(self.at + [0]) + 1
        self.cos, self.sin = tables(self.positions, dims)
        self.gains = [codes(1 + 0.3 * np.random.RandomState(seed + i).randn(d), dtype) for i in (7, 8)] if gains else [None, None]
        self.adjacent, self.eps = adjacent, 1e-5
        flat = u32([0] * first + self.at + [0xFFFFFFFF] * pad) if at is not None else None
        up = lambda x: None if x is None else b.up(x)  # noqa: E731
        self.rotary = xpu.Rotary(self.positions, dims, b.up(self.cos), b.up(self.sin),
                                 xpu.ADJACENT if adjacent else xpu.HALVES, up(flat), up(self.gains[0]), up(self.gains[1]),
                                 self.eps)
        self.batch = xpu.Batch(len(rows), self.total, self.tables.shape[1], b.up(self.tables), b.up(self.starts),
                               b.up(u32(contexts)))
        self.dk, self.dv, self.dq = b.up(self.k), b.up(self.v, pad=16), b.up(self.q)
        self.out = np.full((self.total, self.strides[3]), GUARD, np.uint16)
        self.dout = b.up(self.out)
        if in_place:
            self.dout, self.out, self.strides[3] = self.dq, self.q.copy(), self.strides[2]

    def call(self, append=None):
        print(f"rows {self.rows[:6]} contexts {self.contexts[:6]} heads {self.heads} kv {self.pool.kv} d {self.d} page "
              f"{self.pool.page} dtype {self.dtype} dims {self.rotary.dims} pairs {self.rotary.pairs}", flush=True)
        ks, vs, qs, outs = self.strides
        (append or self.rt.cache_append_rotary)(
            self.pool.cache, self.batch, 1, self.dk, self.dv, rotary=self.rotary, heads=self.heads,
            q=self.dq if self.heads else None, q_out=self.dout if self.heads else None, k_stride=ks, v_stride=vs,
            q_stride=qs, out_stride=outs)
        self.rt.synchronize()

    def rows_of(self, x, heads):
        """The batch's rows in order, [rows, heads, d]."""
        a, n = int(self.starts[0]), sum(self.rows)
        return x[a: a + n, : heads * self.d].reshape(n, heads, self.d)

    def want(self, x, heads, gain):
        y, size = turned(values(self.rows_of(x, heads), self.dtype), self.at, self.cos, self.sin, self.adjacent,
                         None if gain is None else values(gain, self.dtype), self.eps)
        return y, size

    def check_q(self):
        got = self.rt.download(self.dout, self.out.size, np.uint16).reshape(self.out.shape)
        if self.heads:
            y, size = self.want(self.q, self.heads, self.gains[0])
            check(values(self.rows_of(got, self.heads), self.dtype), y, bound(y, size, self.dtype), "q")
        left = got.copy()
        a = int(self.starts[0])
        left[a: a + sum(self.rows), : self.heads * self.d] = self.out[a: a + sum(self.rows), : self.heads * self.d]
        assert np.array_equal(left, self.out)  # the rest is as it was

    def check_pool(self):
        kv, pool = self.pool.kv, self.pool
        y, size = self.want(self.k, kv, self.gains[1])
        got = self.rt.download(pool.dk, pool.k.size, np.uint16).reshape(pool.k.shape)
        i = 0
        for s, (r, c) in enumerate(zip(self.rows, self.contexts)):
            for j in range(r):
                p, slot = pool.place(self.tables[s], c + j)
                check(values(got[1, p, :, slot], self.dtype), y[i], bound(y[i], size[i], self.dtype), f"k row {i}")
                pool.k[1, p, :, slot] = got[1, p, :, slot]
                pool.v[1, p, :, slot] = self.rows_of(self.v, kv)[i]
                i += 1
        pool.verify()


ROWS = [([1], [0], 0), ([1, 1, 1], [15, 16, 200], 0), ([0, 40, 0, 1, 130], [5, 60, 9, 0, 255], 2), ([1] * 70, [7] * 70, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kv,page", [(64, 4, 1, 16), (64, 3, 3, 64), (128, 16, 8, 16), (128, 5, 5, 256)])
@pytest.mark.parametrize("rows,contexts,first", ROWS)
def test_append_rotary(rt, dtype, d, heads, kv, page, rows, contexts, first):
    with Buffers(rt) as b:
        t = Turn(rt, b, rows, contexts, heads, kv, d, page, dtype, d, gains=True, first=first, pad=3)
        t.call()
        t.check_q()
        t.check_pool()


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("gains", [False, True])
@pytest.mark.parametrize("d,dims", [(64, 16), (64, 48), (64, 64), (128, 32), (128, 80), (128, 112), (128, 128)])
def test_parts_of_a_head(rt, d, dims, adjacent, gains):
    with Buffers(rt) as b:
        t = Turn(rt, b, [5, 1, 19], [3, 40, 0], 6, 2, d, 16, xpu.FP16, dims, adjacent, gains)
        t.call()
        t.check_q()
        t.check_pool()


@pytest.mark.parametrize("heads,in_place", [(0, False), (7, True), (64, False)])
def test_without_queries_and_in_place(rt, heads, in_place):
    with Buffers(rt) as b:
        t = Turn(rt, b, [3, 20], [10, 0], heads, 2, 64, 32, xpu.BF16, 64, gains=True, in_place=in_place)
        t.call()
        t.check_q()
        t.check_pool()


def test_positions_of_a_tree(rt):
    """Nodes are turned by their depth, stored where they come."""
    with Buffers(rt) as b:
        t = Turn(rt, b, [6, 3], [30, 7], 4, 2, 128, 16, xpu.BF16, 128, first=1, pad=2, at=[30, 31, 31, 32, 32, 31, 7, 8, 8],
                 positions=40)
        t.call()
        t.check_q()
        t.check_pool()


def test_columns_of_one_buffer(rt):
    """Q, K and V as a projection leaves them, Q turned in place."""
    heads, kv, d, n = 4, 2, 64, 9
    with Buffers(rt) as b:
        t = Turn(rt, b, [n], [20], heads, kv, d, 16, xpu.BF16, d, gains=True, strides=False)
        width = (heads + 2 * kv) * d
        buffer = np.concatenate([t.q, t.k, t.v], 1)
        ptr = b.up(buffer)
        t.dq = t.dout = ptr
        t.dk, t.dv = ptr + 2 * heads * d, ptr + 2 * (heads + kv) * d
        t.strides = [width] * 4
        t.call()
        got = rt.download(ptr, buffer.size, np.uint16).reshape(buffer.shape)
        assert np.array_equal(got[:, heads * d:], buffer[:, heads * d:])
        y, size = t.want(t.q, heads, t.gains[0])
        check(values(got[:, : heads * d].reshape(n, heads, d), t.dtype), y, bound(y, size, t.dtype))
        t.check_pool()


def test_rows_without_a_place_or_a_position(rt):
    """A page past the pool: Q is turned all the same. A position past the
    tables: NaN, and nothing is written. Starts that do not fit: left alone."""
    with Buffers(rt) as b:
        t = Turn(rt, b, [4, 4], [14, 2], 2, 2, 64, 16, xpu.BF16, 64)
        tables_ = t.tables.copy()
        tables_[0, 1] = t.pool.n_pages
        rt.copy_to(t.batch.tables, tables_)
        short = xpu.Rotary(17, 64, t.rotary.cos, t.rotary.sin)
        t.rotary, t.positions = short, 17
        t.call()
        got = rt.download(t.dout, t.out.size, np.uint16).reshape(t.out.shape)
        y, size = t.want(t.q, 2, None)
        rows = values(t.rows_of(got, 2), t.dtype)
        assert np.isnan(rows[3]).all()  # position 17
        check(rows[[0, 1, 2, 4, 5, 6, 7]], y[[0, 1, 2, 4, 5, 6, 7]], bound(y, size, t.dtype)[[0, 1, 2, 4, 5, 6, 7]])
        new = rt.download(t.pool.dk, t.pool.k.size, np.uint16).reshape(t.pool.k.shape)
        yk, sk = t.want(t.k, 2, None)
        for i, s, pos in [(0, 0, 14), (1, 0, 15), (4, 1, 2), (5, 1, 3), (6, 1, 4), (7, 1, 5)]:
            p, slot = t.pool.place(tables_[s], pos)
            check(values(new[1, p, :, slot], t.dtype), yk[i], bound(yk[i], sk[i], t.dtype))
            t.pool.k[1, p, :, slot], t.pool.v[1, p, :, slot] = new[1, p, :, slot], t.rows_of(t.v, 2)[i]
        t.pool.verify(status=1)
        rt.copy_to(t.dout, t.out)
        for starts in ([0, 0xFFFFFFF0, 8], [9, 3, 1]):
            t.batch.starts = b.up(u32(starts))
            t.call()
        assert np.array_equal(rt.download(t.dout, t.out.size, np.uint16).reshape(t.out.shape), t.out)
        t.pool.verify(status=1)


def test_many_sequences(rt):
    """More than 64, some without rows."""
    rows = [i % 3 for i in range(200)]
    with Buffers(rt) as b:
        t = Turn(rt, b, rows, [i % 37 for i in range(200)], 2, 1, 64, 16, xpu.FP16, 64, first=1, pad=1)
        t.call()
        t.check_q()
        t.check_pool()


def test_values_that_are_not_finite(rt):
    """A NaN or an infinity stays within its pair, or with gains within its head."""
    with Buffers(rt) as b:
        t = Turn(rt, b, [3], [5], 2, 1, 64, 16, xpu.BF16, 64, strides=False)
        t.q[0, 3], t.q[1, 64 + 40] = 0x7FC0, 0x7F80
        rt.copy_to(t.dq, t.q)
        t.call()
        got = values(t.rows_of(rt.download(t.dout, t.out.size, np.uint16).reshape(t.out.shape), 2), t.dtype)
        odd = np.zeros(got.shape, bool)
        odd[0, 0, [3, 35]] = odd[1, 1, [8, 40]] = True
        assert (~np.isfinite(got) == odd).all()
