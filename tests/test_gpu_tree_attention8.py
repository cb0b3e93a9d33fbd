"""xpu_tree_attention8 on gfx950 against attention in 64 bits over what the
codes and scales stand for (the bound is derived in cache_util.py): trees,
chains and single tokens, contexts that end inside a block or a tile, cut into
chunks or not, windows of many pages, what unseen positions hold, wrong pages
and lengths, strides."""
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache8_util import BLOCK, Pool8, codes8
from cache_util import GUARD, Buffers, attend, check, normal, u32, values
from test_gpu_tree_attention import tree_masks

pytestmark = pytest.mark.gpu
TYPES = [xpu.BF16, xpu.FP16]
NAN8 = 0x7F


class Case8:
    """Sequences over pages in random order. Positions behind a sequence's end,
    and pages of no sequence, hold NaN with any scale."""

    def __init__(self, rt, b, nodes, contexts, heads, kv, d, page, dtype, seed, masked=True, first=0, spare=3, empty=False,
                 spread=3):
        rng = random.Random(seed)
        self.rt, self.nodes, self.contexts, self.heads, self.kv, self.d, self.dtype = rt, nodes, contexts, heads, kv, d, dtype
        ends = [n + c for n, c in zip(nodes, contexts)]
        held = [-(-e // page) for e in ends]
        ids = list(range(sum(held) + spare))
        rng.shuffle(ids)
        self.pool = pool = Pool8(rt, b, len(ids), kv, d, page, 2, dtype, seed)
        self.pitch = max(max(held), 1) + 1
        self.tables = np.full((len(nodes), self.pitch), 0xFFFFFFFF, np.uint32)  # not looked at past the end
        self.starts = u32(np.cumsum([first] + list(nodes)))
        self.rows = int(self.starts[-1]) + spare
        r, at = np.random.RandomState(seed + 1), 0
        for n in "kv":
            pool.codes[n][:] = NAN8
            pool.scales[n][:] = r.randint(0, 256, pool.scales[n].shape)
        for s, (e, m) in enumerate(zip(ends, held)):
            self.tables[s, :m] = ids[at: at + m]
            at += m
            for n in "kv":
                for p in range(0, e, BLOCK):
                    id, slot = pool.place(self.tables[s], p)
                    rows = min(BLOCK, e - p)
                    pool.codes[n][1, id, :, slot: slot + rows] = codes8(np.clip(r.randn(kv, rows, d) * 100, -440, 440))
                    pool.scales[n][1, id, :, slot // BLOCK] = 127 - 7 + r.randint(-spread, 2, kv)
        self.q = normal((self.rows, heads, d), seed + 1, dtype)
        self.masks = [tree_masks(n, rng, empty) for n in nodes] if masked else None
        self.out = np.full(self.q.shape, GUARD, np.uint16)
        self.b = b

    def seen(self, s):
        n, c = self.nodes[s], self.contexts[s]
        seen = np.ones((n, n + c), bool)
        for i in range(n):
            for j in range(n):
                seen[i, c + j] = j <= i if self.masks is None else self.masks[s][i] >> j & 1
        return seen

    def expected(self, scale, only=None):
        want, tol = values(self.out, self.dtype).copy(), np.zeros(self.out.shape)
        q, group = values(self.q, self.dtype), self.heads // self.kv
        for s, n in enumerate(self.nodes):
            if only is not None and s not in only:
                continue
            a, seen, at = int(self.starts[s]), self.seen(s), list(range(n + self.contexts[s]))
            for h in range(self.kv):
                k, v = (self.pool.read(m, 1, self.tables[s], at, h) for m in "kv")
                for i in range(h * group, (h + 1) * group):
                    want[a:a + n, i], tol[a:a + n, i] = attend(q[a:a + n, i], k, v, seen, scale, self.dtype, 64)
        return want, tol

    def run(self, scale=None, **over):
        pool, b, rt = self.pool, self.b, self.rt
        print(f"tree attention 8 nodes {self.nodes[:8]} contexts {self.contexts[:8]} heads {self.heads}/{self.kv} d {self.d} "
              f"page {pool.page} dtype {self.dtype} masked {self.masks is not None}", flush=True)
        for n in "kv":
            rt.copy_to(pool.ptr[n], pool.raw(n))
        batch = xpu.Batch(len(self.nodes), self.rows, self.pitch, b.up(self.tables), b.up(self.starts), b.up(u32(self.contexts)))
        vis = None
        if self.masks is not None:  # the bits past a sequence's nodes are not looked at
            flat = [(m | ~((1 << n) - 1)) & (1 << 64) - 1 for n, ms in zip(self.nodes, self.masks) for m in ms]
            first = int(self.starts[0])
            vis = b.up(np.array([0] * first + flat + [0] * (self.rows - first - len(flat)), np.uint64))
        size = rt.tree_attention8_workspace(pool.cache, batch, self.heads)
        out = b.up(self.out)
        rt.tree_attention8(pool.cache, batch, 1, self.heads, b.up(self.q), out, b.alloc(size), size, visible=vis, scale=scale)
        rt.synchronize()
        got = rt.download(out, self.out.size, np.uint16).reshape(self.out.shape)
        return got, int(rt.download(pool.status, 1, np.uint32)[0])

    def verify(self, scale=None):
        got, status = self.run(scale)
        want, tol = self.expected(self.d ** -0.5 if scale is None else scale)
        check(values(got, self.dtype), want, tol)
        assert status == 0
        return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kv,page", [(64, 2, 1, 16), (64, 6, 2, 64), (128, 8, 8, 16), (128, 8, 2, 32)])
@pytest.mark.parametrize("nodes,contexts", [([1], [0]), ([1], [37]), ([3, 0, 17, 64], [16, 5, 31, 0]), ([64], [200]),
                                            ([1, 2, 5, 9, 12], [15, 32, 100, 63, 1])])
@pytest.mark.parametrize("masked", [True, False])
def test_tree_attention8(rt, dtype, d, heads, kv, page, nodes, contexts, masked):
    with Buffers(rt) as b:
        Case8(rt, b, nodes, contexts, heads, kv, d, page, dtype, 3, masked, first=2, empty=masked).verify()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kv,page,nodes,contexts", [
    (128, 4, 1, 16, [1], [9000]), (128, 2, 2, 256, [30, 1], [5000, 3]), (64, 2, 1, 16, [64, 2], [4099, 8000]),
    (64, 8, 1, 32, [7], [20011])])
def test_long_contexts(rt, dtype, d, heads, kv, page, nodes, contexts):
    """Cut into chunks, and walked in several windows of 64 blocks by a wavefront."""
    with Buffers(rt) as b:
        Case8(rt, b, nodes, contexts, heads, kv, d, page, dtype, 4).verify()


def test_many_kv_heads_walk_many_windows(rt):
    """So many kv heads that the keys are not cut: 33 tiles and more to a wavefront."""
    with Buffers(rt) as b:
        Case8(rt, b, [2] * 3, [5003, 4300, 130], 256, 256, 64, 16, xpu.BF16, 5, spare=0).verify()


def test_many_sequences(rt):
    nodes, contexts = [i % 4 for i in range(130)], [(i * 37) % 150 for i in range(130)]
    with Buffers(rt) as b:
        Case8(rt, b, nodes, contexts, 4, 2, 64, 16, xpu.FP16, 6, first=1).verify()


def test_chains_of_many_rows(rt):
    """A further part of a prompt."""
    with Buffers(rt) as b:
        Case8(rt, b, [150, 1, 70], [33, 10, 0], 4, 2, 64, 16, xpu.BF16, 7, masked=False).verify()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [40, 70])
def test_scales_far_apart(rt, dtype, spread):
    """Blocks from 2^-spread of the others' size, far below the type's normal range in fp16."""
    with Buffers(rt) as b:
        Case8(rt, b, [5, 9], [60, 130], 4, 2, 128, 16, dtype, 8, spread=spread).verify()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_unseen_nodes_hold(rt, dtype):
    """NaN in K and V of nodes that rows do not see: those rows keep every bit."""
    with Buffers(rt) as b:
        c = Case8(rt, b, [6, 20], [40, 13], 4, 2, 64, 16, dtype, 9)
        c.masks = [[1 << i for i in range(n)] for n in c.nodes]
        c.masks[0][5] |= 1 << 2
        clean = c.verify()
        for s, node, heads in ((0, 2, (0, 1)), (1, 17, (1,))):
            p, slot = c.pool.place(c.tables[s], c.contexts[s] + node)
            for n in "kv":
                for h in heads:
                    c.pool.codes[n][1, p, h, slot, 3::7] = NAN8
        got, _ = c.run()
        rows = values(got, dtype)
        a0, a1 = int(c.starts[0]), int(c.starts[1])
        for i in range(c.rows):
            sees0, sees1 = i in (a0 + 2, a0 + 5), i == a1 + 17
            for h in range(4):
                if sees0 or (sees1 and h >= 2):
                    assert np.isnan(rows[i, h]).any(), (i, h)
                else:
                    assert np.array_equal(got[i, h], clean[i, h]), (i, h)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_infinite_in_the_type(rt, dtype):
    """A block's scale at which its largest codes pass the type's range: unseen
    they do not matter, seen they are infinite."""
    with Buffers(rt) as b:
        c = Case8(rt, b, [18], [32], 2, 1, 64, 16, dtype, 10)
        c.masks = [[1 << i for i in range(18)]]
        p, slot = c.pool.place(c.tables[0], 48)
        c.pool.codes["v"][1, p, 0, slot: slot + 2] = 0x08  # 2^-6
        c.pool.codes["v"][1, p, 0, slot, 5] = 0x7E         # 448
        c.pool.scales["v"][1, p, 0, 0] = 247 if dtype == xpu.BF16 else 127 + 8
        c.pool.scales["k"][1, p, 0, 0] = 120
        c.masks[0][17] |= 1 << 16
        got, _ = c.run()
        rows = values(got, dtype)[int(c.starts[0]):]
        assert np.isfinite(rows[:16]).all()
        assert np.isinf(rows[16:18, :, 5]).all()
        others = np.delete(rows[16:18], 5, axis=2)
        assert np.isfinite(others).all()


def test_rows_that_see_nothing(rt):
    with Buffers(rt) as b:
        c = Case8(rt, b, [3, 1], [0, 0], 2, 1, 64, 16, xpu.BF16, 11)
        c.masks = [[0, 1, 0], [0]]
        got = c.verify()
        assert (got[[0, 2, 3]] == 0).all()


def test_wrong_pages_and_lengths(rt):
    """A page past the pool, a context past the table, more than 64 nodes: those
    rows are NaN, the others right, and the status says so."""
    with Buffers(rt) as b:
        for wrong in ("page", "context", "nodes"):
            c = Case8(rt, b, [3, 2, 65 if wrong == "nodes" else 4], [50, 40, 20], 4, 2, 64, 16, xpu.BF16, 12)
            want, tol = c.expected(64 ** -0.5, only=(0, 1) if wrong == "nodes" else (0, 2))
            bad = 2 if wrong == "nodes" else 1
            if wrong == "page":
                c.tables[1, 1] = c.pool.n_pages
            if wrong == "context":
                c.contexts[1] = 0xFFFFFFFF
            got, status = c.run()
            a, e = int(c.starts[bad]), int(c.starts[bad + 1])
            want[a:e], tol[a:e] = np.nan, 0
            assert status == 1
            check(values(got, c.dtype), want, tol, wrong)


def test_strides_and_layers(rt):
    """q and out as columns of one buffer."""
    with Buffers(rt) as b:
        c = Case8(rt, b, [4, 7], [100, 3], 4, 2, 64, 16, xpu.FP16, 13)
        want, tol = c.expected(64 ** -0.5)
        width = 4 * 64
        buffer = np.full((c.rows, 2 * width + 8), GUARD, np.uint16)
        buffer[:, :width] = c.q.reshape(c.rows, width)
        ptr = b.up(buffer)
        for n in "kv":
            rt.copy_to(c.pool.ptr[n], c.pool.raw(n))
        batch = xpu.Batch(2, c.rows, c.pitch, b.up(c.tables), b.up(c.starts), b.up(u32(c.contexts)))
        vis = b.up(np.array([m for ms in c.masks for m in ms] + [0] * 3, np.uint64))
        size = rt.tree_attention8_workspace(c.pool.cache, batch, 4)
        rt.tree_attention8(c.pool.cache, batch, 1, 4, ptr, ptr + 2 * width, b.alloc(size), size, visible=vis,
                           q_stride=2 * width + 8, out_stride=2 * width + 8)
        rt.synchronize()
        got = rt.download(ptr, buffer.size, np.uint16).reshape(buffer.shape)
        assert np.array_equal(got[:, :width], buffer[:, :width]) and (got[:, 2 * width:] == GUARD).all()
        check(values(got[:, width: 2 * width].reshape(c.rows, 4, 64), c.dtype), want, tol)
