"""The paged cache on gfx950: rows appended, drafts kept and pages copied bit
for bit, and a serving loop of all the operators together against attention in
64 bits over what each sequence holds."""
import ctypes
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, Buffers, attend, check, normal, u32, values
from xpu_playground_amd.cache import Pages, renumber

pytestmark = pytest.mark.gpu


class Pool:
    """A cache on the device and what it should hold."""

    def __init__(self, rt, b, n_pages, kv=2, d=64, page=16, layers=3, dtype=xpu.BF16, seed=1):
        self.rt, self.kv, self.d, self.page, self.layers, self.n_pages, self.dtype = rt, kv, d, page, layers, n_pages, dtype
        shape = (layers, n_pages, kv, page, d)
        self.k, self.v = normal(shape, seed, dtype), normal(shape, seed + 1, dtype)
        self.dk, self.dv, self.status = b.up(self.k), b.up(self.v), b.up(u32([0]))
        self.cache = xpu.Cache(dtype, layers, kv, d, page, n_pages, self.dk, self.dv, self.status)

    def verify(self, status=0):
        self.rt.synchronize()
        for ptr, want in ((self.dk, self.k), (self.dv, self.v)):
            got = self.rt.download(ptr, want.size, np.uint16).reshape(want.shape)
            bad = np.argwhere(got != want)
            assert not len(bad), f"{len(bad)} elements differ, first {bad[0]}"
        assert int(self.rt.download(self.status, 1, np.uint32)[0]) == status

    def place(self, table, pos):
        return int(table[pos // self.page]), pos % self.page


def tables_of(sizes, page, n_pages, rng, pitch=None):
    ids = list(range(n_pages))
    rng.shuffle(ids)
    held, out, at = [-(-s // page) for s in sizes], [], 0
    pitch = pitch or max(held) + 1
    for h in held:
        out.append(ids[at: at + h] + [0xFFFFFFFF] * (pitch - h))
        at += h
    assert at <= n_pages
    return u32(out)


@pytest.mark.parametrize("d,kv", [(64, 1), (64, 2), (64, 5), (128, 8), (128, 3)])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("rows,contexts,first", [
    ([1], [0], 0), ([1, 1, 1], [15, 16, 17], 0), ([0, 40, 0, 1, 300], [5, 60, 9, 0, 255], 2), ([1] * 70, [7] * 70, 0)])
def test_append(rt, d, kv, page, rows, contexts, first):
    rng = random.Random(1)
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool(rt, b, sum(-(-s // page) for s in sizes) + 2, kv, d, page)
        tables, starts = tables_of(sizes, page, pool.n_pages, rng), u32(np.cumsum([first] + rows))
        total = int(starts[-1]) + 3
        ks, vs = kv * d + 8, kv * d + 24
        k, v = normal((total, ks), 5, pool.dtype), normal((total, vs), 6, pool.dtype)
        batch = xpu.Batch(len(rows), total, tables.shape[1], b.up(tables), b.up(starts), b.up(u32(contexts)))
        print(f"append d {d} kv {kv} page {page} rows {rows[:6]} contexts {contexts[:6]}", flush=True)
        rt.cache_append(pool.cache, batch, 1, b.up(k), b.up(v, pad=16), ks, vs)
        for s, (r, c) in enumerate(zip(rows, contexts)):
            for i in range(r):
                p, slot = pool.place(tables[s], c + i)
                pool.k[1, p, :, slot] = k[starts[s] + i, : kv * d].reshape(kv, d)
                pool.v[1, p, :, slot] = v[starts[s] + i, : kv * d].reshape(kv, d)
        pool.verify()


def test_append_leaves_what_it_cannot_place(rt):
    """A page past the pool, positions past the table, starts that do not fit:
    those rows are dropped and the status says so."""
    with Buffers(rt) as b:
        pool = Pool(rt, b, 4)
        k, v = normal((12, 128), 5, pool.dtype), normal((12, 128), 6, pool.dtype)
        tables = u32([[0, 4], [1, 2]])
        batch = xpu.Batch(2, 12, 2, b.up(tables), b.up(u32([0, 4, 8])), b.up(u32([14, 30])))
        rt.cache_append(pool.cache, batch, 0, b.up(k), b.up(v))
        for s, i, p, slot in [(0, 0, 0, 14), (0, 1, 0, 15), (1, 4, 2, 14), (1, 5, 2, 15)]:
            pool.k[0, p, :, slot], pool.v[0, p, :, slot] = k[i].reshape(2, 64), v[i].reshape(2, 64)
        pool.verify(status=1)
        for starts, context in ([0, 0xFFFFFFF0, 8], [0, 0]), ([6, 3, 1], [0, 0]), ([0, 0, 4], [0, 0xFFFFFFFE]):
            batch = xpu.Batch(2, 12, 2, b.up(tables), b.up(u32(starts)), b.up(u32(context)))
            rt.cache_append(pool.cache, batch, 0, b.up(k), b.up(v))
        pool.verify(status=1)


@pytest.mark.parametrize("d,kv", [(64, 1), (64, 3), (128, 2)])
@pytest.mark.parametrize("page", [16, 32])
def test_keep(rt, d, kv, page):
    """Paths, repeats, reversals and nothing at all, across page ends."""
    rng = random.Random(2)
    rows = [1, 5, 64, 0, 26, 64, 7, 33]
    contexts = [0, 14, 31, 9, 100, 3, 16, 60]
    kept = [[0], [1, 3, 4], list(range(63, -1, -1)), [], [0, 0, 25, 25, 3], sorted(rng.sample(range(64), 40)), [],
            [rng.randrange(33) for _ in range(33)]]
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool(rt, b, sum(-(-s // page) for s in sizes) + 1, kv, d, page)
        tables, starts = tables_of(sizes, page, pool.n_pages, rng), u32(np.cumsum([0] + rows))
        batch = xpu.Batch(len(rows), int(starts[-1]), tables.shape[1], b.up(tables), b.up(starts), b.up(u32(contexts)))
        flat = u32([i for r, ids in zip(rows, kept) for i in ids + [0xFFFFFFFF] * (r - len(ids))])
        new = b.up(u32([GUARD] * len(rows)))
        print(f"keep d {d} kv {kv} page {page}", flush=True)
        rt.cache_keep(pool.cache, batch, b.up(flat), b.up(u32([len(ids) for ids in kept])), new)
        for pools in (pool.k, pool.v):
            for s, ids in enumerate(kept):
                old = [pools[:, pool.place(tables[s], contexts[s] + i)[0], :, pool.place(tables[s], contexts[s] + i)[1]].copy()
                       for i in ids]
                for j, row in enumerate(old):
                    p, slot = pool.place(tables[s], contexts[s] + j)
                    pools[:, p, :, slot] = row
        pool.verify()
        assert list(rt.download(new, len(rows), np.uint32)) == [c + len(ids) for c, ids in zip(contexts, kept)]


def test_keep_leaves_what_does_not_fit(rt):
    """Counts past the rows or past 64, nodes that do not exist, a page past
    the pool: left alone, and the status says so."""
    with Buffers(rt) as b:
        pool = Pool(rt, b, 9, kv=1)
        tables = u32([[0, 1, 9, 9, 9, 9], [2, 9, 9, 9, 9, 9], [3, 4, 5, 6, 7, 9]])
        starts, contexts = [0, 4, 8, 80], [0, 14, 0]
        batch = xpu.Batch(3, 80, 6, b.up(tables), b.up(u32(starts)), b.up(u32(contexts)))
        kept = np.zeros(80, np.uint32)
        kept[:4] = [3, 4, 0xFFFFFFFF, 0]
        kept[4:8] = [1, 3, 1, 1]
        new = b.up(u32([GUARD] * 3))
        rt.cache_keep(pool.cache, batch, b.up(kept), b.up(u32([4, 2, 65])), new)
        for pools in (pool.k, pool.v):
            old = pools.copy()
            pools[:, 0, :, 0], pools[:, 0, :, 3] = old[:, 0, :, 3], old[:, 0, :, 0]
            pools[:, 2, :, 14] = old[:, 2, :, 15]  # node 3 of the second would come from page 9
        pool.verify(status=1)
        assert list(rt.download(new, 3, np.uint32)) == [4, 16, GUARD]
        rt.cache_keep(pool.cache, batch, b.up(kept), b.up(u32([5, 5, 0xFFFFFFFF])), new)
        pool.verify(status=1)


def test_keep_without_rows_gives_the_contexts(rt):
    with Buffers(rt) as b:
        pool, n = Pool(rt, b, 2), 70
        batch = xpu.Batch(n, 0, 1, b.up(u32([0] * n)), b.up(u32([0] * (n + 1))), b.up(u32(range(n))))
        new = b.up(u32([GUARD] * n))
        rt.cache_keep(pool.cache, batch, None, b.up(u32([0] * n)), new)
        pool.verify()
        assert list(rt.download(new, n, np.uint32)) == list(range(n))


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
def test_decode_steps_as_two_graphs(rt, dtype):
    """Append, attention and the step to the next context captured together:
    two graphs that hand the contexts to and fro, replayed with eager work
    between, over a padded batch."""
    kv, heads, d, page, n, pad = 2, 8, 128, 16, 3, 2
    contexts, steps = [14, 300, 0], 6
    rng = random.Random(8)
    with Buffers(rt) as b:
        sizes = [c + steps for c in contexts]
        pool = Pool(rt, b, sum(-(-s // page) for s in sizes) + 1, kv, d, page, 1, dtype)
        tables = tables_of(sizes, page, pool.n_pages, rng)
        dt, starts = b.up(tables), b.up(u32([0, 1, 2, 3]))
        both = [b.up(u32(contexts)), b.up(u32([GUARD] * n))]
        rows = [np.full((n + pad, h, d), GUARD, np.uint16) for h in (heads, kv, kv)]
        dq, dk, dv = (b.up(r) for r in rows)
        out, kept, counts = b.up(rows[0]), b.up(u32([0] * (n + pad))), b.up(u32([1] * n))
        batches = [xpu.Batch(n, n + pad, tables.shape[1], dt, starts, c) for c in both]
        size = rt.tree_attention_workspace(pool.cache, batches[0], heads)
        workspace, graphs = b.alloc(size), []
        for i in range(2):
            xpu.check(rt.lib.xpu_rt_capture_begin(rt.handle))
            rt.cache_append(pool.cache, batches[i], 0, dk, dv)
            rt.tree_attention(pool.cache, batches[i], 0, heads, dq, out, workspace, size)
            rt.cache_keep(pool.cache, batches[i], kept, counts, both[1 - i])
            graph = ctypes.c_void_p()
            xpu.check(rt.lib.xpu_rt_capture_end(rt.handle, ctypes.byref(graph)))
            graphs.append(graph)
        for step in range(steps):
            q, k, v = (normal(r[:n].shape, 30 + 3 * step + i, dtype) for i, r in enumerate(rows))
            for ptr, part, whole in ((dq, q, rows[0]), (dk, k, rows[1]), (dv, v, rows[2])):
                rt.copy_to(ptr, np.concatenate([part, whole[n:]]))
            xpu.check(rt.lib.xpu_rt_graph_launch(rt.handle, graphs[step % 2]))
            for s in range(n):
                p, slot = pool.place(tables[s], contexts[s] + step)
                pool.k[0, p, :, slot], pool.v[0, p, :, slot] = k[s], v[s]
            pool.verify()
            assert list(rt.download(both[(step + 1) % 2], n, np.uint32)) == [c + step + 1 for c in contexts]
            got = rt.download(out, (n + pad) * heads * d, np.uint16).reshape(n + pad, heads, d)
            assert (got[n:] == GUARD).all()
            for s in range(n):
                at = [pool.place(tables[s], p) for p in range(contexts[s] + step + 1)]
                for h in range(heads):
                    keys, vals = (np.array([x[0, p, h // 4, slot] for p, slot in at]) for x in (pool.k, pool.v))
                    want, tol = attend(values(q[s:s + 1, h], dtype), values(keys, dtype), values(vals, dtype),
                                       np.ones((1, len(at)), bool), d ** -0.5, dtype, 64)
                    check(values(got[s:s + 1, h], dtype), want, tol, f"step {step} sequence {s} head {h}")
            # the same again, eagerly, into another context
            spare = b.alloc(4 * n)
            rt.tree_attention(pool.cache, batches[step % 2], 0, heads, dq, out, workspace, size)
            rt.cache_keep(pool.cache, batches[step % 2], kept, counts, spare)
            rt.synchronize()
            again = rt.download(out, got.size, np.uint16).reshape(got.shape)
            assert np.array_equal(again, got)
        for graph in graphs:
            rt.lib.xpu_rt_graph_destroy(graph)


@pytest.mark.parametrize("d,kv,page,n", [(64, 1, 16, 1), (64, 3, 16, 7), (128, 8, 64, 20), (128, 2, 256, 3), (64, 1, 16, 900)])
def test_copy(rt, d, kv, page, n):
    """Up to more pairs than one launch takes."""
    rng = random.Random(3)
    with Buffers(rt) as b:
        pool = Pool(rt, b, 2 * n + 3, kv, d, page, layers=2)
        ids = rng.sample(range(pool.n_pages), 2 * n)
        src, dst = ids[:n], ids[n:]
        if n > 2:
            src[1] = src[0]  # one page to several
        print(f"copy d {d} kv {kv} page {page} n {n}", flush=True)
        rt.cache_copy(pool.cache, src, dst)
        for pools in (pool.k, pool.v):
            pools[:, dst] = pools[:, src]
        pool.verify()
        with pytest.raises(xpu.XpuError, match="exist"):
            rt.cache_copy(pool.cache, [0], [pool.n_pages])
        pool.verify()
        rt.cache_copy(pool.cache, [], [])


def test_copies_are_captured_with_their_pairs(rt):
    """The pairs are read at the call: the caller's arrays may change before a replay."""
    with Buffers(rt) as b:
        pool = Pool(rt, b, 6)
        src, dst = u32([0, 1]), u32([4, 5])
        xpu.check(rt.lib.xpu_rt_capture_begin(rt.handle))
        rt.cache_copy(pool.cache, src, dst)
        graph = ctypes.c_void_p()
        xpu.check(rt.lib.xpu_rt_capture_end(rt.handle, ctypes.byref(graph)))
        src[:], dst[:] = 2, 3
        for i in range(3):
            fresh = normal(pool.k.shape, 20 + i, pool.dtype)
            pool.k[:] = fresh
            rt.copy_to(pool.dk, pool.k)
            xpu.check(rt.lib.xpu_rt_graph_launch(rt.handle, graph))
            pool.k[:, [4, 5]], pool.v[:, [4, 5]] = pool.k[:, [0, 1]], pool.v[:, [0, 1]]
            pool.verify()
        rt.lib.xpu_rt_graph_destroy(graph)


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
def test_a_serving_loop(rt, dtype):
    """Two prompts in, one forked, drafts verified and kept, tokens decoded,
    one conversation ended and the pages compacted: after every step the
    attention is that over what each sequence should hold."""
    kv, heads, d, page, layers, scale = 2, 4, 64, 16, 2, 64 ** -0.5
    rng = random.Random(4)
    with Buffers(rt) as b:
        pool, pages = Pool(rt, b, 40, kv, d, page, layers, dtype), Pages(40)
        seqs, step = [], [0]  # a sequence: its table and, per layer, its keys and values

        def grow(s, n):
            held = len(s["table"]) * page
            more = -(-(s["len"] + n - held) // page) if s["len"] + n > held else 0
            s["table"] += [int(i) for i in pages.take(more)]
            first = s["len"] // page
            last = (s["len"] + n - 1) // page + 1
            ids, src, dst = pages.own(s["table"][first:last])  # the pages that take new rows
            s["table"][first:last] = [int(i) for i in ids]
            rt.cache_copy(pool.cache, src, dst)

        def feed(rows, masks=None):
            """Appends `rows[i]` rows to each sequence in every layer and attends."""
            for s, n in zip(seqs, rows):
                if n:
                    grow(s, n)
            pitch = max(len(s["table"]) for s in seqs)
            tables = u32([s["table"] + [0xFFFFFFFF] * (pitch - len(s["table"])) for s in seqs])
            starts = u32(np.cumsum([0] + rows))
            total = int(starts[-1])
            batch = xpu.Batch(len(seqs), total, pitch, b.up(tables), b.up(starts), b.up(u32([s["len"] for s in seqs])))
            visible = None
            if masks:
                visible = b.up(np.array([m for ms in masks for m in ms], np.uint64))
            for layer in range(layers):
                step[0] += 3
                q, k, v = (normal((total, h, d), 50 + step[0] + i, dtype) for i, h in enumerate((heads, kv, kv)))
                out = b.up(np.full(q.shape, GUARD, np.uint16))
                rt.cache_append(pool.cache, batch, layer, b.up(k), b.up(v))
                size = rt.tree_attention_workspace(pool.cache, batch, heads)
                rt.tree_attention(pool.cache, batch, layer, heads, b.up(q), out, b.alloc(size), size, visible=visible)
                rt.synchronize()
                got = values(rt.download(out, q.size, np.uint16).reshape(q.shape), dtype)
                for i, (s, n) in enumerate(zip(seqs, rows)):
                    a = int(starts[i])
                    s["k"][layer] = np.concatenate([s["k"][layer], k[a:a + n]])
                    s["v"][layer] = np.concatenate([s["v"][layer], v[a:a + n]])
                    c = s["len"]
                    seen = np.ones((n, c + n), bool)
                    for r in range(n):
                        for j in range(n):
                            seen[r, c + j] = masks[i][r] >> j & 1 if masks else j <= r
                    for h in range(heads):
                        want, tol = attend(values(q[a:a + n, h], dtype), values(s["k"][layer][:, h // 2], dtype),
                                           values(s["v"][layer][:, h // 2], dtype), seen, scale, dtype, 64)
                        check(got[a:a + n, h], want, tol, f"step {step[0]} sequence {i} layer {layer} head {h}")
            return batch

        def prompt(lengths):
            """New sequences through prompt_attention, their rows appended."""
            starts = u32(np.cumsum([0] + lengths))
            for n in lengths:
                seqs.append({"table": [], "len": 0, "k": [np.zeros((0, kv, d), np.uint16)] * layers,
                             "v": [np.zeros((0, kv, d), np.uint16)] * layers})
                grow(seqs[-1], n)
            new = seqs[-len(lengths):]
            pitch = max(len(s["table"]) for s in new)
            tables = u32([s["table"] + [0xFFFFFFFF] * (pitch - len(s["table"])) for s in new])
            ds = b.up(starts)
            batch = xpu.Batch(len(new), int(starts[-1]), pitch, b.up(tables), ds, b.up(u32([0] * len(new))))
            packed = xpu.Packed(dtype, heads, kv, d, len(new), int(starts[-1]), ds)
            for layer in range(layers):
                step[0] += 3
                q, k, v = (normal((int(starts[-1]), h, d), 50 + step[0] + i, dtype) for i, h in enumerate((heads, kv, kv)))
                dk, dv, out = b.up(k), b.up(v), b.alloc(q.nbytes)
                rt.prompt_attention(packed, b.up(q), dk, dv, out)
                rt.cache_append(pool.cache, batch, layer, dk, dv)
                rt.synchronize()
                got = values(rt.download(out, q.size, np.uint16).reshape(q.shape), dtype)
                for i, s in enumerate(new):
                    a, n = int(starts[i]), lengths[i]
                    s["k"][layer], s["v"][layer] = k[a:a + n], v[a:a + n]
                    for h in range(heads):
                        want, tol = attend(values(q[a:a + n, h], dtype), values(k[a:a + n, h // 2], dtype),
                                           values(v[a:a + n, h // 2], dtype), np.tri(n, dtype=bool), scale, dtype)
                        check(got[a:a + n, h], want, tol, f"prompt {i} layer {layer} head {h}")
            for s, n in zip(new, lengths):
                s["len"] = n

        prompt([37, 130])
        # a fork of the second: all its pages shared
        pages.share(seqs[1]["table"])
        seqs.append({**seqs[1], "table": list(seqs[1]["table"]), "k": list(seqs[1]["k"]), "v": list(seqs[1]["v"])})
        for _ in range(2):  # drafts: a chain, a bush, a random tree
            trees = [[(2 << i) - 1 for i in range(5)], [1, 3, 5, 9, 17, 33], []]
            for i in range(20):
                p = rng.randint(-1, i - 1)
                trees[2].append((trees[2][p] if p >= 0 else 0) | 1 << i)
            batch = feed([5, 6, 20], trees)
            paths = []
            for ms in trees:
                m = rng.choice(ms)
                paths.append([j for j in range(64) if m >> j & 1])
            flat = [i for ms, p in zip(trees, paths) for i in p + [0] * (len(ms) - len(p))]
            new = b.alloc(12)
            rt.cache_keep(pool.cache, batch, b.up(u32(flat)), b.up(u32([len(p) for p in paths])), new)
            rt.synchronize()
            for s, p in zip(seqs, paths):
                rows = list(range(s["len"])) + [s["len"] + i for i in p]
                s["k"], s["v"] = [x[rows] for x in s["k"]], [x[rows] for x in s["v"]]
                s["len"] += len(p)
            assert list(rt.download(new, 3, np.uint32)) == [s["len"] for s in seqs]
        for rows in ([1, 1, 1], [0, 1, 17]):
            feed(rows)
            for s, n in zip(seqs, rows):
                s["len"] += n
        pages.release(seqs.pop(0)["table"])
        src, dst = pages.compact()
        rt.cache_copy(pool.cache, src, dst)
        for s in seqs:
            s["table"] = [int(i) for i in renumber(src, dst, s["table"])]
        feed([1, 3])
        assert int(rt.download(pool.status, 1, np.uint32)[0]) == 0
