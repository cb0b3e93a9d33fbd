"""Steps of a draft-tree decode on gfx950 with the calls together: rotated rows
appended to an 8-bit cache, attention over it, tokens drawn from what comes out,
accepted nodes kept; eager, checked against 64 bits call by call, and as one
captured graph replayed over a second cache, which has to hold the same bytes
after every step. The batch has rows behind its last sequence, and a sequence
without rows."""
import ctypes
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache8_util import Pool8, values8
from cache_util import GUARD, Buffers, attend, check, normal, u32, values
from rotary_util import tables as rotary_tables, turned
from test_gpu_sample import expected
from test_gpu_tree_attention import tree_masks

pytestmark = pytest.mark.gpu
HEADS, KV, LAYERS, PAGE, STEPS, PAD = 4, 2, 2, 16, 4, 3


class Side:
    """A cache and the buffers of its steps."""

    def __init__(self, rt, b, d, dtype, nodes, n_pages, table, contexts, cos, sin):
        self.rt, self.b, self.nodes = rt, b, nodes
        self.pool = Pool8(rt, b, n_pages, KV, d, PAGE, LAYERS, dtype, seed=3)
        self.rows, n = sum(nodes) + PAD, len(nodes)
        self.starts = u32(np.cumsum([0] + list(nodes)))
        zeros = lambda count, kind=np.uint32: b.up(np.zeros(count, kind))  # noqa: E731
        self.at = {"q": zeros((LAYERS, self.rows, HEADS, d), np.uint16), "k": zeros((LAYERS, self.rows, KV, d), np.uint16),
                   "v": zeros((LAYERS, self.rows, KV, d), np.uint16), "out": zeros((LAYERS, self.rows, HEADS, d), np.uint16),
                   "places": zeros(self.rows), "visible": zeros(self.rows, np.uint64), "random": zeros(self.rows, np.float32),
                   "temperature": zeros(self.rows, np.float32), "kept": zeros(self.rows), "counts": zeros(n),
                   "tokens": zeros(self.rows), "new": zeros(n), "context": b.up(u32(contexts))}
        self.turned = b.up(np.zeros((self.rows, HEADS, d), np.uint16))
        self.batch = xpu.Batch(n, self.rows, table.shape[1], b.up(table), b.up(self.starts), self.at["context"])
        gain = b.up(normal((d,), 9, dtype))
        self.rotary = xpu.Rotary(len(cos), d, b.up(cos), b.up(sin), at=self.at["places"], q_gain=gain, k_gain=gain)
        self.gain = values(normal((d,), 9, dtype), dtype)
        self.sampling = xpu.Sampling(dtype, self.rows, HEADS * d, self.at["random"], self.at["temperature"])
        self.sizes = (rt.tree_attention8_workspace(self.pool.cache, self.batch, HEADS), rt.sample_workspace(self.sampling))
        self.work = [b.alloc(max(s, 16)) for s in self.sizes]
        self.d = d

    def upload(self, step):
        for name, array in step.items():
            self.rt.copy_to(self.at[name], array)

    def layer(self, i):
        rt, at, size = self.rt, self.at, 2 * self.rows * self.d
        rt.cache8_append(self.pool.cache, self.batch, i, at["k"] + i * size * KV, at["v"] + i * size * KV, self.rotary, HEADS,
                         at["q"] + i * size * HEADS, self.turned)
        rt.tree_attention8(self.pool.cache, self.batch, i, HEADS, self.turned, at["out"] + i * size * HEADS, self.work[0],
                           self.sizes[0], visible=at["visible"])

    def finish(self):
        last = self.at["out"] + (LAYERS - 1) * 2 * self.rows * self.d * HEADS
        self.rt.sample(self.sampling, last, self.at["tokens"], self.work[1], self.sizes[1])
        self.rt.cache8_keep(self.pool.cache, self.batch, self.at["kept"], self.at["counts"], self.at["new"])

    def down(self, name, count, kind=np.uint32):
        return self.rt.download(self.at[name], count, kind)


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
@pytest.mark.parametrize("d", [64, 128])
def test_steps_of_a_draft_tree(rt, dtype, d):
    rng = random.Random(5)
    nodes, contexts = [5, 1, 0, 26], [0, 30, 7, 13]
    pitch = (max(contexts) + STEPS * 26 + 26) // PAGE + 1
    ids = list(range(len(nodes) * pitch))
    rng.shuffle(ids)
    table = u32(ids).reshape(len(nodes), pitch)
    cos, sin = rotary_tables(pitch * PAGE, d)
    n_in, total = sum(nodes), sum(nodes) + PAD
    with Buffers(rt) as b:
        eager, graph = (Side(rt, b, d, dtype, nodes, len(ids), table, contexts, cos, sin) for _ in range(2))
        pool, handle, starts = eager.pool, ctypes.c_void_p(), eager.starts
        for step in range(STEPS):
            print(f"d {d} dtype {dtype} step {step} contexts {contexts}", flush=True)
            masks = [tree_masks(n, rng) for n in nodes]
            flat = [m for ms in masks for m in ms]
            places = [c + bin(m).count("1") - 1 for c, ms in zip(contexts, masks) for m in ms]
            kept = [[i for i in range(n) if ms and ms[n - 1] >> i & 1] for n, ms in zip(nodes, masks)]  # the last node's path
            rows = {"q": normal((LAYERS, total, HEADS, d), 11 + step, dtype), "k": normal((LAYERS, total, KV, d), 31 + step, dtype),
                    "v": normal((LAYERS, total, KV, d), 51 + step, dtype)}
            data = {**rows, "out": np.full((LAYERS, total, HEADS, d), GUARD, np.uint16), "places": u32(places + [0] * PAD),
                    "visible": np.array(flat + [0] * PAD, np.uint64),
                    "random": np.random.RandomState(step).rand(total).astype(np.float32) * np.float32(0.999),
                    "temperature": np.where(np.arange(total) % 4 == 3, 0, 0.1 + 0.2 * step).astype(np.float32),
                    "kept": u32([i for n, k in zip(nodes, kept) for i in k + [0xFFFFFFFF] * (n - len(k))] + [0] * PAD),
                    "counts": u32([len(k) for k in kept]), "context": u32(contexts)}
            eager.upload(data)
            graph.upload(data)
            # call by call
            for i in range(LAYERS):
                before = {n: (pool.codes[n].copy(), pool.scales[n].copy()) for n in "kv"}
                eager.layer(i)
                rt.synchronize()
                for n in "kv":
                    pool.codes[n], pool.scales[n] = (x.copy() for x in pool.parts(pool.load(n)))
                    for other in set(range(LAYERS)) - {i}:
                        assert np.array_equal(pool.codes[n][other], before[n][0][other])
                got = rt.download(eager.at["out"], LAYERS * total * HEADS * d, np.uint16).reshape(LAYERS, total, HEADS, d)[i]
                assert (got[n_in:] == GUARD).all()
                q = values(rt.download(eager.turned, total * HEADS * d, np.uint16).reshape(total, HEADS, d), dtype)
                y, size = turned(values(rows["k"][i], dtype)[:n_in], places, cos, sin, gain=eager.gain, eps=1e-6)
                for s, (n, c) in enumerate(zip(nodes, contexts)):
                    a, at = int(starts[s]), list(range(c + n))
                    seen = np.ones((n, n + c), bool)
                    seen[:, c:] = [[m >> j & 1 for j in range(n)] for m in masks[s]] if n else True
                    for h in range(KV):
                        k, v = (pool.read(m, i, table[s], at, h) for m in "kv")
                        for j in range(n):
                            p, slot = pool.place(table[s], c + j)
                            scale = int(pool.scales["k"][i, p, h, slot // 16])
                            x = np.ldexp(values8(pool.codes["k"][i, p, h, slot]), scale - 127)
                            tol = 2.0 ** -4 * np.abs(y[a + j, h]) + 2.0 ** (scale - 137) + 1.1 * 2.0 ** -18 * size[a + j, h]
                            check(x, y[a + j, h], tol, f"sequence {s} node {j}")
                        for m in range(h * HEADS // KV, (h + 1) * HEADS // KV):
                            want, tol = attend(q[a:a + n, m], k, v, seen, d ** -0.5, dtype, 64)
                            check(values(got[a:a + n, m], dtype), want, tol, f"layer {i} sequence {s} head {m}")
            eager.finish()
            rt.synchronize()
            logits = values(got, dtype).reshape(total, -1)
            want = [expected(logits[r], data["temperature"][r], u=data["random"][r])[0] for r in range(total)]
            tokens = eager.down("tokens", total)
            assert np.array_equal(tokens, u32(want))
            for s, k in enumerate(kept):
                pool.keep(table[s], contexts[s], k, nodes[s])
            pool.verify()
            # as a graph
            if step == 0:
                for i in range(LAYERS):
                    graph.layer(i)
                graph.finish()
                rt.synchronize()
                assert np.array_equal(graph.down("tokens", total), tokens)
                for n in "kv":  # back, for the replay
                    rt.copy_to(graph.pool.ptr[n], graph.pool.raw(n))
                xpu.check(rt.lib.xpu_rt_capture_begin(rt.handle))
                for i in range(LAYERS):
                    graph.layer(i)
                graph.finish()
                xpu.check(rt.lib.xpu_rt_capture_end(rt.handle, ctypes.byref(handle)))
                graph.upload(data)
            xpu.check(rt.lib.xpu_rt_graph_launch(rt.handle, handle))
            rt.synchronize()
            assert np.array_equal(graph.down("tokens", total), tokens)
            assert np.array_equal(graph.down("out", LAYERS * total * HEADS * d, np.uint16),
                                  eager.down("out", LAYERS * total * HEADS * d, np.uint16))
            for n in "kv":
                assert np.array_equal(graph.pool.load(n), pool.load(n))
            new = eager.down("new", len(nodes))
            contexts = [c + len(k) for c, k in zip(contexts, kept)]
            assert list(new) == contexts and list(graph.down("new", len(nodes))) == contexts
        rt.lib.xpu_rt_graph_destroy(handle)
