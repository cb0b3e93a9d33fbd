"""xpu_tree_attention on gfx950 against attention in 64 bits (the bound is
derived in cache_util.py): trees, chains and single tokens over pages in any
order, contexts that end inside a page or a tile, cut into chunks or not, what
unseen positions hold, wrong pages and lengths, strides, capture."""
import ctypes
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, INF, NAN, Buffers, attend, check, normal, u32, values

pytestmark = pytest.mark.gpu

TYPES = [xpu.BF16, xpu.FP16]


def tree_masks(n, rng, empty=False):
    """Ancestors and self of every node of a random tree."""
    masks = []
    for i in range(n):
        parent = rng.randint(max(-1, i - 4), i - 1)
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    if empty and n:
        masks[rng.randrange(n)] = 0
    return masks


class Case:
    """Sequences over pages in random order. Positions behind a sequence's
    end, and pages of no sequence, hold NaN."""

    def __init__(self, nodes, contexts, heads, kv, d, page, dtype, seed, masked=True, layers=2, first=0, spare=3,
                 gain=1.0, empty=False):
        rng = random.Random(seed)
        self.nodes, self.contexts, self.heads, self.kv, self.d, self.page, self.dtype = \
            nodes, contexts, heads, kv, d, page, dtype
        ends = [n + c for n, c in zip(nodes, contexts)]
        held = [-(-e // page) for e in ends]
        ids = list(range(sum(held) + spare))
        rng.shuffle(ids)
        self.n_pages, self.layers = len(ids), layers
        self.pitch = max(max(held), 1) + 1
        self.tables = np.full((len(nodes), self.pitch), 0xFFFFFFFF, np.uint32)  # not looked at past the end
        self.starts = u32(np.cumsum([first] + list(nodes)))
        self.rows = int(self.starts[-1]) + spare
        self.k = np.full((layers, self.n_pages, kv, page, d), NAN[dtype], np.uint16)
        self.v = self.k.copy()
        self.keys, self.vals, at = [], [], 0
        for s, (e, m) in enumerate(zip(ends, held)):
            self.tables[s, :m] = ids[at: at + m]
            at += m
            k, v = normal((e, kv, d), seed + 10 + s, dtype, gain), normal((e, kv, d), seed + 900 + s, dtype)
            self.keys.append(k)
            self.vals.append(v)
            for p in range(e):
                self.k[1, self.tables[s, p // page], :, p % page] = k[p]
                self.v[1, self.tables[s, p // page], :, p % page] = v[p]
        self.q = normal((self.rows, heads, d), seed + 1, dtype, gain)
        self.masks = [tree_masks(n, rng, empty) for n in nodes] if masked else None
        self.out = np.full(self.q.shape, GUARD, np.uint16)

    def visible(self):
        if self.masks is None:
            return None
        # the bits past a sequence's nodes are not looked at
        flat = [m | (~((1 << n) - 1) & (1 << 64) - 1) for n, ms in zip(self.nodes, self.masks) for m in ms]
        first = int(self.starts[0])
        return np.array([0] * first + flat + [0] * (self.rows - first - len(flat)), np.uint64)

    def seen(self, s):
        n, c = self.nodes[s], self.contexts[s]
        seen = np.zeros((n, n + c), bool)
        seen[:, :c] = True
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
            a, seen = int(self.starts[s]), self.seen(s)
            k, v = values(self.keys[s], self.dtype), values(self.vals[s], self.dtype)
            for h in range(self.heads):
                want[a:a + n, h], tol[a:a + n, h] = attend(q[a:a + n, h], k[:, h // group], v[:, h // group], seen,
                                                           scale, self.dtype, 64)
        return want, tol

    def device(self, b, status=None):
        cache = xpu.Cache(self.dtype, self.layers, self.kv, self.d, self.page, self.n_pages, b.up(self.k), b.up(self.v),
                          status)
        batch = xpu.Batch(len(self.nodes), self.rows, self.pitch, b.up(self.tables), b.up(self.starts),
                          b.up(u32(self.contexts)))
        vis = self.visible()
        size = b.rt.tree_attention_workspace(cache, batch, self.heads)
        return dict(cache=cache, batch=batch, layer=1, heads=self.heads, q=b.up(self.q), out=b.up(self.out),
                    workspace=b.alloc(size), workspace_bytes=size, visible=None if vis is None else b.up(vis))

    def run(self, rt, scale=None):
        print(f"tree attention nodes {self.nodes[:8]} contexts {self.contexts[:8]} heads {self.heads}/{self.kv} d {self.d} "
              f"page {self.page} dtype {self.dtype} masked {self.masks is not None}", flush=True)
        with Buffers(rt) as b:
            status = b.up(u32([0]))
            args = self.device(b, status)
            rt.tree_attention(**args, scale=scale)
            rt.synchronize()
            got = rt.download(args["out"], self.out.size, np.uint16).reshape(self.out.shape)
            return got, int(rt.download(status, 1, np.uint32)[0])

    def verify(self, rt, scale=None):
        got, status = self.run(rt, scale)
        want, tol = self.expected(self.d ** -0.5 if scale is None else scale)
        check(values(got, self.dtype), want, tol)
        assert status == 0
        return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_single_tokens(rt, dtype, d, page):
    contexts = [0, 1, 15, 16, 31, 32, 33, 127, 128, 500]
    Case([1] * len(contexts), contexts, 4, 2, d, page, dtype, 1, masked=False).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,heads,kv", [(16, 4, 2), (32, 2, 2), (64, 8, 1), (16, 12, 2)])
def test_trees(rt, dtype, d, page, heads, kv):
    Case([1, 5, 0, 26, 64, 33, 7], [0, 17, 40, 31, 130, 300, 64], heads, kv, d, page, dtype, 2).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nodes,contexts", [
    ([64], [0]), ([64], [5000]), ([1], [4999]), ([3], [3001]), ([20, 1, 64], [2000, 3000, 10]), ([64] * 3, [31, 32, 33])])
def test_long_contexts_are_cut(rt, dtype, nodes, contexts):
    """More chunks than one, joined in order; short sequences beside long ones."""
    Case(nodes, contexts, 4, 2, 128, 16, dtype, 3).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes,contexts", [([200, 65, 1], [0, 100, 700]), ([129], [1000]), ([64, 64], [0, 64])])
def test_chains_of_any_length(rt, dtype, d, nodes, contexts):
    Case(nodes, contexts, 4, 2, d, 32, dtype, 4, masked=False).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 8), (32, 1), (40, 4), (3, 3)])
def test_head_layouts(rt, dtype, heads, kv):
    Case([3, 9], [100, 37], heads, kv, 64, 16, dtype, 5).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_see_nothing(rt, dtype):
    """An empty mask over an empty context gives zeros; over a context, that context."""
    case = Case([4, 9, 40], [0, 70, 0], 4, 2, 128, 16, dtype, 6, empty=True)
    got = case.verify(rt)
    for s in (0, 2):
        for i, m in enumerate(case.masks[s]):
            assert (m == 0) == (not got[case.starts[s] + i].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,gain", [(0.02, 1.0), (1.0, 1.0), (0.125, 6.0)])
def test_scales(rt, dtype, scale, gain):
    Case([20, 5], [700, 2000], 2, 1, 128, 16, dtype, 7, gain=gain).verify(rt, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("context", [0, 10, 64, 600])
def test_unseen_nodes_take_no_part(rt, dtype, d, bad, context):
    """A branch whose keys and values are not finite reaches only the rows that
    see it."""
    case = Case([40, 12], [context, 50], 4, 2, d, 16, dtype, 8)
    node, code = 17, (NAN if bad == "nan" else INF)[dtype]
    want, tol = case.expected(d ** -0.5)
    page, slot = case.tables[0, (context + node) // 16], (context + node) % 16
    case.k[1, page, 0, slot, 5] = code
    case.v[1, page, 1, slot, 9] = code
    got, status = case.run(rt)
    got = values(got, dtype)
    sees = np.array([m >> node & 1 for m in case.masks[0]], bool)
    assert sees.any() and not sees.all() and status == 0
    check(got[40:52], want[40:52], tol[40:52])
    check(got[:40][~sees], want[:40][~sees], tol[:40][~sees], "rows that do not see it")
    with np.errstate(invalid="ignore"):
        assert not np.isfinite(got[:40][sees][:, 2:, 9]).any()
        if bad == "nan":
            assert np.isnan(got[:40][sees][:, :2]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("context", [40, 700, 2999, 9000])
@pytest.mark.parametrize("heads,kv", [(4, 2), (40, 2)])
def test_infinities_that_rows_see(rt, dtype, context, heads, kv):
    """An infinite value comes out as itself, wherever the cut puts it; the other dims are not touched."""
    case = Case([3, 4], [context, 50], heads, kv, 64, 16, dtype, 18, masked=False)
    want, tol = case.expected(64 ** -0.5)
    spots = sorted({0, context // 2, context - 1, context})
    for dim, at in enumerate(spots):
        case.v[1, case.tables[0, at // 16], :, at % 16, 7 + dim] = INF[dtype] | (0x8000 if dim % 2 else 0)
        want[:3, :, 7 + dim] = -np.inf if dim % 2 else np.inf
    got, status = case.run(rt)
    check(values(got, dtype), want, tol)
    assert status == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["id", "id in the middle", "context", "nodes"])
def test_pages_and_lengths_that_do_not_exist(rt, dtype, what):
    """That sequence's rows are NaN and the status says so; the others are served."""
    nodes = [3, 70, 2] if what == "nodes" else [3, 6, 2]
    case = Case(nodes, [40, 900, 33], 4, 2, 128, 16, dtype, 9, masked=False)
    want, tol = case.expected(128 ** -0.5, only=(0, 2))
    if what == "nodes":
        case.masks = [[(1 << i + 1) - 1 for i in range(min(n, 64))] + [0] * max(n - 64, 0) for n in nodes]
    elif what == "context":
        case.contexts = [40, case.pitch * 16 - 5, 33]
    else:
        case.tables[1, 0 if what == "id" else 30] = case.n_pages
    got, status = case.run(rt)
    got, a, b = values(got, dtype), int(case.starts[1]), int(case.starts[2])
    assert status == 1 and np.isnan(got[a:b]).all()
    for part in (slice(0, a), slice(b, None)):
        check(got[part], want[part], tol[part])


def test_lengths_beyond_all_bounds(rt):
    """Contexts and starts of random bits: rows stay, or become NaN; nothing else happens."""
    case = Case([3, 6, 2], [40, 90, 33], 4, 2, 128, 16, xpu.BF16, 10, masked=False)
    want, tol = case.expected(128 ** -0.5, only=(0,))
    case.contexts = [40, 0xFFFFFFFF, 0x80000001]
    got, status = case.run(rt)
    got = values(got, xpu.BF16)
    check(got[:3], want[:3], tol[:3])
    assert status == 1 and np.isnan(got[3:11]).all()
    check(got[11:], want[11:], tol[11:])
    case.contexts, case.starts = [40, 90, 33], u32([0, 3, 1, 4000000000])
    got, _ = case.run(rt)
    check(values(got, xpu.BF16)[:3], want[:3], tol[:3])
    assert (got[3:] == GUARD).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nodes, contexts, heads, kv, d", [
    ([1], [17000], 3, 1, 128),            # a row of 128 chunks or more: sixteen wavefronts, an odd head
    ([2, 1, 2], [900, 17000, 130], 4, 4, 64),  # the same, with rows of few chunks and of none
    ([41], [1500], 32, 8, 64),            # four wavefronts a join
    ([110], [700], 32, 4, 64),            # one
    ([1, 70, 41], [3000, 0, 700], 30, 10, 128),
])
def test_joins_by_any_number_of_wavefronts(rt, dtype, nodes, contexts, heads, kv, d):
    Case(nodes, contexts, heads, kv, d, 64, dtype, 21, masked=False, layers=2, spare=1).verify(rt)


@pytest.mark.parametrize("n, few, kv", [(1, 64, 8), (5, 64, 8), (20, 30, 8), (46, 3, 8), (60, 3, 8), (64, 30, 2), (64, 1, 16)])
def test_ragged_batches_are_cut_to_fit_or_not(rt, n, few, kv):
    """Every work item runs, and every row is written, however the rows fill a round of the chip."""
    rng = random.Random(n * 100 + few)
    nodes = [rng.randint(1, few) for _ in range(n)]
    contexts = [int(60 * 80 ** rng.random()) for _ in range(n)]
    Case(nodes, contexts, 2 * kv, kv, 64, 64, xpu.BF16, 23, layers=2).verify(rt)


def test_more_work_than_the_workspace_holds(rt):
    """Starts that go back give more work items than ascending ones could:
    rows that would be joined from behind the workspace are left, with status."""
    heads, d, page, n = 8, 64, 16, 4001
    rows, pitch = 20, 61
    starts = u32([0, 16] * ((n - 1) // 2) + [16, 20])  # the first rows 2000 times, then the last ones
    with Buffers(rt) as b:
        status, pool = b.up(u32([0])), np.zeros((1, 1, page, d), np.uint16)
        cache = xpu.Cache(xpu.BF16, 1, 1, d, page, 1, b.up(pool), b.up(pool), status)
        batch = xpu.Batch(n, rows, pitch, b.up(np.zeros((n, pitch), np.uint32)), b.up(starts), b.up(u32([0] * (n - 1) + [960])))
        out = np.full((rows, heads, d), GUARD, np.uint16)
        size, to = rt.tree_attention_workspace(cache, batch, heads), b.up(out)
        rt.tree_attention(cache=cache, batch=batch, layer=0, heads=heads, q=b.up(np.zeros_like(out)), out=to,
                          workspace=b.alloc(size), workspace_bytes=size)
        rt.synchronize()
        got = rt.download(to, out.size, np.uint16).reshape(out.shape)
        assert int(rt.download(status, 1, np.uint32)[0]) == 1
    assert (got[16:] == GUARD).all() and (got[:16] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_rows_of_no_sequence(rt, dtype):
    """Pages with layers inside, q as a part of a wider row, rows before the
    first and behind the last sequence."""
    case = Case([2, 30], [77, 500], 4, 2, 64, 32, dtype, 11, first=2)
    want, tol = case.expected(64 ** -0.5)
    page = case.kv * case.page * case.d
    wide = np.full((case.rows, 5 * 64 + 8), GUARD, np.uint16)
    wide[:, 64:320] = case.q.reshape(case.rows, -1)
    with Buffers(rt) as b:
        k, v = (np.full((case.n_pages, case.layers * page + 16), NAN[dtype], np.uint16) for _ in range(2))
        for pool, src in ((k, case.k), (v, case.v)):
            pool[:, : case.layers * page] = src.transpose(1, 0, 2, 3, 4).reshape(case.n_pages, -1)
        args = case.device(b)
        args["cache"] = xpu.Cache(dtype, case.layers, case.kv, case.d, case.page, case.n_pages, b.up(k, pad=16),
                                  b.up(v, pad=48), layer_stride=page, page_stride=case.layers * page + 16)
        out = np.full((case.rows, 272), GUARD, np.uint16)
        args.update(q=b.up(wide) + 128, q_stride=5 * 64 + 8, out=b.up(out), out_stride=272)
        rt.tree_attention(**args)
        rt.synchronize()
        got = rt.download(args["out"], out.size, np.uint16).reshape(out.shape)
    assert (got[:, 256:] == GUARD).all()
    check(values(got[:, :256].reshape(case.out.shape), dtype), want, tol)


def test_pages_past_four_gigabytes(rt):
    """Page offsets that 32 bits do not hold, in elements and in bytes."""
    dtype, d, page, kv = xpu.BF16, 128, 16, 2
    case = Case([3, 1], [90, 20], 4, kv, d, page, dtype, 12)
    stride = 1 << 28  # 512 MiB between pages
    want, tol = case.expected(d ** -0.5)
    n = kv * page * d
    with Buffers(rt) as b:
        args = case.device(b)
        size = ((case.n_pages - 1) * stride + n) * 2
        k, v = b.alloc(size), b.alloc(size)
        assert size > 5 << 30
        for i in range(case.n_pages):
            rt.copy_to(k + i * stride * 2, case.k[1, i])
            rt.copy_to(v + i * stride * 2, case.v[1, i])
        args["cache"] = xpu.Cache(dtype, 1, kv, d, page, case.n_pages, k, v, page_stride=stride)
        args["layer"] = 0
        rt.tree_attention(**args)
        rt.synchronize()
        got = rt.download(args["out"], case.out.size, np.uint16).reshape(case.out.shape)
    check(values(got, dtype), want, tol)


def test_a_workspace_that_is_too_small_is_refused(rt):
    case = Case([3], [3000], 4, 2, 64, 16, xpu.BF16, 13)
    with Buffers(rt) as b:
        args = case.device(b)
        assert args["workspace_bytes"] > 0
        for change in (dict(workspace_bytes=args["workspace_bytes"] - 1), dict(workspace=None),
                       dict(workspace=args["workspace"] + 4)):
            with pytest.raises(xpu.XpuError, match="workspace"):
                rt.tree_attention(**{**args, **change})
        short = xpu.Batch(1, 3, 4, args["batch"].tables, args["batch"].starts, args["batch"].context)
        assert rt.tree_attention_workspace(args["cache"], short, 4) == 0  # never cut


def test_captured_graphs_share_a_workspace(rt):
    cases = [Case([20, 1], [2000, 900], 4, 2, 128, 16, xpu.BF16, 14), Case([1, 1, 1], [3000, 5, 700], 4, 2, 128, 16, xpu.BF16, 15)]
    with Buffers(rt) as b:
        calls = [c.device(b) for c in cases]
        size = max(c["workspace_bytes"] for c in calls)
        workspace = b.alloc(size)
        runs = []
        for case, args in zip(cases, calls):
            args.update(workspace=workspace, workspace_bytes=size)
            rt.tree_attention(**args)
            rt.synchronize()
            eager = rt.download(args["out"], case.out.size, np.uint16)
            want, tol = case.expected(128 ** -0.5)
            check(values(eager.reshape(case.out.shape), xpu.BF16), want, tol)
            xpu.check(rt.lib.xpu_rt_capture_begin(rt.handle))
            rt.tree_attention(**args)
            graph = ctypes.c_void_p()
            xpu.check(rt.lib.xpu_rt_capture_end(rt.handle, ctypes.byref(graph)))
            runs.append((case, args, eager, graph))
        for _ in range(3):
            for case, args, eager, graph in runs:  # without a wait between the two graphs
                rt.copy_to(args["out"], case.out)
                xpu.check(rt.lib.xpu_rt_graph_launch(rt.handle, graph))
            rt.synchronize()
            for case, args, eager, graph in runs:
                assert np.array_equal(rt.download(args["out"], eager.size, np.uint16), eager)
                rt.tree_attention(**args)
            rt.synchronize()
            for case, args, eager, graph in runs:
                assert np.array_equal(rt.download(args["out"], eager.size, np.uint16), eager)
        for run in runs:
            rt.lib.xpu_rt_graph_destroy(run[3])


def test_many_sequences(rt):
    """More sequences than a wavefront counts at once, some without rows."""
    rng = random.Random(16)
    nodes = [rng.choice([0, 1, 1, 2, 5]) for _ in range(150)]
    Case(nodes, [rng.randint(0, 60) for _ in nodes], 2, 1, 64, 16, xpu.FP16, 16).verify(rt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, d, few", [(2, 64, 1), (8, 128, 9)])
def test_many_sequences_with_long_ones_among_them(rt, dtype, heads, d, few):
    """The long ones' keys are cut, whichever 64 sequences they are among."""
    nodes, contexts = [few] * 140, [5] * 140
    for s, n, c in ((3, 20, 3000), (64, 1, 9000), (127, 11, 700), (139, 30, 5000)):
        nodes[s], contexts[s] = n, c
    Case(nodes, contexts, heads, 1, d, 32, dtype, 18, layers=2).verify(rt)
