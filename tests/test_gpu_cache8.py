"""The 8-bit paged cache on gfx950, byte for byte: new rows (codes, scales,
earlier rows of a block whose scale grows), rotated rows within their bound,
kept drafts, copied pages, pools that are not dense or pass 32 bits."""
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache8_util import BLOCK, Pool8, rescaled, scale_byte, values8
from cache_util import GUARD, Buffers, check, codes, normal, u32, values
from test_gpu_cache import tables_of
from test_gpu_rotary import ROWS, Turn

pytestmark = pytest.mark.gpu
TYPES = [xpu.BF16, xpu.FP16]


def f32(code, dtype):
    return values(code, dtype).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,kv,page", [(64, 1, 16), (64, 3, 64), (128, 8, 16), (128, 2, 256)])
@pytest.mark.parametrize("rows,contexts,first", ROWS + [([3, 16, 33, 2], [14, 32, 31, 0xF], 1)])
def test_append(rt, dtype, d, kv, page, rows, contexts, first):
    """Without a rotation. Rows of very different sizes, so that scales grow."""
    rng = random.Random(1)
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool8(rt, b, sum(-(-s // page) for s in sizes) + 2, kv, d, page, 2, dtype)
        tables, starts = tables_of(sizes, page, pool.n_pages, rng), u32(np.cumsum([first] + rows))
        total = int(starts[-1]) + 3
        ks, vs = kv * d + 8, kv * d + 24
        size = 2.0 ** np.random.RandomState(3).randint(-12, 9, (total, 1))
        k, v = codes(np.random.RandomState(4).randn(total, ks) * size, dtype), codes(np.random.RandomState(5).randn(total, vs) / size, dtype)
        batch = xpu.Batch(len(rows), total, tables.shape[1], b.up(tables), b.up(starts), b.up(u32(contexts)))
        print(f"append8 d {d} kv {kv} page {page} rows {rows[:6]} contexts {contexts[:6]}", flush=True)
        rt.cache8_append(pool.cache, batch, 1, b.up(k), b.up(v, pad=16), k_stride=ks, v_stride=vs)
        for s, (r, c) in enumerate(zip(rows, contexts)):
            a = int(starts[s])
            pool.append(1, tables[s], c, {n: f32(x[a: a + r, : kv * d], dtype).reshape(r, kv, d) for n, x in (("k", k), ("v", v))})
        pool.verify()


def test_values_at_the_edges(rt):
    """Zeros, the largest and smallest numbers, powers of two and 448 times them,
    infinities and NaN, ties of the rounding, a scale that falls and then grows."""
    rows = np.zeros((64, 2, 64), np.float32)
    big = np.float32(3.38e38)
    for i, x in enumerate([0.0, big, 1e-38, 448.0, 449.0, 1.0, 2.0 ** -100, 3.5, 3.515625, 2.0 ** -92]):
        rows[16 * (i % 4), i % 2, 5 * (i // 4): 5 * (i // 4) + 3] = [x, -x, x / 2]
    rows[17, 0, :3] = [np.inf, -np.inf, np.nan]
    rows[33, 1, :] = np.nan  # a row without a finite value
    rows[50, 0] = np.linspace(-1, 1, 64)
    rows[51, 0] = 1 + np.arange(64) / 64  # ties between codes
    for dtype in TYPES:
        with Buffers(rt) as b:
            pool = Pool8(rt, b, 8, 2, 64, 16, 1, dtype)
            tables = u32([[3, 1, 4, 5, 0]])
            at = 0
            for n in (1, 2, 13, 1, 30, 17):  # blocks are begun, met again and crossed
                k = codes(np.clip(rows, -6e4, 6e4) if dtype == xpu.FP16 else rows, dtype)[at: at + n]
                batch = xpu.Batch(1, n, 5, b.up(tables), b.up(u32([0, n])), b.up(u32([at])))
                rt.cache8_append(pool.cache, batch, 0, b.up(k), b.up(k[::-1].copy()))
                pool.append(0, tables[0], at, {"k": f32(k, dtype), "v": f32(k[::-1].copy(), dtype)})
                pool.verify()
                at += n


def test_a_scale_follows_the_rows(rt):
    """Decode steps: the scale of a block is the largest that its rows needed so
    far, a new block begins anew, and a value is within half a code's step of it."""
    rng = np.random.RandomState(6)
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 4, 1, 64, 16, 1, xpu.BF16)
        tables = u32([[2, 0, 1]])
        dt, ds = b.up(tables), b.up(u32([0, 1]))
        x = values(codes(rng.randn(40, 1, 64) * 2.0 ** rng.randint(-3, 4, (40, 1, 1)), xpu.BF16), xpu.BF16)
        for i in range(40):
            row = codes(x[i: i + 1], xpu.BF16)
            batch = xpu.Batch(1, 1, 3, dt, ds, b.up(u32([i])))
            rt.cache8_append(pool.cache, batch, 0, b.up(row), b.up(row))
            pool.append(0, tables[0], i, {"k": x[i: i + 1].astype(np.float32), "v": x[i: i + 1].astype(np.float32)})
        pool.verify()
        for first in (0, 16, 32):
            rows = x[first: first + 16, 0]
            got = pool.read("k", 0, tables[0], list(range(first, first + len(rows))), 0)
            p, _ = pool.place(tables[0], first)
            scale = 2.0 ** (int(pool.scales["k"][0, p, 0, 0]) - 127)
            assert scale == 2.0 ** (scale_byte(np.abs(rows).max()) - 127)
            # the first rounding is off by 2^-4 of the value, or below the normal
            # codes by half of 2^-9 scales; a code is rounded again only where it
            # leaves the normal ones as the scale grows, by half of 2^-9 new scales
            grown = 1 + np.array([len({scale_byte(np.abs(rows[: j + 1]).max()) for j in range(i, len(rows))}) - 1
                                  for i in range(len(rows))])[:, None]
            assert (np.abs(got - rows) <= 2.0 ** -4 * np.abs(rows) + grown * 2.0 ** -10 * scale).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,heads,kv,page,adjacent,dims", [(64, 4, 1, 16, False, 64), (128, 16, 8, 16, False, 128),
                                                           (128, 5, 5, 64, True, 96), (64, 0, 2, 32, False, 32)])
@pytest.mark.parametrize("rows,contexts,first", ROWS)
def test_append_rotary(rt, dtype, d, heads, kv, page, adjacent, dims, rows, contexts, first):
    """Q as xpu_cache_append_rotary; V byte for byte; K within half a code of the
    rotation in 64 bits, with the scale of its largest value (which may be off
    by the FP32 error where it is next to a border)."""
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool8(rt, b, sum(-(-s // page) for s in sizes) + 2, kv, d, page, 2, dtype)
        t = Turn(rt, b, rows, contexts, heads, kv, d, page, dtype, dims, adjacent, gains=True, first=first, pad=3, pool=pool)
        t.call(rt.cache8_append)
        t.check_q()
        y, size = t.want(t.k, kv, t.gains[1])
        v = f32(t.rows_of(t.v, kv), dtype)
        got_codes, got_scales = pool.parts(pool.load("k"))
        i = 0
        for s, (r, c) in enumerate(zip(rows, contexts)):
            pool.append(1, t.tables[s], c, {"v": v[i: i + r]})
            for start in range(c // BLOCK * BLOCK, c + r, BLOCK) if r else ():
                low, high = max(start, c), min(start + BLOCK, c + r)
                p, slot = pool.place(t.tables[s], start)
                new, err = y[i + low - c: i + high - c], 2.0 ** -18 * size[i + low - c: i + high - c]
                for h in range(kv):
                    top, off = np.abs(new[:, h]).max(), err[:, h].max()
                    now = int(got_scales[1, p, h, slot // BLOCK])
                    old = int(pool.scales["k"][1, p, h, slot // BLOCK]) if low > start else 0
                    assert max(scale_byte(top - off), old) <= now <= max(scale_byte(top + off), old)
                    at = got_codes[1, p, h, slot + low - start: slot + high - start]
                    value = np.ldexp(values8(at), now - 127)
                    tol = 2.0 ** -4 * np.abs(new[:, h]) + 2.0 ** (now - 127 - 10) + 1.1 * err[:, h]
                    check(value, new[:, h], tol, f"sequence {s} position {low} head {h}")
                    if low > start:
                        before = pool.codes["k"][1, p, h, slot: slot + low - start]
                        before[:] = rescaled(before, old - now)
                    pool.codes["k"][1, p, h, slot + low - start: slot + high - start] = at
                    pool.scales["k"][1, p, h, slot // BLOCK] = now
            i += r
        pool.verify()


def test_append_leaves_what_it_cannot_place(rt):
    """A page past the pool, positions past the table or the tables of angles,
    starts that do not fit, and rows that two sequences claim."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 5, 2, 64, 16, 1)
        k, v = normal((12, 128), 5, pool.dtype), normal((12, 128), 6, pool.dtype)
        fk, fv = f32(k, pool.dtype).reshape(12, 2, 64), f32(v, pool.dtype).reshape(12, 2, 64)
        tables = u32([[0, 5], [1, 2]])
        dk, dv, dt = b.up(k), b.up(v), b.up(tables)
        batch = xpu.Batch(2, 12, 2, dt, b.up(u32([0, 4, 8])), b.up(u32([14, 30])))
        rt.cache8_append(pool.cache, batch, 0, dk, dv)
        pool.append(0, tables[0], 14, {"k": fk[:2], "v": fv[:2]})
        pool.append(0, tables[1], 30, {"k": fk[4:6], "v": fv[4:6]})
        pool.verify(status=1)
        for starts, context in ([0, 0xFFFFFFF0, 8], [0, 0]), ([6, 3, 1], [0, 0]), ([0, 0, 4], [0, 0xFFFFFFFE]):
            rt.cache8_append(pool.cache, xpu.Batch(2, 12, 2, dt, b.up(u32(starts)), b.up(u32(context))), 0, dk, dv)
        pool.verify(status=1)
        # positions 3 and up have no angles: not written, and not in the scale
        cos, sin = np.ones((3, 32), np.float32), np.zeros((3, 32), np.float32)
        rotary = xpu.Rotary(3, 64, b.up(cos), b.up(sin), eps=0.0)
        rt.cache8_append(pool.cache, xpu.Batch(1, 5, 1, b.up(u32([[3]])), b.up(u32([0, 5])), b.up(u32([0]))), 0, dk, dv, rotary)
        pool.append(0, u32([3]), 0, {"k": fk[:5], "v": fv[:5]}, skip=(3, 4))
        pool.verify(status=1)
        # rows 2 and 3 are the first sequence's; the second has rows 4 and 5 at positions 2 and 3
        rt.copy_to(pool.status, u32([0]))
        rt.cache8_append(pool.cache, xpu.Batch(3, 12, 1, b.up(u32([[3], [4], [4]])), b.up(u32([0, 4, 2, 6])), b.up(u32([0, 0, 0]))),
                         0, dk, dv)
        pool.append(0, u32([3]), 0, {"k": fk[:4], "v": fv[:4]})
        rt.synchronize()
        got, scales = pool.parts(pool.load("k"))
        for h in range(2):
            value = np.ldexp(values8(got[0, 4, h, 2:4]), int(scales[0, 4, h, 0]) - 127)
            assert (np.abs(value - fk[4:6, h]) <= 2.0 ** -4 * np.abs(fk[4:6, h]) + 2.0 ** (int(scales[0, 4, h, 0]) - 137)).all()


def test_many_sequences(rt):
    rows, contexts = [(i * 7) % 5 for i in range(300)], [(i * 11) % 40 for i in range(300)]
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool8(rt, b, sum(-(-s // 16) for s in sizes) + 1, 1, 64, 16, 1)
        tables, starts = tables_of(sizes, 16, pool.n_pages, random.Random(9)), u32(np.cumsum([2] + rows))
        total = int(starts[-1]) + 1
        k, v = normal((total, 64), 5, pool.dtype), normal((total, 64), 6, pool.dtype)
        starts[150] = 0xFFFFFFFF  # sequences 149 and 150 have no rows then
        batch = xpu.Batch(300, total, tables.shape[1], b.up(tables), b.up(starts), b.up(u32(contexts)))
        rt.cache8_append(pool.cache, batch, 0, b.up(k), b.up(v))
        for s, (r, c) in enumerate(zip(rows, contexts)):
            if s not in (149, 150):
                a = int(starts[s])
                pool.append(0, tables[s], c, {n: f32(x[a: a + r], pool.dtype).reshape(r, 1, 64) for n, x in (("k", k), ("v", v))})
        pool.verify()


@pytest.mark.parametrize("d,kv", [(64, 1), (64, 3), (128, 2)])
@pytest.mark.parametrize("page", [16, 32])
def test_keep(rt, d, kv, page):
    """Paths, repeats, reversals and nothing at all, across blocks and pages."""
    rng = random.Random(2)
    rows = [1, 5, 64, 0, 26, 64, 7, 33, 64]
    contexts = [0, 14, 31, 9, 100, 3, 16, 60, 15]
    kept = [[0], [1, 3, 4], list(range(63, -1, -1)), [], [0, 0, 25, 25, 3], sorted(rng.sample(range(64), 40)), [],
            [rng.randrange(33) for _ in range(33)], list(range(64))]
    with Buffers(rt) as b:
        sizes = [r + c for r, c in zip(rows, contexts)]
        pool = Pool8(rt, b, sum(-(-s // page) for s in sizes) + 1, kv, d, page, 3)
        tables, starts = tables_of(sizes, page, pool.n_pages, rng), u32(np.cumsum([0] + rows))
        batch = xpu.Batch(len(rows), int(starts[-1]), tables.shape[1], b.up(tables), b.up(starts), b.up(u32(contexts)))
        flat = u32([i for r, ids in zip(rows, kept) for i in ids + [0xFFFFFFFF] * (r - len(ids))])
        new = b.up(u32([GUARD] * len(rows)))
        print(f"keep8 d {d} kv {kv} page {page}", flush=True)
        rt.cache8_keep(pool.cache, batch, b.up(flat), b.up(u32([len(ids) for ids in kept])), new)
        for s, ids in enumerate(kept):
            pool.keep(tables[s], contexts[s], ids, rows[s])
        pool.verify()
        assert list(rt.download(new, len(rows), np.uint32)) == [c + len(ids) for c, ids in zip(contexts, kept)]


def test_keep_leaves_what_does_not_fit(rt):
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 9, 1)
        tables = u32([[0, 1, 9, 9, 9, 9], [2, 9, 9, 9, 9, 9], [3, 4, 5, 6, 7, 9]])
        starts, contexts = [0, 4, 8, 80], [0, 14, 0]
        batch = xpu.Batch(3, 80, 6, b.up(tables), b.up(u32(starts)), b.up(u32(contexts)))
        kept = np.zeros(80, np.uint32)
        kept[:4] = [3, 4, 0xFFFFFFFF, 0]
        kept[4:8] = [1, 3, 1, 1]
        new = b.up(u32([GUARD] * 3))
        rt.cache8_keep(pool.cache, batch, b.up(kept), b.up(u32([4, 2, 65])), new)
        pool.keep(tables[0], 0, [3, 4, 0xFFFFFFFF, 0], 4)
        pool.keep(tables[1], 14, [1, 3], 4)
        pool.verify(status=1)
        assert list(rt.download(new, 3, np.uint32)) == [4, 16, GUARD]
        rt.cache8_keep(pool.cache, batch, b.up(kept), b.up(u32([5, 5, 0xFFFFFFFF])), new)
        pool.verify(status=1)


@pytest.mark.parametrize("d,kv,page,n", [(64, 1, 16, 1), (64, 3, 16, 7), (128, 8, 64, 20), (128, 5, 256, 3), (64, 1, 16, 900)])
def test_copy(rt, d, kv, page, n):
    """Codes and scales, up to more pairs than one launch takes; what lies behind
    a page's bytes stays."""
    rng = random.Random(3)
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 2 * n + 3, kv, d, page)
        assert rt.cache8_page_bytes(pool.cache) == pool.bytes
        # a pad that differs from page to page, behind the copied bytes
        raw = {m: pool.raw(m) for m in "kv"}
        for m in "kv":
            raw[m][:, :, pool.bytes:] = np.arange(pool.n_pages, dtype=np.uint8)[None, :, None]
            rt.copy_to(pool.ptr[m], raw[m])
        ids = rng.sample(range(pool.n_pages), 2 * n)
        src, dst = ids[:n], ids[n:]
        if n > 2:
            src[1] = src[0]
        rt.cache8_copy(pool.cache, src, dst)
        rt.synchronize()
        for m in "kv":
            raw[m][:, dst, : pool.bytes] = raw[m][:, src, : pool.bytes]
            assert np.array_equal(pool.load(m), raw[m])
        with pytest.raises(xpu.XpuError, match="exist"):
            rt.cache8_copy(pool.cache, [0], [pool.n_pages])


def test_pages_past_32_bits(rt):
    """K and V in one buffer, 256 MiB between pages: offsets of 5 GiB."""
    stride, pages, kv, d = 1 << 28, 20, 2, 128
    with Buffers(rt) as b:
        base = b.alloc(stride * (pages - 1) + (1 << 16))
        at = 1 << 15  # V's bytes of a page
        cache = xpu.Cache8(xpu.BF16, 1, kv, d, 16, pages, base, base + at, layer_stride=0, page_stride=stride)
        size = rt.cache8_page_bytes(cache)
        k, v = normal((30, kv, d), 1, xpu.BF16), normal((30, kv, d), 2, xpu.BF16)
        tables = u32([[19, 18]])
        for p in (18, 19, 2, 3):
            rt.copy_to(base + p * stride, np.zeros(1 << 16, np.uint8))
        batch = xpu.Batch(1, 30, 2, b.up(tables), b.up(u32([0, 30])), b.up(u32([0])))
        rt.cache8_append(cache, batch, 0, b.up(k), b.up(v))
        rt.cache8_copy(cache, [19, 18], [2, 3])
        q = normal((1, 4, d), 3, xpu.BF16)
        outs = []
        for table in (tables, u32([[2, 3]])):
            one = xpu.Batch(1, 1, 2, b.up(table), b.up(u32([0, 1])), b.up(u32([29])))
            outs.append(b.alloc(q.nbytes))
            need = rt.tree_attention8_workspace(cache, one, 4)
            rt.tree_attention8(cache, one, 0, 4, b.up(q), outs[-1], b.alloc(need), need)
        rt.cache8_keep(cache, xpu.Batch(1, 30, 2, batch.tables, batch.starts, batch.context), b.up(u32(range(29, -1, -1))),
                       b.up(u32([30])))
        rt.synchronize()
        small = Pool8(rt, b, 20, kv, d, 16, 1)  # the same, dense
        for n in "kv":
            small.codes[n][:] = small.scales[n][:] = 0
        small.append(0, tables[0], 0, {"k": f32(k, xpu.BF16), "v": f32(v, xpu.BF16)})
        for n, shift in (("k", 0), ("v", at)):
            want = small.raw(n)[0]
            for p, of in ((2, 19), (3, 18)):
                got = rt.download(base + p * stride + shift, size, np.uint8)
                assert np.array_equal(got[: kv * 16 * d + kv], want[of][: kv * 16 * d + kv])
        a, c = (rt.download(o, q.size, np.uint16) for o in outs)
        assert np.array_equal(a, c)
        small.keep(tables[0], 0, list(range(29, -1, -1)), 30)
        for n, shift in (("k", 0), ("v", at)):
            want = small.raw(n)[0]
            for p in (18, 19):
                got = rt.download(base + p * stride + shift, size, np.uint8)
                assert np.array_equal(got[: kv * 16 * d + kv], want[p][: kv * 16 * d + kv]), (n, p)


def test_layers_within_pages(rt):
    """[page][layer] order, pages of the least stride."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 6, 1, 64, 16, 3)
        size = pool.bytes
        order = {n: np.ascontiguousarray(pool.raw(n)[:, :, :size].transpose(1, 0, 2)) for n in "kv"}
        ptr = {n: b.up(order[n]) for n in "kv"}
        cache = xpu.Cache8(pool.dtype, 3, 1, 64, 16, 6, ptr["k"], ptr["v"], pool.status, layer_stride=size, page_stride=3 * size)
        tables = u32([[4, 2]])
        k, v = normal((20, 1, 64), 1, pool.dtype), normal((20, 1, 64), 2, pool.dtype)
        batch = xpu.Batch(1, 20, 2, b.up(tables), b.up(u32([0, 20])), b.up(u32([5])))
        rt.cache8_append(cache, batch, 2, b.up(k), b.up(v))
        rt.cache8_keep(cache, batch, b.up(u32([19, 3] + [0] * 18)), b.up(u32([2])))
        pool.append(2, tables[0], 5, {"k": f32(k, pool.dtype), "v": f32(v, pool.dtype)})
        pool.keep(tables[0], 5, [19, 3], 20)
        rt.synchronize()
        for n in "kv":
            got = rt.download(ptr[n], order[n].size, np.uint8).reshape(order[n].shape)
            assert np.array_equal(got, pool.raw(n)[:, :, :size].transpose(1, 0, 2))
