"""The 8-bit paged cache on gfx950 where rows are left out: rows without angles,
without a place, that an earlier sequence claims; kept nodes that do not exist;
and how far rows are off that share a block with rejected and moved ones."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache8_util import BLOCK, Pool8, rescaled, scale_byte, values8
from cache_util import Buffers, codes, normal, u32, values
from test_gpu_cache8 import TYPES, f32

pytestmark = pytest.mark.gpu


def written(pool, layer, table, context, rows, skip=()):
    """What an append makes of rows whose `skip` are written to neither pool."""
    for n, x in rows.items():
        held = pool.codes, pool.scales
        pool.codes, pool.scales = {"k": held[0][n]}, {"k": held[1][n]}
        pool.append(layer, table, context, {"k": x}, skip)
        pool.codes, pool.scales = held


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,kv,page", [(64, 2, 16), (128, 1, 32)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rows_without_angles_are_not_written(rt, dtype, d, kv, page, adjacent):
    """Neither K nor V, nor do they take part in their blocks' scales, however
    large: first, in between, last and all of a block's rows; the rows before the
    batch's in the block stay as they are. cos 1 and sin 0 turn nothing, so K is
    byte for byte too."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 6, kv, d, page, 1, dtype)
        tables, n = u32([[4, 1, 3, 2]]), 37
        k, v = normal((n, kv * d), 5, dtype), normal((n, kv * d), 6, dtype)
        fk, fv = (f32(x, dtype).reshape(n, kv, d) for x in (k, v))
        before = normal((3, kv * d), 7, dtype)
        fb = f32(before, dtype).reshape(3, kv, d)
        rt.cache8_append(pool.cache, xpu.Batch(1, 3, 4, b.up(tables), b.up(u32([0, 3])), b.up(u32([0]))), 0, b.up(before), b.up(before))
        pool.append(0, tables[0], 0, {"k": fb, "v": fb})
        pool.verify()
        cos, sin = np.ones((3, d // 2), np.float32), np.zeros((3, d // 2), np.float32)
        skip = [0, 5, 12] + list(range(13, 29)) + [36]  # positions 3, 8, 15; block 1 (16 .. 31); 39
        for i in skip:
            k[i] = v[i] = codes(np.full(kv * d, 3e4), dtype)
        at = u32([9 if i in skip else i % 3 for i in range(n)])
        at[36] = 0xFFFFFFFF
        rotary = xpu.Rotary(3, d, b.up(cos), b.up(sin), xpu.ADJACENT if adjacent else xpu.HALVES, b.up(at))
        batch = xpu.Batch(1, n, 4, b.up(tables), b.up(u32([0, n])), b.up(u32([3])))
        print(f"append8 without angles d {d} kv {kv} page {page} dtype {dtype}", flush=True)
        rt.cache8_append(pool.cache, batch, 0, b.up(k), b.up(v), rotary)
        written(pool, 0, tables[0], 3, {"k": fk, "v": fv}, skip)
        pool.verify(status=1)


def test_rows_without_a_place_or_a_position(rt):
    """A page past the pool, positions past the table, starts that do not fit, and
    positions past the tables of angles in a block that they begin."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 5, 2, 64, 16, 1)
        k, v = normal((12, 128), 5, pool.dtype), normal((12, 128), 6, pool.dtype)
        fk, fv = f32(k, pool.dtype).reshape(12, 2, 64), f32(v, pool.dtype).reshape(12, 2, 64)
        tables = u32([[0, 5], [1, 2]])
        dk, dv, dt = b.up(k), b.up(v), b.up(tables)
        rt.cache8_append(pool.cache, xpu.Batch(2, 12, 2, dt, b.up(u32([0, 4, 8])), b.up(u32([14, 30]))), 0, dk, dv)
        written(pool, 0, tables[0], 14, {"k": fk[:2], "v": fv[:2]})
        written(pool, 0, tables[1], 30, {"k": fk[4:6], "v": fv[4:6]})
        pool.verify(status=1)
        for starts, context in ([0, 0xFFFFFFF0, 8], [0, 0]), ([6, 3, 1], [0, 0]), ([0, 0, 4], [0, 0xFFFFFFFE]):
            rt.cache8_append(pool.cache, xpu.Batch(2, 12, 2, dt, b.up(u32(starts)), b.up(u32(context))), 0, dk, dv)
        pool.verify(status=1)
        cos, sin = np.ones((3, 32), np.float32), np.zeros((3, 32), np.float32)
        rotary = xpu.Rotary(3, 64, b.up(cos), b.up(sin), eps=0.0)
        rt.copy_to(pool.status, u32([0]))
        rt.cache8_append(pool.cache, xpu.Batch(1, 5, 1, b.up(u32([[3]])), b.up(u32([0, 5])), b.up(u32([0]))), 0, dk, dv, rotary)
        written(pool, 0, u32([3]), 0, {"k": fk[:5], "v": fv[:5]}, skip=(3, 4))
        pool.verify(status=1)


@pytest.mark.parametrize("d,kv,layers,seqs", [(64, 1, 1, 1), (128, 2, 1, 3), (64, 2, 3, 2), (64, 8, 4, 40)])
@pytest.mark.parametrize("more", [0, 20])
def test_a_kept_node_that_does_not_exist(rt, d, kv, layers, seqs, more):
    """The place it would have gone to holds the value that it held, also where
    the block's scale grows by a row from another block. more: nodes kept
    besides, for the form that takes more than 16. 40 sequences: more parts than
    blocks at once."""
    rng = np.random.RandomState(1)
    context, n = 3, 40
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 3 * seqs, kv, d, 16, layers)
        tables = u32(rng.permutation(3 * seqs).reshape(seqs, 3))
        for name in "kv":  # a block's scale is larger than the one's before it
            for t in tables:
                pool.scales[name][:, t] = np.array([110, 112, 115])[None, :, None, None]
            rt.copy_to(pool.ptr[name], pool.raw(name))
        kept = [0xFFFFFFFF, 17, 64, 2, n] + list(range(more))  # 17: position 20, of the second block
        flat = u32(np.tile(kept + [0] * (n - len(kept)), seqs))
        batch = xpu.Batch(seqs, n * seqs, 3, b.up(tables), b.up(u32(np.arange(seqs + 1) * n)), b.up(u32([context] * seqs)))
        print(f"keep8 d {d} kv {kv} layers {layers} seqs {seqs} more {more}", flush=True)
        rt.cache8_keep(pool.cache, batch, b.up(flat), b.up(u32([len(kept)] * seqs)))
        for t in tables:
            # the nodes that do not exist stay where they are
            pool.keep(t, context, [i if i < n else j for j, i in enumerate(kept)], n)
        pool.verify(status=1)


def test_a_kept_node_whose_page_does_not_exist(rt):
    """The same where a node's own page is missing; a place whose page is missing
    gets nothing."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 4, 2, 64, 16, 2)
        tables = u32([[0, 9, 2], [1, 3, 9]])
        for name in "kv":
            for p, s in ((0, 110), (2, 118), (1, 111), (3, 114)):
                pool.scales[name][:, p] = s
            rt.copy_to(pool.ptr[name], pool.raw(name))
        # sequence 0: node 13 (position 16) is on the missing page, node 30 (position 33) raises page 0's scale.
        # sequence 1: node 31 (position 34) is on the missing page
        kept = [[13, 30, 1] + list(range(3, 20)), [31, 14, 15, 2]]
        flat = u32(sum((ids + [0] * (40 - len(ids)) for ids in kept), []))
        batch = xpu.Batch(2, 80, 3, b.up(tables), b.up(u32([0, 40, 80])), b.up(u32([3, 3])))
        rt.cache8_keep(pool.cache, batch, b.up(flat), b.up(u32([len(ids) for ids in kept])))
        for t, ids in zip(tables, kept):
            pool.keep(t, 3, [i if int(t[(3 + i) // 16]) < 4 else j for j, i in enumerate(ids)], 40)
        pool.verify(status=1)


@pytest.mark.parametrize("starts", [[0, 5, 3, 8], [0, 20, 3, 24]])
def test_rows_that_an_earlier_sequence_claims(rt, starts):
    """The last sequence begins with rows of the first; those behind them are its
    own alone, in a block of which it has no earlier rows: what the block held
    before is not in their scale."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 8, 2, 64, 16, 1)
        for n in "kv":
            pool.scales[n][:] = 200
            rt.copy_to(pool.ptr[n], pool.raw(n))
        n, first = starts[3], starts[1]
        k, v = normal((n, 128), 5, pool.dtype), normal((n, 128), 6, pool.dtype)
        tables = u32([[0, 1], [2, 3], [4, 5]])
        batch = xpu.Batch(3, n, 2, b.up(tables), b.up(u32(starts)), b.up(u32([0, 0, 0])))
        rt.cache8_append(pool.cache, batch, 0, b.up(k), b.up(v))
        rt.synchronize()
        for name, x in (("k", k), ("v", v)):
            got, scales = pool.parts(pool.load(name))
            rows = f32(x, pool.dtype).reshape(n, 2, 64)
            for i in range(first, n):
                p, slot = pool.place(tables[2], i - starts[2])
                block = [j for j in range(starts[2], n) if (j - starts[2]) // BLOCK == (i - starts[2]) // BLOCK]
                for h in range(2):
                    scale = int(scales[0, p, h, 0])
                    assert scale <= scale_byte(np.abs(rows[block, h]).max())  # with or without the claimed rows
                    value = np.ldexp(values8(got[0, p, h, slot]), scale - 127)
                    assert (np.abs(value - rows[i, h]) <= 2.0 ** -4 * np.abs(rows[i, h]) + 2.0 ** (scale - 127 - 10)).all()


def test_rows_behind_claimed_ones_in_a_block_with_earlier_rows(rt):
    """Here the last sequence has 5 positions in the block, which are rescaled
    where its own row raises the scale."""
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 8, 1, 64, 16, 1)
        tables = u32([[0], [1], [2]])
        before = normal((5, 64), 7, pool.dtype)
        rt.cache8_append(pool.cache, xpu.Batch(1, 5, 1, b.up(tables[2:]), b.up(u32([0, 5])), b.up(u32([0]))), 0, b.up(before), b.up(before))
        fb = f32(before, pool.dtype).reshape(5, 1, 64)
        pool.append(0, tables[2], 0, {"k": fb, "v": fb})
        rows = normal((6, 64), 8, pool.dtype, 40.0)
        batch = xpu.Batch(3, 6, 1, b.up(tables), b.up(u32([0, 5, 3, 6])), b.up(u32([0, 0, 5])))
        rt.cache8_append(pool.cache, batch, 0, b.up(rows), b.up(rows))
        rt.synchronize()
        got, scales = pool.parts(pool.load("k"))
        scale, old = int(scales[0, 2, 0, 0]), int(pool.scales["k"][0, 2, 0, 0])
        assert scale > old
        a, c = got[0, 2, 0, :5].copy(), rescaled(pool.codes["k"][0, 2, 0, :5], old - scale)
        assert np.array_equal(values8(a), values8(c))
        x = f32(rows, pool.dtype)[5]
        value = np.ldexp(values8(got[0, 2, 0, 7]), scale - 127)
        assert (np.abs(value - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** (scale - 127 - 10)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_beside_rejected_and_moved_ones(rt, dtype):
    """Rows are off by 2^-4 of themselves and 2^-9 of their block's scale at most:
    the first rounding is off by 2^-4 of the value or, below the normal codes, by
    2^-10 of the scale then; as a scale grows, codes that leave the normal ones are
    rounded again, by 2^-10 of the scale it gets; scales grow by factors of two and
    more, so these add up to less than 2^-9 of the last. The last is what the
    largest row needed that came to the block or to the block of a row moved here,
    rejected ones included."""
    rng = np.random.RandomState(2)
    with Buffers(rt) as b:
        pool = Pool8(rt, b, 4, 1, 64, 16, 1, dtype)
        tables = u32([[2, 0, 1]])
        dt, up = b.up(tables), lambda *x: b.up(u32(x))
        held = {}  # position -> row

        def append(at, size):
            row = codes(rng.randn(len(size), 64) * np.array(size, float)[:, None] * 2.0 ** rng.randint(-14, 1, (len(size), 64)), dtype)
            rt.cache8_append(pool.cache, xpu.Batch(1, len(size), 3, dt, up(0, len(size)), up(at)), 0, b.up(row), b.up(row))
            held.update((at + i, x) for i, x in enumerate(values(row, dtype)))
            return values(row, dtype)

        def far(n, tops):
            rt.synchronize()
            for name in "kv":
                got, scales = pool.parts(pool.load(name))
                for pos in range(n):
                    p, slot = pool.place(tables[0], pos)
                    scale = 2.0 ** (int(scales[0, p, 0, 0]) - 127)
                    assert scale == 2.0 ** (scale_byte(tops[pos // BLOCK]) - 127)
                    value = np.ldexp(values8(got[0, p, 0, slot]), int(scales[0, p, 0, 0]) - 127)
                    x = held[pos]
                    assert (np.abs(value - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -9 * scale).all(), (name, pos)

        tops = [np.abs(append(0, [1.0] * 5)).max()]
        far(5, tops)
        for size in (4.0, 9.0, 64.0):  # drafts that are rejected
            tops[0] = max(tops[0], np.abs(append(5, [0.5, size, 1.0])).max())
            far(5, tops)
        tops[0] = max(tops[0], np.abs(append(5, [1.0])).max())
        far(6, tops)
        # a draft into the next two blocks, of which the small row at position 20 is kept: it
        # brings the scale of its block, which a large row beside it has set
        rows = append(6, [1.0] * 10 + [3e3] + [1.0] * 15)
        tops = [max(tops[0], np.abs(rows[:10]).max()), np.abs(rows[10:]).max()]
        rt.cache8_keep(pool.cache, xpu.Batch(1, 26, 3, dt, up(0, 26), up(6)), up(*([14, 3] + [0] * 24)), up(2))
        held.update({6: rows[14], 7: rows[3]})
        assert tops[1] > 8 * tops[0]
        far(8, [tops[1]])
