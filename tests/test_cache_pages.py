"""xpu_pages_*: holders of pages, forks, copy on write, compaction, against a
model in Python; everything here runs on the host."""
import ctypes
import random

import numpy as np
import pytest

import xpu_playground_amd as xpu
from xpu_playground_amd.cache import Pages, renumber


def test_take_gives_the_lowest_ids():
    p = Pages(5)
    assert list(p.take(3)) == [0, 1, 2] and p.free == 2
    p.release([1])
    assert list(p.take(2)) == [1, 3] and p.free == 1
    assert [p.holders(i) for i in range(5)] == [1, 1, 1, 1, 0]


def test_a_fork_copies_only_the_pages_it_writes():
    p = Pages(8)
    table = p.take(3)
    fork = table.copy()
    p.share(fork)
    assert [p.holders(i) for i in table] == [2, 2, 2]
    last, src, dst = p.own(fork[-1:])
    assert list(src) == [2] and list(dst) == [3] and list(last) == [3]
    assert p.holders(2) == 1 and p.holders(3) == 1
    last, src, dst = p.own(table[-1:])  # the other holder has it alone now
    assert not len(src) and not len(dst) and list(last) == [2]
    p.release(table)
    assert [p.holders(i) for i in range(4)] == [1, 1, 0, 1]


def test_compaction_moves_the_last_pages_to_the_first_gaps():
    p = Pages(10)
    p.take(9)
    p.release([0, 2, 3, 8])
    p.share([7])
    src, dst = p.compact()
    assert sorted(zip(src, dst)) == [(5, 0), (6, 2), (7, 3)]
    assert [p.holders(i) for i in range(10)] == [1, 1, 1, 2, 1, 0, 0, 0, 0, 0]
    assert list(renumber(src, dst, [7, 1, 5, 9])) == [3, 1, 0, 9]
    assert list(p.take(2)) == [5, 6]
    assert not len(p.compact()[0])


@pytest.mark.parametrize("call", [
    lambda p: p.take(3), lambda p: p.take(1 << 31), lambda p: p.share([4]), lambda p: p.share([0, 99]),
    lambda p: p.release([0, 1, 0, 0]), lambda p: p.release([4]), lambda p: p.release([0, 0xFFFFFFFF]),
    lambda p: p.own([5]), lambda p: p.own([1, 1]), lambda p: p.own([0, 1, 2]), lambda p: p.holders(6)])
def test_a_refused_call_changes_nothing(call):
    p = Pages(6)
    p.take(4)
    p.share([0, 1, 2])
    state = [p.holders(i) for i in range(6)], p.free
    assert state == ([2, 2, 2, 1, 0, 0], 2)
    with pytest.raises(xpu.XpuError):
        call(p)
    assert ([p.holders(i) for i in range(6)], p.free) == state


def test_null_arguments():
    lib, n = xpu.library(), ctypes.c_uint32()
    assert lib.xpu_pages_create(4, None) == 1
    assert lib.xpu_pages_create(0, ctypes.byref(ctypes.c_void_p())) == 1
    assert lib.xpu_pages_take(None, 1, ctypes.addressof(n)) == 1
    assert lib.xpu_pages_share(None, ctypes.addressof(n), 1) == 1
    assert lib.xpu_pages_release(None, None, 0) == 1
    assert lib.xpu_pages_own(None, None, 0, None, None, ctypes.byref(n)) == 1
    assert lib.xpu_pages_compact(None, None, None, None) == 1
    assert lib.xpu_pages_free_count(None, ctypes.byref(n)) == 1
    assert lib.xpu_pages_renumber(None, None, 1, None, 0) == 1
    lib.xpu_pages_destroy(None)
    p = Pages(2)
    assert lib.xpu_pages_take(p.handle, 1, None) == 1 and p.free == 2
    assert lib.xpu_pages_take(p.handle, 0, None) == 0
    p.share([])
    p.release([])


@pytest.mark.parametrize("seed", range(6))
def test_random_use_against_a_model(seed):
    """Sequences that grow, fork, write, end and compact: no page is ever lost,
    shared by mistake or copied without need."""
    rng, n = random.Random(seed), 40
    p, tables, content = Pages(n), [], {}  # content: what each page holds, by id
    stamp = 0
    for _ in range(400):
        act = rng.randrange(6)
        if act <= 1:
            k = rng.randint(1, 5)
            if k <= p.free:
                ids = list(p.take(k))
                for i in ids:
                    stamp += 1
                    content[i] = stamp
                if tables and rng.random() < 0.5:
                    t = rng.choice(tables)
                    t[0] += ids
                    t[1] += [content[i] for i in ids]
                else:
                    tables.append([ids, [content[i] for i in ids]])
            else:
                with pytest.raises(xpu.XpuError):
                    p.take(k)
        elif act == 2 and tables:
            t = rng.choice(tables)
            p.share(t[0])
            tables.append([list(t[0]), list(t[1])])
        elif act == 3 and tables:
            t = rng.choice(tables)
            at = rng.sample(range(len(t[0])), rng.randint(0, len(t[0])))
            shared = sum(p.holders(t[0][i]) > 1 for i in at)
            if shared > p.free:
                with pytest.raises(xpu.XpuError):
                    p.own([t[0][i] for i in at])
                continue
            ids, src, dst = p.own([t[0][i] for i in at])
            assert len(src) == shared
            for a, b in zip(src, dst):
                content[int(b)] = content[int(a)]
            for i, new in zip(at, ids):
                t[0][i] = int(new)
                assert p.holders(int(new)) == 1
                stamp += 1
                content[int(new)] = t[1][i] = stamp  # a write
        elif act == 4 and tables:
            p.release(tables.pop(rng.randrange(len(tables)))[0])
        elif act == 5:
            src, dst = p.compact()
            assert len(set(src) | set(dst)) == 2 * len(src)
            content.update({int(b): content[int(a)] for a, b in zip(src, dst)})
            for t in tables:
                t[0][:] = [int(i) for i in renumber(src, dst, t[0])]
            used = {i for t in tables for i in t[0]}
            assert used == set(range(len(used)))
        held = np.zeros(n, int)
        for ids, stamps in tables:
            for i, s in zip(ids, stamps):
                held[i] += 1
                assert content[i] == s
        assert [p.holders(i) for i in range(n)] == list(held)
        assert p.free == int((held == 0).sum())
