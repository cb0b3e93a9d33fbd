"""How xpu_cache_copy checks its pairs, on the host (a null runtime is the last
thing that the call looks at): against a model, and at a cost that goes by the
pairs and not by the pool."""
import random
import time

import numpy as np
import pytest

import xpu_playground_amd as xpu

A = 1 << 20  # stands for device memory: never touched here


def copy(n_pages, src, dst):
    s, d = np.array(src, np.uint32), np.array(dst, np.uint32)
    c = xpu.Cache(0, 1, 1, 64, 16, n_pages, A, 2 * A)
    assert xpu.library().xpu_cache_copy(None, c, s.ctypes.data, d.ctypes.data, len(s)) == 1
    return xpu.library().xpu_last_error().decode()


def model(n_pages, src, dst):
    to = set()
    for a, b in zip(src, dst):
        if a >= n_pages or b >= n_pages:
            return f"page {max(a, b)} does not exist"
        if b in to:
            return f"page {b} is copied to twice"
        to.add(b)
    for i in range(len(src)):
        if src[i] in to:
            return f"page {src[i]} is copied to and from"
    return "null runtime"


@pytest.mark.parametrize("n_pages", [1, 2, 9, 64, 1000, 100000, (1 << 30) - 1])
@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 400, 401, 3000])
def test_pairs_against_a_model(n_pages, n):
    rng = random.Random(n)
    if n_pages < 2 * n:
        # more pairs than pages: some page is written twice, or does not exist
        ids = [rng.randrange(n_pages + 1) for _ in range(2 * n)]
        assert copy(n_pages, ids[:n], ids[n:]).split(": ")[1] == model(n_pages, ids[:n], ids[n:])
        return
    step = rng.choice([1, 2, 1 << 5]) if n_pages < 1 << 20 else rng.choice([1, 1 << 16])  # ids that share their low bits
    ids = [i * step % n_pages for i in range(2 * n)]
    if len(set(ids)) < 2 * n:
        ids = list(range(2 * n))
    rng.shuffle(ids)
    src, dst = ids[:n], ids[n:]
    assert copy(n_pages, src, dst).endswith("null runtime")
    src[n // 2:] = src[: n - n // 2]  # a page may be copied to several
    assert copy(n_pages, src, dst).endswith("null runtime")
    for spoil in ("twice", "from", "src", "dst"):
        s, d = list(src), list(dst)
        i, j = rng.randrange(n), rng.randrange(n)
        if spoil == "twice" and n > 1:
            d[i] = d[i - 1]
        elif spoil == "from":
            s[i] = d[j]
        elif spoil == "src":
            s[i] = rng.choice([n_pages, n_pages + 2, 0xFFFFFFFF])
        elif spoil == "dst":
            d[i] = n_pages
        assert copy(n_pages, s, d).split(": ")[1] == model(n_pages, s, d), spoil


def test_the_pool_does_not_count():
    """One copy in the largest pool there can be at this page size: no work or memory per page
    (a byte for each would be 1 GiB)."""
    best = min(timed() for _ in range(3))
    assert best < 0.02, best


def timed():
    start = time.perf_counter()
    assert copy((1 << 30) - 1, [5, 9], [1000000000, 7]).endswith("null runtime")
    return time.perf_counter() - start
