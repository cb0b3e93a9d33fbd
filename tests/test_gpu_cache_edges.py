"""The paged cache's row operations on numbers that do not fit: what they
leave, what they serve all the same, and what the status says."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, Buffers, normal, u32
from test_gpu_cache import Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,kv", [(64, 1), (128, 3)])
@pytest.mark.parametrize("what", ["past the pool", "past the table"])
@pytest.mark.parametrize("count", [5, 20])
def test_keep_reports_missing_pages_of_nodes_that_stay(rt, d, kv, what, count):
    """Kept nodes that are in their place already need no copy, but a page of
    theirs that does not exist sets the status as for any other row. A missing
    page of nodes that are not kept, or behind the sequence, does not."""
    page, rows, context = 16, count + 20, 14
    with Buffers(rt) as b:
        pool = Pool(rt, b, 5, kv, d, page)
        missing = [0, pool.n_pages, 2, 3]
        pitch = 4 if what == "past the pool" else 1
        tables = u32([missing[:pitch]])
        batch = xpu.Batch(1, rows, pitch, b.up(tables), b.up(u32([0, rows])), b.up(u32([context])))
        kept = b.up(u32(range(rows)))
        print(f"keep d {d} kv {kv} {what} count {count}", flush=True)
        for n, status in ((0, 0), (2, 0), (count, 1)):
            new = b.up(u32([GUARD]))
            rt.cache_keep(pool.cache, batch, kept, b.up(u32([n])), new)
            pool.verify(status=status)
            assert list(rt.download(new, 1, np.uint32)) == [context + n]
