"""xpu_tree_attention at its edges: rows that see nothing of missing pages, out
beside q in one buffer, what unseen nodes hold."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from cache_util import GUARD, INF, NAN, Buffers, attend, check, normal, u32, values
from test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nodes,missing", [(3, 0), (20, 1), (40, 0), (40, 2), (64, 3)])
def test_rows_that_see_nothing_of_missing_pages(rt, dtype, d, nodes, missing):
    """No context, one row masked to nothing and one page past the pool: every
    element of the sequence's rows is NaN, also those that wavefronts store
    which did not meet the page. The sequence beside it is served, its row that
    sees nothing with zeros."""
    heads, kv, page, n_pages = 4, 2, 16, 9
    pool_k, pool_v = (normal((1, n_pages, kv, page, d), s, dtype) for s in (1, 2))
    tables = u32([[0, 1, 2, 3], [4, 5, 6, 7]])
    tables[0, missing] = n_pages
    rows = nodes + 5
    masks = [(1 << i + 1) - 1 for i in range(nodes)] + [(1 << i + 1) - 1 for i in range(5)]
    masks[1] = masks[nodes + 2] = 0
    q = normal((rows, heads, d), 3, dtype)
    print(f"tree attention d {d} dtype {dtype} nodes {nodes} missing page {missing}", flush=True)
    with Buffers(rt) as b:
        status = b.up(u32([0]))
        cache = xpu.Cache(dtype, 1, kv, d, page, n_pages, b.up(pool_k), b.up(pool_v), status)
        batch = xpu.Batch(2, rows, 4, b.up(tables), b.up(u32([0, nodes, rows])), b.up(u32([0, 0])))
        out = b.up(np.full(q.shape, GUARD, np.uint16))
        size = rt.tree_attention_workspace(cache, batch, heads)
        rt.tree_attention(cache, batch, 0, heads, b.up(q), out, b.alloc(size), size,
                          visible=b.up(np.array(masks, np.uint64)))
        rt.synchronize()
        got = values(rt.download(out, q.size, np.uint16).reshape(q.shape), dtype)
        assert int(rt.download(status, 1, np.uint32)[0]) == 1
    assert np.isnan(got[:nodes]).all(), np.argwhere(~np.isnan(got[:nodes]))[:4]
    assert not got[nodes + 2].any()
    for h in range(heads):
        seen = np.array([[m >> j & 1 for j in range(5)] for m in masks[nodes:]], bool)
        want, tol = attend(values(q[nodes:, h], dtype), values(pool_k[0, 4, h // 2, :5], dtype),
                           values(pool_v[0, 4, h // 2, :5], dtype), seen, d ** -0.5, dtype)
        check(got[nodes:, h], want, tol, f"head {h}")


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("before", [False, True])
def test_out_beside_q_in_one_buffer(rt, dtype, d, before):
    """q and out as columns of one buffer, in either order, with a cut and an
    uncut sequence; nothing but the sequences' columns of out changes."""
    case = Case([3, 40], [2000, 20], 4, 2, d, 16, dtype, 31, first=1)
    want, tol = case.expected(d ** -0.5)
    width = case.heads * d
    x = np.full((case.rows, 2 * width + 8), GUARD, np.uint16)
    at_q, at_out = (width + 8, 0) if before else (0, width + 8)
    x[:, at_q:at_q + width] = case.q.reshape(case.rows, -1)
    with Buffers(rt) as b:
        args, at = case.device(b), b.up(x)
        args.update(q=at + 2 * at_q, out=at + 2 * at_out, q_stride=x.shape[1], out_stride=x.shape[1])
        rt.tree_attention(**args)
        rt.synchronize()
        y = rt.download(at, x.size, np.uint16).reshape(x.shape)
    check(values(y[:, at_out:at_out + width].reshape(case.out.shape), dtype), want, tol)
    y[:, at_out:at_out + width] = GUARD
    assert np.array_equal(y, x)


@pytest.mark.parametrize("dtype", [xpu.BF16, xpu.FP16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("context", [0, 10, 64, 3000])
def test_unseen_nodes_change_no_bit(rt, dtype, d, bad, context):
    """The rows that do not see a node give the same bits whatever its key and value are."""
    case, node = Case([40, 12], [context, 50], 4, 2, d, 16, dtype, 8), 17
    clean = case.run(rt)[0]
    page, slot = case.tables[0, (context + node) // 16], (context + node) % 16
    case.k[1, page, :, slot] = case.v[1, page, :, slot] = (NAN if bad == "nan" else INF)[dtype]
    got = case.run(rt)[0]
    blind = np.array([not m >> node & 1 for m in case.masks[0]] + [True] * (case.rows - 40), bool)
    assert 20 < blind.sum() < case.rows
    assert np.array_equal(got[blind], clean[blind])
    assert not np.isfinite(values(got[~blind], dtype)).any()
