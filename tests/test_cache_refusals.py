"""What the paged cache's entry points refuse, without a GPU: a null runtime is
the last thing that a call looks at, so a call that is right in everything else
names it, and any other error is the argument's. And the kernels' checks of the
numbers that live on the device, which are the same functions on host arrays."""
import ctypes

import numpy as np
import pytest

import xpu_playground_amd as xpu

A = 1 << 20  # stands for device memory: never touched here
INVALID = 1


def lib():
    return xpu.library()


def cache(**over):
    args = dict(dtype=0, layers=2, kv_heads=2, head_dim=64, page_size=16, n_pages=8, k=A, v=2 * A)
    strides = {k: over.pop(k) for k in ("layer_stride", "page_stride", "status") if k in over}
    return xpu.Cache(**{**args, **over}, **strides)


def batch(**over):
    return xpu.Batch(**{**dict(n_seqs=2, rows=10, table_pitch=4, tables=3 * A, starts=4 * A, context=5 * A), **over})


def packed(**over):
    return xpu.Packed(**{**dict(dtype=0, heads=4, kv_heads=2, head_dim=64, n_seqs=2, q_rows=10, q_starts=4 * A), **over})


def said(rc):
    return rc, lib().xpu_last_error().decode()


def append(c=None, b=None, layer=0, k=6 * A, k_stride=128, v=7 * A, v_stride=128):
    return said(lib().xpu_cache_append(None, c or cache(), b or batch(), layer, k, k_stride, v, v_stride))


def tree(c=None, b=None, layer=0, heads=4, scale=1.0, q=6 * A, q_stride=256, visible=None, out=7 * A, out_stride=256):
    return said(lib().xpu_tree_attention(None, c or cache(), b or batch(), layer, heads, scale, q, q_stride, visible,
                                         out, out_stride, 8 * A, 1 << 40))


def keep(c=None, b=None, kept=6 * A, counts=7 * A, new=8 * A):
    return said(lib().xpu_cache_keep(None, c or cache(), b or batch(), kept, counts, new))


def copy(c=None, src=(0, 1), dst=(2, 3)):
    s, d = np.array(src, np.uint32), np.array(dst, np.uint32)
    return said(lib().xpu_cache_copy(None, c or cache(), s.ctypes.data, d.ctypes.data, len(s)))


def prompt(p=None, q=6 * A, k=7 * A, v=8 * A, out=9 * A):
    return said(lib().xpu_prompt_attention(None, p or packed(), q, k, v, out))


@pytest.mark.parametrize("call", [append, tree, keep, copy, prompt])
def test_right_arguments_get_as_far_as_the_runtime(call):
    rc, text = call()
    assert rc == INVALID and text.endswith("null runtime"), text


@pytest.mark.parametrize("call", [append, tree, keep, copy])
@pytest.mark.parametrize("over,word", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=512), "page_size"), (dict(page_size=48), "page_size"),
    (dict(layers=0), "positive"), (dict(kv_heads=0), "positive"), (dict(n_pages=0), "positive"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(k=A + 8), "aligned"), (dict(v=A + 2), "aligned"),
    (dict(status=A + 2), "aligned"), (dict(page_stride=2044), "multiples of 8"),
    (dict(page_stride=2040), "overlap"), (dict(layer_stride=8 * 2048 - 8), "overlap"), (dict(layer_stride=0), "overlap"),
    (dict(page_stride=1 << 41), "2^40"), (dict(kv_heads=5000), "4096")])
def test_caches_that_are_refused(call, over, word):
    rc, text = call(c=cache(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


def test_layers_within_pages_are_accepted():
    """[page][layer] order: the page stride spans the layers."""
    rc, text = append(c=cache(layer_stride=2048, page_stride=2 * 2048))
    assert rc == INVALID and text.endswith("null runtime"), text
    rc, text = append(c=cache(layer_stride=2048, page_stride=2 * 2048 - 8))
    assert rc == INVALID and "overlap" in text


@pytest.mark.parametrize("call", [append, tree, keep])
@pytest.mark.parametrize("over,word", [
    (dict(rows=1 << 31), "rows"), (dict(n_seqs=1 << 24), "sequences"), (dict(table_pitch=0), "table_pitch"),
    (dict(tables=None), "null"), (dict(starts=None), "null"), (dict(context=None), "null"), (dict(starts=A + 2), "aligned"),
    (dict(tables=A + 1), "aligned"), (dict(context=A + 3), "aligned")])
def test_batches_that_are_refused(call, over, word):
    rc, text = call(b=batch(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("kwargs,word", [
    (dict(layer=2), "layer"), (dict(k=None), "null k"), (dict(v=None), "null v"), (dict(k=A + 8), "aligned"),
    (dict(k_stride=120), "k_stride"), (dict(v_stride=132), "v_stride"), (dict(k_stride=1 << 24), "k_stride")])
def test_append_refuses(kwargs, word):
    rc, text = append(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("kwargs,word", [
    (dict(layer=2), "layer"), (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=3e38), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=None), "null q"), (dict(out=None), "null out"), (dict(q=A + 4), "aligned"), (dict(q_stride=255), "q_stride"),
    (dict(out_stride=248), "out_stride"), (dict(visible=A + 4), "visible"), (dict(out=6 * A), "overlap"),
    (dict(out=6 * A + 256), "overlap"), (dict(b=batch(rows=1 << 25), out=1 << 50), "rows")])
def test_tree_attention_refuses(kwargs, word):
    rc, text = tree(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("kwargs,word", [
    (dict(kept=None), "null"), (dict(counts=None), "null"), (dict(kept=A + 2), "aligned"), (dict(new=A + 2), "aligned"),
    (dict(new=5 * A), "overlap"), (dict(new=7 * A + 4), "overlap"), (dict(new=4 * A + 8), "overlap"),
    (dict(new=6 * A + 36), "overlap"), (dict(b=batch(rows=0, starts=None)), "null"), (dict(b=batch(rows=0), counts=None), "null")])
def test_keep_refuses(kwargs, word):
    rc, text = keep(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("src,dst,word", [
    ([8], [0], "does not exist"), ([0], [8], "does not exist"), ([0], [0xFFFFFFFF], "does not exist"),
    ([0, 1], [2, 2], "twice"), ([0, 1], [1, 2], "to and from"), ([1, 0], [2, 1], "to and from"), ([3], [3], "to and from")])
def test_copy_refuses(src, dst, word):
    rc, text = copy(src=src, dst=dst)
    assert rc == INVALID and word in text, text


@pytest.mark.parametrize("over,word", [
    (dict(dtype=2), "dtype"), (dict(head_dim=80), "head_dim"), (dict(heads=5), "heads"), (dict(kv_heads=0), "heads"),
    (dict(scale=0.0), "scale"), (dict(q_rows=1 << 31), "rows"), (dict(n_seqs=1 << 24), "sequences"),
    (dict(k_rows=11), "k_rows"), (dict(q_starts=None), "q_starts"), (dict(q_starts=A + 2), "aligned"),
    (dict(k_starts=A + 2), "aligned"), (dict(q_stride=248), "q_stride"), (dict(k_stride=120), "k_stride"),
    (dict(v_stride=130), "v_stride"), (dict(out_stride=1 << 24), "out_stride")])
def test_prompt_attention_refuses(over, word):
    rc, text = prompt(packed(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("kwargs,word", [
    (dict(q=None), "null q"), (dict(k=None), "null k"), (dict(v=None), "null v"), (dict(out=None), "null out"),
    (dict(q=A + 8), "aligned"), (dict(out=6 * A + 16), "out must be q"), (dict(p=packed(out_stride=264), out=6 * A), "out must be q")])
def test_prompt_attention_refuses_pointers(kwargs, word):
    rc, text = prompt(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


def test_page_ids_that_32_bits_do_not_hold():
    for ids in ([-1], np.array([-1]), np.array([1 << 32]), [0.5], [[1]]):
        with pytest.raises(ValueError, match="page ids"):
            xpu.page_ids(ids)
    assert xpu.page_ids([]).dtype == np.uint32 and list(xpu.page_ids(np.array([3, 0xFFFFFFFF]))) == [3, 0xFFFFFFFF]


def test_null_descriptions():
    n = ctypes.c_uint64()
    assert lib().xpu_cache_append(None, None, batch(), 0, A, 128, A, 128) == INVALID
    assert lib().xpu_cache_keep(None, cache(), None, A, A, None) == INVALID
    assert lib().xpu_prompt_attention(None, None, A, A, A, A) == INVALID
    assert lib().xpu_tree_attention_workspace(None, None, batch(), 4, ctypes.byref(n)) == INVALID
    assert lib().xpu_tree_attention_workspace(None, cache(), batch(), 4, None) == INVALID


# ---- the kernels' own checks

def element(page_size, n_pages, stride, table, pos, d=64):
    fn = lib().xpu_internal_cache_element
    fn.restype = ctypes.c_uint64
    fn.argtypes = [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64,
                   ctypes.c_uint32]
    t = np.array(table, np.uint32)
    at = fn(page_size, n_pages, stride, t.ctypes.data, len(t), pos, d)
    return None if at == (1 << 64) - 1 else at


def test_elements_of_positions():
    table = [3, 0, 9, 0xFFFFFFFF]
    assert element(16, 9, 5000, table, 0) == 15000
    assert element(16, 9, 5000, table, 17) == 64
    assert element(16, 9, 5000, table, 15) == 15000 + 15 * 64
    for pos in (32, 47, 48, 63, 64, 1 << 31, (1 << 32) + 5, (1 << 64) - 1):  # pages 9 and 2^32 - 1 of 9; past the table
        assert element(16, 9, 5000, table, pos) is None, pos
    # offsets past 32 bits
    assert element(256, 1 << 20, 1 << 22, [1 << 19], 255, 128) == (1 << 41) + 255 * 128


def lengths(lo, hi, context, rows, pitch, page):
    out = (ctypes.c_uint32 * 5)()
    lib().xpu_internal_cache_lengths(lo, hi, context, rows, pitch, page, out)
    return tuple(out)


def test_lengths_are_cut_to_the_table_and_the_batch():
    assert lengths(3, 10, 20, 10, 2, 16) == (3, 7, 20, 27, 0)
    assert lengths(3, 10, 25, 10, 2, 16) == (3, 7, 25, 32, 0)
    assert lengths(3, 10, 26, 10, 2, 16) == (3, 7, 26, 32, 1)
    assert lengths(3, 10, 0xFFFFFFFF, 10, 2, 16) == (3, 7, 32, 32, 1)
    assert lengths(10, 3, 20, 10, 4, 16)[:2] == (0, 0)
    assert lengths(3, 11, 20, 10, 4, 16)[:2] == (0, 0)
    assert lengths(5, 5, 20, 10, 4, 16)[:2] == (5, 0)
    assert lengths(0, 1, 0xFFFFFFFF, 1, 0xFFFFFFFF, 256) == (0, 1, 0x7FFFFFFF, 0x7FFFFFFF, 1)
