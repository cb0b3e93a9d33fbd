"""What the rotated append, the 8-bit cache and the sampling refuse, without a
GPU: a null runtime is the last thing that a call looks at, so a call that is
right in everything else names it, and any other error is the argument's."""
import ctypes

import numpy as np
import pytest

import xpu_playground_amd as xpu
from test_cache_refusals import A, INVALID, batch, lib, said
from test_cache_refusals import cache as cache16

U64 = ctypes.c_uint64


def cache(**over):
    args = dict(dtype=0, layers=2, kv_heads=2, head_dim=64, page_size=16, n_pages=8, k=A, v=2 * A)
    strides = {k: over.pop(k) for k in ("layer_stride", "page_stride", "status") if k in over}
    return xpu.Cache8(**{**args, **over}, **strides)


def rotary(**over):
    return xpu.Rotary(**{**dict(positions=100, dims=64, cos=10 * A, sin=11 * A), **over})


def append(c=None, b=None, layer=0, turn=0, heads=4, q=12 * A, q_stride=256, q_out=13 * A, out_stride=256, k=6 * A,
           k_stride=128, v=7 * A, v_stride=128):
    return said(lib().xpu_cache8_append(None, c or cache(), b or batch(), layer, rotary() if turn == 0 else turn, heads, q,
                                        q_stride, q_out, out_stride, k, k_stride, v, v_stride))


def append16(c=None, b=None, layer=0, turn=0, heads=4, q=12 * A, q_stride=256, q_out=13 * A, out_stride=256, k=6 * A,
             k_stride=128, v=7 * A, v_stride=128):
    return said(lib().xpu_cache_append_rotary(None, c or cache16(), b or batch(), layer, rotary() if turn == 0 else turn,
                                              heads, q, q_stride, q_out, out_stride, k, k_stride, v, v_stride))


def tree(c=None, b=None, layer=0, heads=4, scale=1.0, q=6 * A, q_stride=256, visible=None, out=7 * A, out_stride=256):
    return said(lib().xpu_tree_attention8(None, c or cache(), b or batch(), layer, heads, scale, q, q_stride, visible,
                                          out, out_stride, 8 * A, 1 << 40))


def keep(c=None, b=None, kept=6 * A, counts=7 * A, new=8 * A):
    return said(lib().xpu_cache8_keep(None, c or cache(), b or batch(), kept, counts, new))


def copy(c=None, src=(0, 1), dst=(2, 3)):
    s, d = np.array(src, np.uint32), np.array(dst, np.uint32)
    return said(lib().xpu_cache8_copy(None, c or cache(), s.ctypes.data, d.ctypes.data, len(s)))


def sampling(**over):
    return xpu.Sampling(**{**dict(dtype=0, rows=3, vocab=1000, random=A, temperature=2 * A, top_k=3 * A, top_p=4 * A,
                                  min_p=5 * A), **over})


def sample(s=None, logits=6 * A, tokens=7 * A, probability=8 * A, workspace=9 * A, size=1 << 40):
    return said(lib().xpu_sample(None, s or sampling(), logits, tokens, probability, workspace, size))


@pytest.mark.parametrize("call", [append, append16, tree, keep, copy, sample])
def test_right_arguments_get_as_far_as_the_runtime(call):
    rc, text = call()
    assert rc == INVALID and text.endswith("null runtime"), text


def test_page_bytes():
    n = U64()
    for kv, page, d, want in [(1, 16, 64, 1040), (8, 16, 128, 16400), (8, 64, 128, 65568), (3, 256, 64, 49200), (17, 16, 64, 17440)]:
        assert lib().xpu_cache8_page_bytes(cache(kv_heads=kv, page_size=page, head_dim=d), ctypes.byref(n)) == 0
        assert n.value == want
        c = cache(kv_heads=kv, page_size=page, head_dim=d)
        assert c.page_stride % 128 == 0 and 0 <= c.page_stride - want < 128 and c.layer_stride == 8 * c.page_stride
    assert lib().xpu_cache8_page_bytes(None, ctypes.byref(n)) == INVALID
    assert lib().xpu_cache8_page_bytes(cache(), None) == INVALID
    assert lib().xpu_cache8_page_bytes(cache(page_size=24), ctypes.byref(n)) == INVALID


@pytest.mark.parametrize("call", [append, tree, keep, copy])
@pytest.mark.parametrize("over,word", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(head_dim=96), "head_dim"), (dict(head_dim=256), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=512), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=0, page_stride=2080), "page_size"), (dict(layers=0), "positive"), (dict(kv_heads=0), "positive"),
    (dict(n_pages=0), "positive"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(k=A + 8), "aligned"),
    (dict(v=A + 2), "aligned"), (dict(status=A + 2), "aligned"), (dict(page_stride=2088), "multiples of 16"),
    (dict(layer_stride=(1 << 20) + 8), "multiples of 16"), (dict(page_stride=2048), "overlap"),
    (dict(page_stride=2064, layer_stride=8 * 2064 - 16), "overlap"), (dict(layer_stride=0), "overlap"),
    (dict(page_stride=1 << 41), "2^40"), (dict(kv_heads=5000), "4096")])
def test_caches_that_are_refused(call, over, word):
    rc, text = call(c=cache(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


def test_layers_within_pages_are_accepted():
    rc, text = append(c=cache(layer_stride=2064, page_stride=2 * 2064))
    assert rc == INVALID and text.endswith("null runtime"), text
    rc, text = append(c=cache(layer_stride=2064, page_stride=2 * 2064 - 16))
    assert rc == INVALID and "overlap" in text


@pytest.mark.parametrize("call", [append, append16, tree, keep])
@pytest.mark.parametrize("over,word", [
    (dict(rows=1 << 31), "rows"), (dict(n_seqs=1 << 24), "sequences"), (dict(table_pitch=0), "table_pitch"),
    (dict(tables=None), "null"), (dict(starts=None), "null"), (dict(context=None), "null"), (dict(starts=A + 2), "aligned"),
    (dict(tables=A + 1), "aligned"), (dict(context=A + 3), "aligned")])
def test_batches_that_are_refused(call, over, word):
    rc, text = call(b=batch(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("call", [append, append16])
@pytest.mark.parametrize("kwargs,word", [
    (dict(layer=2), "layer"), (dict(k=None), "null k"), (dict(v=None), "null v"), (dict(k=A + 8), "aligned"),
    (dict(k_stride=120), "k_stride"), (dict(v_stride=132), "v_stride"), (dict(k_stride=1 << 24), "k_stride"),
    (dict(heads=65537), "heads"), (dict(q=None), "null q"), (dict(q_out=None), "null q_out"), (dict(q=A + 8), "aligned"),
    (dict(q_stride=248), "q_stride"), (dict(out_stride=260), "q_out_stride"), (dict(q_out=12 * A + 16), "q_out must be q"),
    (dict(q_out=12 * A, out_stride=264), "q_out must be q"), (dict(q_out=6 * A), "k or v"), (dict(q_out=7 * A - 256), "k or v")])
def test_appends_refuse(call, kwargs, word):
    rc, text = call(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("call", [append, append16])
@pytest.mark.parametrize("over,word", [
    (dict(pairs=2), "pairs"), (dict(pairs=-1), "pairs"), (dict(positions=0), "positions"), (dict(dims=0), "dims"),
    (dict(dims=24), "dims"), (dict(dims=80), "dims"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(cos=None), "cos"), (dict(sin=None), "sin"), (dict(cos=A + 8), "aligned"),
    (dict(sin=A + 4), "aligned"), (dict(at=A + 2), "at"), (dict(q_gain=A + 8), "gains"), (dict(k_gain=A + 2), "gains")])
def test_rotations_that_are_refused(call, over, word):
    rc, text = call(turn=rotary(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


def test_without_a_rotation():
    rc, text = append(turn=None, heads=0)
    assert text.endswith("null runtime")
    rc, text = append(turn=None, heads=4)
    assert rc == INVALID and "without rotary" in text
    rc, text = append16(turn=None, heads=0)
    assert rc == INVALID and "null rotary" in text
    for call in (append, append16):  # without heads Q is not looked at
        rc, text = call(heads=0, q=None, q_out=A + 1, q_stride=3)
        assert text.endswith("null runtime")


@pytest.mark.parametrize("call", [append, append16])
def test_queries_in_place_and_beside_the_keys(call):
    assert call(q_out=12 * A)[1].endswith("null runtime")
    # columns [q | k | v] of one buffer, Q in place
    rc, text = call(q=A, q_out=A, k=A + 512, v=A + 768, q_stride=512, out_stride=512, k_stride=512, v_stride=512)
    assert text.endswith("null runtime"), text
    rc, text = call(q=A, q_out=A + 256, k=A + 512, v=A + 768, q_stride=512, out_stride=512, k_stride=512, v_stride=512)
    assert rc == INVALID
    # k reaches into the next row's queries
    rc, text = call(q=A, q_out=A, k=A + 896, v=4 * A, q_stride=512, out_stride=512, k_stride=512)
    assert rc == INVALID and "k or v" in text


@pytest.mark.parametrize("kwargs,word", [
    (dict(layer=2), "layer"), (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=3e38), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(q=None), "null q"), (dict(out=None), "null out"), (dict(q=A + 4), "aligned"), (dict(q_stride=255), "q_stride"),
    (dict(out_stride=248), "out_stride"), (dict(visible=A + 4), "visible"), (dict(out=6 * A), "overlap"),
    (dict(out=6 * A + 256), "overlap"), (dict(b=batch(rows=1 << 25), out=1 << 50), "rows")])
def test_tree_attention8_refuses(kwargs, word):
    rc, text = tree(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("kwargs,word", [
    (dict(kept=None), "null"), (dict(counts=None), "null"), (dict(kept=A + 2), "aligned"), (dict(new=A + 2), "aligned"),
    (dict(new=5 * A), "overlap"), (dict(new=7 * A + 4), "overlap"), (dict(new=4 * A + 8), "overlap"),
    (dict(new=6 * A + 36), "overlap")])
def test_keep_refuses(kwargs, word):
    rc, text = keep(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("src,dst,word", [
    ([8], [0], "does not exist"), ([0], [8], "does not exist"), ([0, 1], [2, 2], "twice"), ([0, 1], [1, 2], "to and from")])
def test_copy_refuses(src, dst, word):
    rc, text = copy(src=src, dst=dst)
    assert rc == INVALID and word in text, text


@pytest.mark.parametrize("over,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1), "vocab"),
    (dict(rows=1 << 23), "rows"), (dict(stride=999), "stride"), (dict(stride=1 << 40), "stride"), (dict(random=None), "random"),
    (dict(random=A + 2), "aligned"), (dict(temperature=A + 1), "aligned"), (dict(top_k=A + 2), "aligned"),
    (dict(top_p=A + 3), "aligned"), (dict(min_p=A + 2), "aligned")])
def test_samplings_that_are_refused(over, word):
    rc, text = sample(sampling(**over))
    assert rc == INVALID and word in text and "runtime" not in text, text


@pytest.mark.parametrize("kwargs,word", [
    (dict(logits=None), "logits"), (dict(logits=6 * A + 1), "logits"), (dict(s=sampling(dtype=2), logits=6 * A + 2), "logits"),
    (dict(tokens=None), "tokens"), (dict(tokens=7 * A + 2), "tokens"), (dict(probability=8 * A + 1), "probability"),
    (dict(probability=7 * A + 8), "overlap"), (dict(tokens=6 * A + 5996), "logits"), (dict(probability=6 * A + 5996), "logits"),
    (dict(tokens=A + 8), "numbers"), (dict(probability=5 * A - 8), "numbers")])
def test_sample_refuses(kwargs, word):
    rc, text = sample(**kwargs)
    assert rc == INVALID and word in text and "runtime" not in text, text


def test_numbers_that_may_be_left_out():
    rc, text = sample(sampling(temperature=None, top_k=None, top_p=None, min_p=None), probability=None)
    assert text.endswith("null runtime")
    assert sample(sampling(rows=0, random=None), logits=None, tokens=None)[1].endswith("null runtime")


def test_null_descriptions():
    n = U64()
    assert lib().xpu_cache8_append(None, None, batch(), 0, rotary(), 0, None, 0, None, 0, A, 128, A, 128) == INVALID
    assert lib().xpu_cache8_append(None, cache(), None, 0, rotary(), 0, None, 0, None, 0, A, 128, A, 128) == INVALID
    assert lib().xpu_cache_append_rotary(None, None, batch(), 0, rotary(), 0, None, 0, None, 0, A, 128, A, 128) == INVALID
    assert lib().xpu_cache8_keep(None, cache(), None, A, A, None) == INVALID
    assert lib().xpu_cache8_copy(None, None, None, None, 0) == INVALID
    assert lib().xpu_tree_attention8_workspace(None, None, batch(), 4, ctypes.byref(n)) == INVALID
    assert lib().xpu_tree_attention8_workspace(None, cache(), batch(), 4, None) == INVALID
    assert lib().xpu_sample(None, None, A, A, None, None, 0) == INVALID
    assert lib().xpu_sample_workspace(None, None, ctypes.byref(n)) == INVALID
    assert lib().xpu_sample_workspace(None, sampling(), None) == INVALID


def test_sizes_that_fields_do_not_hold():
    for make in (lambda: cache(n_pages=1 << 32), lambda: cache(layers=-1), lambda: rotary(dims=1 << 32),
                 lambda: rotary(positions=-1), lambda: sampling(vocab=1 << 32), lambda: sampling(rows=-1),
                 lambda: sampling(stride=1 << 64)):
        with pytest.raises(ValueError, match="fit"):
            make()
