"""Arguments of the paged cache's calls at the border of what is refused, on
the host: a null runtime is the last thing that a call looks at."""
import numpy as np
import pytest

import xpu_playground_amd as xpu
from test_cache_refusals import A, INVALID, batch, packed, prompt, tree
from xpu_playground_amd.cache import Pages

Q = 6 * A  # 10 rows of 4 heads x 64: 512 bytes each


@pytest.mark.parametrize("stride,columns", [  # elements
    (512, 256), (512, -256), (528, 256), (528, 264), (528, -264), (528, -272), (1024, 256), (1024, 768), (1024, -512)])
def test_out_may_be_other_columns_of_the_buffer_that_holds_q(stride, columns):
    """Rows the same stride apart that share no byte do not overlap, on either
    side of q and whole rows away from it too."""
    for rows_away in (0, 1, -1, 3):
        at = Q + 2 * columns + 2 * stride * rows_away
        for rc, text in (tree(q_stride=stride, out=at, out_stride=stride),
                         prompt(packed(q_stride=stride, out_stride=stride), q=Q, out=at)):
            assert rc == INVALID and text.endswith("null runtime"), text


@pytest.mark.parametrize("stride", [512, 528])
@pytest.mark.parametrize("columns", [8, 248, -8, -248, 0, 280])
def test_out_that_shares_columns_with_q_is_refused(stride, columns):
    for rows_away in (0, 1, -2, 9 if columns < 256 else 8):  # behind q's last row there is none to share with
        at = Q + 2 * columns + 2 * stride * rows_away
        rc, text = tree(q_stride=stride, out=at, out_stride=stride)
        assert rc == INVALID and "overlap" in text, text
        if columns or rows_away:
            rc, text = prompt(packed(q_stride=stride, out_stride=stride), q=Q, out=at)
            assert rc == INVALID and "overlap" in text, text
    # past q's last row, or before its first, there is nothing to share
    for rows_away in (10, -10):
        rc, text = tree(q_stride=stride, out=Q + 2 * stride * rows_away, out_stride=stride)
        assert text.endswith("null runtime"), text


def test_other_strides_that_cross_are_refused():
    rc, text = tree(q_stride=512, out=Q + 512, out_stride=520)
    assert rc == INVALID and "overlap" in text
    rc, text = tree(b=batch(rows=1), q_stride=512, out=Q + 512, out_stride=520)
    assert text.endswith("null runtime"), text


WIDE = [1 << 32, (1 << 32) + 4, -1, -(1 << 32)]


@pytest.mark.parametrize("n", WIDE)
def test_page_counts_that_32_bits_do_not_hold(n):
    """Cut to 32 bits, 2^32 would be nothing, and take() would return what its
    array held before."""
    with pytest.raises(ValueError, match="32"):
        Pages(n)
    p = Pages(8)
    p.take(3)
    for call in (p.take, p.holders):
        with pytest.raises(ValueError, match="32"):
            call(n)
    assert p.free == 5 and [p.holders(i) for i in range(4)] == [1, 1, 1, 0]


def test_page_counts_that_are_no_integers():
    for n in (1.0, "1", None):
        with pytest.raises(TypeError):
            Pages(n)
        p = Pages(2)
        with pytest.raises(TypeError):
            p.take(n)
    assert list(Pages(np.int64(3)).take(np.uint8(2))) == [0, 1]


@pytest.mark.parametrize("n", WIDE)
def test_descriptions_that_their_fields_do_not_hold(n):
    """A size past 32 bits is refused and not taken for what is left of it: a
    Packed of 2^32 rows would be one of none, which does nothing."""
    for make in (lambda: xpu.Packed(0, 4, 2, 64, 2, n, A), lambda: xpu.Packed(0, 4, 2, 64, n, 8, A),
                 lambda: xpu.Packed(0, 4, 2, 64, 2, 8, A, k_rows=n), lambda: xpu.Batch(n, 4, 4, A, A, A),
                 lambda: xpu.Batch(2, n, 4, A, A, A), lambda: xpu.Batch(2, 4, n, A, A, A),
                 lambda: xpu.Batch(n_seqs=2, rows=4, table_pitch=n), lambda: xpu.Cache(0, n, 2, 64, 16, 8, A, A),
                 lambda: xpu.Cache(0, 2, 2, 64, 16, n, A, A, layer_stride=1 << 20),
                 lambda: xpu.Cache(0, 2, 2, 64, 16, 8, A, A, page_stride=(1 << 64) + 2048),
                 lambda: xpu.Packed(0, 4, 2, 64, 2, 8, A, q_stride=-256)):
        with pytest.raises(ValueError, match="bits"):
            make()


def test_descriptions_hold_what_they_were_given():
    b = xpu.Batch(1, (1 << 31) - 1, np.uint32(7), A, A, None)
    assert (b.n_seqs, b.rows, b.table_pitch, b.tables, b.context) == (1, (1 << 31) - 1, 7, A, None)
    b = xpu.Batch(rows=5)
    assert (b.n_seqs, b.rows, b.starts) == (0, 5, None)
    c = xpu.Cache(-1, 4, 2, 64, 16, 0xFFFFFFFF, A, A, layer_stride=(1 << 64) - 8)
    assert (c.dtype, c.n_pages, c.layer_stride, c.page_stride) == (-1, 0xFFFFFFFF, (1 << 64) - 8, 2048)
    p = xpu.Packed(1, 4, 2, 64, 3, 0xFFFFFFFF, A, scale=2)
    assert (p.q_rows, p.k_rows, p.scale, p.q_stride) == (0xFFFFFFFF, 0xFFFFFFFF, 2.0, 256)


@pytest.mark.parametrize("ids", [b"\x01\0\0\0", bytearray(8), b""])
def test_page_ids_are_no_bytes(ids):
    """Four bytes were one id: what a program stores as bytes has to say how."""
    with pytest.raises(ValueError, match="page ids"):
        xpu.page_ids(ids)
    p = Pages(4)
    p.take(2)
    with pytest.raises(ValueError, match="page ids"):
        p.release(ids)
    assert p.free == 2
    assert list(xpu.page_ids(memoryview(np.array([3, 0xFFFFFFFF], np.uint32)))) == [3, 0xFFFFFFFF]
