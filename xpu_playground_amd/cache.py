"""Which pages of a paged KV cache are in use (xpu_pages_*, include/xpu_cache.h).

Host only. The pages themselves, and the operations on them, are
xpu_playground_amd.Cache and Runtime.cache_append / cache_keep / cache_copy /
tree_attention.
"""
from __future__ import annotations

import ctypes
import operator
from ctypes import c_uint32, c_void_p

import numpy as np

from . import check, library, page_ids


def _u32(n) -> int:
    n = operator.index(n)
    if not 0 <= n <= 0xFFFFFFFF:
        raise ValueError(f"{n} is no unsigned 32-bit integer")
    return n


class Pages:
    """Counts the holders of n pages."""

    def __init__(self, n_pages: int):
        self.lib = library()
        self.handle, n_pages = None, _u32(n_pages)
        handle = c_void_p()
        check(self.lib.xpu_pages_create(n_pages, ctypes.byref(handle)))
        self.handle, self.n_pages = handle, n_pages

    def __del__(self):
        if getattr(self, "handle", None):
            self.lib.xpu_pages_destroy(self.handle)
            self.handle = None

    @property
    def free(self) -> int:
        v = c_uint32()
        check(self.lib.xpu_pages_free_count(self.handle, ctypes.byref(v)))
        return v.value

    def holders(self, page: int) -> int:
        v = c_uint32()
        check(self.lib.xpu_pages_holders(self.handle, _u32(page), ctypes.byref(v)))
        return v.value

    def take(self, n: int) -> np.ndarray:
        """n free pages, lowest ids first."""
        n = _u32(n)
        out = np.empty(min(n, self.n_pages), np.uint32)  # a larger n is refused before anything is written
        check(self.lib.xpu_pages_take(self.handle, n, out.ctypes.data))
        return out

    def share(self, ids) -> None:
        """One holder more for each: a forked sequence holds the same pages."""
        a = page_ids(ids)
        check(self.lib.xpu_pages_share(self.handle, a.ctypes.data, len(a)))

    def release(self, ids) -> None:
        """One holder less for each; pages without holders are free."""
        a = page_ids(ids)
        check(self.lib.xpu_pages_release(self.handle, a.ctypes.data, len(a)))

    def own(self, ids) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """(ids, src, dst): the pages as the caller's alone, and the copies
        src[i] -> dst[i] that Runtime.cache_copy has to make first."""
        a = page_ids(ids).copy()
        src, dst, n = np.empty(len(a), np.uint32), np.empty(len(a), np.uint32), c_uint32()
        check(self.lib.xpu_pages_own(self.handle, a.ctypes.data, len(a), src.ctypes.data, dst.ctypes.data,
                                     ctypes.byref(n)))
        return a, src[: n.value].copy(), dst[: n.value].copy()

    def compact(self) -> tuple[np.ndarray, np.ndarray]:
        """(src, dst): moves that leave the pages in use at the lowest ids."""
        src, dst, n = np.empty(self.n_pages, np.uint32), np.empty(self.n_pages, np.uint32), c_uint32()
        check(self.lib.xpu_pages_compact(self.handle, src.ctypes.data, dst.ctypes.data, ctypes.byref(n)))
        return src[: n.value].copy(), dst[: n.value].copy()


def renumber(src, dst, ids) -> np.ndarray:
    """A table's ids after the moves of Pages.compact."""
    s, d, a = page_ids(src), page_ids(dst), page_ids(ids).copy()
    if len(s) != len(d):
        raise ValueError("src and dst must be of one length")
    check(library().xpu_pages_renumber(s.ctypes.data, d.ctypes.data, len(s), a.ctypes.data, len(a)))
    return a
