"""ctypes bindings to the gfx950 hot-path library (build/libxpu_playground.so).

The C ABI is declared in include/xpu_runtime.h, include/xpu_kernels.h,
include/xpu_qwen3.h, include/xpu_cache.h, include/xpu_cache8.h and
include/xpu_sample.h. Every compute call runs the HIP kernels of
build/xpu_kernels.hsaco; there is no CPU fallback: if the library or the code
object is missing, or no gfx950 device is visible, the calls raise.
"""
from __future__ import annotations

import ctypes
import os
import struct
import weakref
from array import array
from ctypes import POINTER, c_char_p, c_double, c_float, c_int, c_size_t, c_uint32, c_uint64, c_void_p

PACKAGE_DIR = os.path.dirname(os.path.abspath(__file__))
BUILD_DIR = os.path.join(PACKAGE_DIR, "build")
LIBRARY_PATH = os.path.join(BUILD_DIR, "libxpu_playground.so")
MODULE_PATH = os.path.join(BUILD_DIR, "xpu_kernels.hsaco")

BF16 = 0
FP16 = 1
FP32 = 2  # of logits (Sampling)

HALVES = 0  # pairs of a rotation (Rotary)
ADJACENT = 1

SAMPLE_NONE = 0xFFFFFFFF  # the token of a row without an answer (Runtime.sample)

XPU_OK = 0


class XpuError(RuntimeError):
    """A C-ABI call returned a nonzero status."""

    def __init__(self, code: int, message: str):
        super().__init__(f"[xpu error {code}] {message}")
        self.code = code


class KernelArg(ctypes.Structure):
    _fields_ = [("size", c_size_t), ("value", c_void_p)]


class Qwen3Config(ctypes.Structure):
    """xpu_qwen3_config (include/xpu_qwen3.h)."""

    _fields_ = [
        ("hidden", c_uint32),
        ("intermediate", c_uint32),
        ("layers", c_uint32),
        ("heads", c_uint32),
        ("kv_heads", c_uint32),
        ("head_dim", c_uint32),
        ("vocab", c_uint32),
        ("rms_eps", c_float),
        ("rope_theta", c_double),
        ("tied", c_uint32),
    ]


def page_ids(ids):
    """Page ids as the C calls take them: one-dimensional uint32."""
    import numpy as np

    if not isinstance(ids, np.ndarray):
        try:
            if isinstance(ids, (bytes, bytearray)):  # array takes these for its memory
                raise TypeError("bytes")
            ids = array("I", ids)
            ids = np.frombuffer(ids, np.uint32) if ids else np.empty(0, np.uint32)
        except (TypeError, OverflowError) as e:
            raise ValueError(f"page ids must be a list of unsigned 32-bit integers: {e}") from None
    elif ids.dtype != np.uint32:
        if ids.size and (ids.dtype.kind not in "iu" or int(ids.min()) < 0 or int(ids.max()) > 0xFFFFFFFF):
            raise ValueError("page ids must be unsigned 32-bit integers")
    if ids.ndim != 1:
        raise ValueError("page ids must be one-dimensional")
    return np.ascontiguousarray(ids, dtype=np.uint32)


def _fit(what: str, layout: struct.Struct, *values) -> None:
    """Raises for integers that their fields do not hold; ctypes would cut them."""
    try:
        layout.pack(*values)
    except struct.error as e:
        raise ValueError(f"{what}: sizes have to fit the 32 or 64 bits of their fields: {e}") from None


class Cache(ctypes.Structure):
    """xpu_cache (include/xpu_cache.h): the pages of a KV cache. k and v are
    device addresses; without strides the pools are [layers][n_pages]
    [kv_heads][page_size][head_dim]."""

    _fields_ = [
        ("dtype", c_int),
        ("layers", c_uint32),
        ("kv_heads", c_uint32),
        ("head_dim", c_uint32),
        ("page_size", c_uint32),
        ("n_pages", c_uint32),
        ("layer_stride", c_uint64),
        ("page_stride", c_uint64),
        ("k", c_void_p),
        ("v", c_void_p),
        ("status", c_void_p),
    ]
    _sizes = struct.Struct("i5I2Q")

    def __init__(self, dtype, layers, kv_heads, head_dim, page_size, n_pages, k=None, v=None, status=None,
                 layer_stride=None, page_stride=None):
        page = kv_heads * page_size * head_dim
        sizes = (dtype, layers, kv_heads, head_dim, page_size, n_pages,
                 n_pages * page if layer_stride is None else layer_stride, page if page_stride is None else page_stride)
        _fit("Cache", self._sizes, *sizes)
        super().__init__(*sizes, k, v, status)


class Cache8(ctypes.Structure):
    """xpu_cache8 (include/xpu_cache8.h): the pages of a KV cache in 8 bits. k
    and v are device addresses, strides are in bytes; without strides the pools
    are [layers][n_pages][page_bytes], page_bytes being a page's codes and
    scales, rounded up to 128."""

    _fields_ = Cache._fields_
    _sizes = Cache._sizes

    def __init__(self, dtype, layers, kv_heads, head_dim, page_size, n_pages, k=None, v=None, status=None,
                 layer_stride=None, page_stride=None):
        if page_stride is None:
            page_stride = -(-(kv_heads * page_size * head_dim + kv_heads * (page_size // 16)) // 128) * 128
        sizes = (dtype, layers, kv_heads, head_dim, page_size, n_pages,
                 n_pages * page_stride if layer_stride is None else layer_stride, page_stride)
        _fit("Cache8", self._sizes, *sizes)
        super().__init__(*sizes, k, v, status)


class Rotary(ctypes.Structure):
    """xpu_rotary (include/xpu_cache.h): how new Q and K rows are turned. cos
    and sin are device addresses of FP32 [positions][dims / 2], at of uint32
    per row, the gains of head_dim elements of the cache's type."""

    _fields_ = [
        ("positions", c_uint32),
        ("dims", c_uint32),
        ("pairs", c_int),
        ("eps", c_float),
        ("cos", c_void_p),
        ("sin", c_void_p),
        ("at", c_void_p),
        ("q_gain", c_void_p),
        ("k_gain", c_void_p),
    ]
    _sizes = struct.Struct("2Ii")

    def __init__(self, positions, dims, cos=None, sin=None, pairs=HALVES, at=None, q_gain=None, k_gain=None, eps=1e-6):
        _fit("Rotary", self._sizes, positions, dims, pairs)
        super().__init__(positions, dims, pairs, eps, cos, sin, at, q_gain, k_gain)


class Sampling(ctypes.Structure):
    """xpu_sampling (include/xpu_sample.h): how the rows' tokens are drawn.
    random, temperature, top_k, top_p and min_p are device addresses, a number
    per row; without a stride the rows are dense."""

    _fields_ = [
        ("dtype", c_int),
        ("rows", c_uint32),
        ("vocab", c_uint32),
        ("stride", c_uint64),
        ("temperature", c_void_p),
        ("top_k", c_void_p),
        ("top_p", c_void_p),
        ("min_p", c_void_p),
        ("random", c_void_p),
    ]
    _sizes = struct.Struct("i2IQ")

    def __init__(self, dtype, rows, vocab, random=None, temperature=None, top_k=None, top_p=None, min_p=None, stride=None):
        sizes = (dtype, rows, vocab, vocab if stride is None else stride)
        _fit("Sampling", self._sizes, *sizes)
        super().__init__(*sizes, temperature, top_k, top_p, min_p, random)


class Batch(ctypes.Structure):
    """xpu_batch (include/xpu_cache.h): sequences with new rows; tables,
    starts and context are device addresses of uint32."""

    _fields_ = [
        ("n_seqs", c_uint32),
        ("rows", c_uint32),
        ("table_pitch", c_uint32),
        ("tables", c_void_p),
        ("starts", c_void_p),
        ("context", c_void_p),
    ]
    _sizes = struct.Struct("3I")

    def __init__(self, n_seqs=0, rows=0, table_pitch=0, tables=None, starts=None, context=None):
        _fit("Batch", self._sizes, n_seqs, rows, table_pitch)
        super().__init__(n_seqs, rows, table_pitch, tables, starts, context)


class Packed(ctypes.Structure):
    """xpu_packed (include/xpu_cache.h): packed prompts; q_starts and k_starts
    are device addresses of n_seqs + 1 uint32. Without strides the rows are
    dense, without k_starts the keys are the queries' rows, and the scale is
    head_dim ** -0.5."""

    _fields_ = [
        ("dtype", c_int),
        ("heads", c_uint32),
        ("kv_heads", c_uint32),
        ("head_dim", c_uint32),
        ("n_seqs", c_uint32),
        ("q_rows", c_uint32),
        ("k_rows", c_uint32),
        ("scale", c_float),
        ("q_starts", c_void_p),
        ("k_starts", c_void_p),
        ("q_stride", c_uint64),
        ("k_stride", c_uint64),
        ("v_stride", c_uint64),
        ("out_stride", c_uint64),
    ]
    _sizes = struct.Struct("i6I4Q")

    def __init__(self, dtype, heads, kv_heads, head_dim, n_seqs, q_rows, q_starts, k_rows=None, k_starts=None,
                 scale=None, q_stride=None, k_stride=None, v_stride=None, out_stride=None):
        def dense(stride, n):
            return n * head_dim if stride is None else stride

        sizes = (dtype, heads, kv_heads, head_dim, n_seqs, q_rows, q_rows if k_rows is None else k_rows)
        strides = dense(q_stride, heads), dense(k_stride, kv_heads), dense(v_stride, kv_heads), dense(out_stride, heads)
        _fit("Packed", self._sizes, *sizes, *strides)
        super().__init__(*sizes, head_dim ** -0.5 if scale is None else scale, q_starts, k_starts, *strides)


_lib = None


def _declare(lib):
    sig = {
        "xpu_last_error": (c_char_p, []),
        "xpu_rt_create": (c_int, [c_char_p, c_int, POINTER(c_void_p)]),
        "xpu_rt_destroy": (None, [c_void_p]),
        "xpu_rt_device_name": (c_int, [c_void_p, c_char_p, c_size_t]),
        "xpu_rt_device_arch": (c_int, [c_void_p, c_char_p, c_size_t]),
        "xpu_rt_device_memory": (c_int, [c_void_p, POINTER(c_uint64)]),
        "xpu_rt_compute_units": (c_int, [c_void_p, POINTER(c_uint32)]),
        "xpu_rt_require_device_and_memory": (c_int, [c_void_p, c_uint64]),
        "xpu_rt_alloc": (c_int, [c_void_p, c_uint64, c_uint64, POINTER(c_void_p)]),
        "xpu_rt_free": (c_int, [c_void_p, c_void_p]),
        "xpu_rt_copy_to_device": (c_int, [c_void_p, c_void_p, c_void_p, c_size_t]),
        "xpu_rt_copy_from_device": (c_int, [c_void_p, c_void_p, c_void_p, c_size_t]),
        "xpu_rt_copy_device": (c_int, [c_void_p, c_void_p, c_void_p, c_size_t]),
        "xpu_rt_memset": (c_int, [c_void_p, c_void_p, c_int, c_size_t]),
        "xpu_rt_launch": (c_int, [c_void_p, c_char_p, c_uint32, POINTER(KernelArg), c_uint32]),
        "xpu_rt_launch_grid": (
            c_int,
            [c_void_p, c_char_p, c_uint32, c_uint32, c_uint32, c_uint32, POINTER(KernelArg), c_uint32],
        ),
        "xpu_module_kernel_names": (c_int, [c_char_p, c_char_p, c_size_t]),
        "xpu_rt_kernel_count": (c_int, [c_void_p, POINTER(c_uint32)]),
        "xpu_rt_module_global": (c_int, [c_void_p, c_char_p, POINTER(c_void_p), POINTER(c_uint64)]),
        "xpu_rt_kernel_name": (c_int, [c_void_p, c_uint32, c_char_p, c_size_t]),
        "xpu_rt_synchronize": (c_int, [c_void_p]),
        "xpu_rt_stream": (c_void_p, [c_void_p]),
        "xpu_rt_event_create": (c_int, [c_void_p, POINTER(c_void_p)]),
        "xpu_rt_event_record": (c_int, [c_void_p, c_void_p]),
        "xpu_rt_event_elapsed_ms": (c_int, [c_void_p, c_void_p, POINTER(c_float)]),
        "xpu_rt_event_destroy": (c_int, [c_void_p]),
        "xpu_rt_capture_begin": (c_int, [c_void_p]),
        "xpu_rt_capture_end": (c_int, [c_void_p, POINTER(c_void_p)]),
        "xpu_rt_graph_launch": (c_int, [c_void_p, c_void_p]),
        "xpu_rt_graph_destroy": (c_int, [c_void_p]),
        "xpu_gemv": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_uint32, c_uint32, c_uint64]),
        "xpu_fill_uniform": (c_int, [c_void_p, c_int, c_void_p, c_uint64, c_uint64]),
        "xpu_fill_reference_gemv": (
            c_int,
            [c_void_p, c_int, c_void_p, c_void_p, c_uint32, c_uint32, c_uint32],
        ),
    }
    optional = {
        "xpu_gemm": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_uint32, c_uint32, c_uint32]),
        "xpu_gemm_noalloc": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_uint32, c_uint32, c_uint32]),
        "xpu_gemm_tile": (c_int, [c_void_p, c_uint32, c_uint32, POINTER(c_uint32), POINTER(c_uint32)]),
        "xpu_qwen3_preset": (c_int, [c_char_p, POINTER(Qwen3Config)]),
        "xpu_qwen3_fill_tensor": (
            c_int,
            [POINTER(Qwen3Config), c_uint64, c_float, c_int, c_uint32, c_void_p, c_uint64],
        ),
        "xpu_qwen3_rope_tables": (c_int, [c_void_p, c_void_p, c_uint32, c_uint32, c_double]),
        "xpu_qwen3_create": (
            c_int,
            [c_void_p, POINTER(Qwen3Config), c_uint32, c_uint64, c_float, POINTER(c_void_p)],
        ),
        "xpu_qwen3_destroy": (None, [c_void_p]),
        "xpu_qwen3_set_mode": (c_int, [c_void_p, c_int]),
        "xpu_qwen3_set_prefill": (c_int, [c_void_p, c_int]),
        "xpu_qwen3_set_attention_split": (c_int, [c_void_p, c_uint32]),
        "xpu_qwen3_set_sampling": (c_int, [c_void_p, c_float, c_uint32, c_float, c_float, c_uint64]),
        "xpu_qwen3_decode": (c_int, [c_void_p, c_uint32, c_uint32, POINTER(c_uint32)]),
        "xpu_qwen3_logits": (c_int, [c_void_p, c_void_p, c_uint64]),
        "xpu_qwen3_hidden": (c_int, [c_void_p, c_void_p, c_uint64]),
        "xpu_qwen3_generate": (
            c_int,
            [
                c_void_p,
                POINTER(c_uint32),
                c_uint32,
                c_uint32,
                c_int,
                POINTER(c_uint32),
                POINTER(c_uint32),
                POINTER(c_double),
                POINTER(c_double),
            ],
        ),
        "xpu_qwen3_read_config": (c_int, [c_char_p, POINTER(Qwen3Config)]),
        "xpu_qwen3_validate_checkpoint": (c_int, [c_char_p, POINTER(Qwen3Config)]),
        "xpu_qwen3_get_config": (c_int, [c_void_p, POINTER(Qwen3Config)]),
        "xpu_qwen3_create_from_checkpoint": (c_int, [c_void_p, c_char_p, c_uint32, POINTER(c_void_p)]),
        "xpu_synth_tokens": (c_int, [c_void_p, c_uint64, c_uint64, c_uint32]),
        "run_gemv": (c_int, [c_int, POINTER(c_char_p)]),
        "run_gemm": (c_int, [c_int, POINTER(c_char_p)]),
        "xpu_cache_append": (
            c_int,
            [c_void_p, POINTER(Cache), POINTER(Batch), c_uint32, c_void_p, c_uint64, c_void_p, c_uint64],
        ),
        "xpu_tree_attention": (
            c_int,
            [
                c_void_p,
                POINTER(Cache),
                POINTER(Batch),
                c_uint32,
                c_uint32,
                c_float,
                c_void_p,
                c_uint64,
                c_void_p,
                c_void_p,
                c_uint64,
                c_void_p,
                c_uint64,
            ],
        ),
        "xpu_tree_attention_workspace": (
            c_int,
            [c_void_p, POINTER(Cache), POINTER(Batch), c_uint32, POINTER(c_uint64)],
        ),
        "xpu_cache_keep": (c_int, [c_void_p, POINTER(Cache), POINTER(Batch), c_void_p, c_void_p, c_void_p]),
        "xpu_cache_copy": (c_int, [c_void_p, POINTER(Cache), c_void_p, c_void_p, c_uint32]),
        "xpu_cache_append_rotary": (
            c_int,
            [c_void_p, POINTER(Cache), POINTER(Batch), c_uint32, POINTER(Rotary), c_uint32] + [c_void_p, c_uint64] * 4,
        ),
        "xpu_cache8_page_bytes": (c_int, [POINTER(Cache8), POINTER(c_uint64)]),
        "xpu_cache8_append": (
            c_int,
            [c_void_p, POINTER(Cache8), POINTER(Batch), c_uint32, POINTER(Rotary), c_uint32] + [c_void_p, c_uint64] * 4,
        ),
        "xpu_tree_attention8": (
            c_int,
            [c_void_p, POINTER(Cache8), POINTER(Batch), c_uint32, c_uint32, c_float, c_void_p, c_uint64, c_void_p]
            + [c_void_p, c_uint64] * 2,
        ),
        "xpu_tree_attention8_workspace": (
            c_int,
            [c_void_p, POINTER(Cache8), POINTER(Batch), c_uint32, POINTER(c_uint64)],
        ),
        "xpu_cache8_keep": (c_int, [c_void_p, POINTER(Cache8), POINTER(Batch), c_void_p, c_void_p, c_void_p]),
        "xpu_cache8_copy": (c_int, [c_void_p, POINTER(Cache8), c_void_p, c_void_p, c_uint32]),
        "xpu_sample": (
            c_int,
            [c_void_p, POINTER(Sampling), c_void_p, c_void_p, c_void_p, c_void_p, c_uint64],
        ),
        "xpu_sample_workspace": (c_int, [c_void_p, POINTER(Sampling), POINTER(c_uint64)]),
        "xpu_prompt_attention": (c_int, [c_void_p, POINTER(Packed), c_void_p, c_void_p, c_void_p, c_void_p]),
        "xpu_pages_create": (c_int, [c_uint32, POINTER(c_void_p)]),
        "xpu_pages_destroy": (None, [c_void_p]),
        "xpu_pages_free_count": (c_int, [c_void_p, POINTER(c_uint32)]),
        "xpu_pages_holders": (c_int, [c_void_p, c_uint32, POINTER(c_uint32)]),
        "xpu_pages_take": (c_int, [c_void_p, c_uint32, c_void_p]),
        "xpu_pages_share": (c_int, [c_void_p, c_void_p, c_uint32]),
        "xpu_pages_release": (c_int, [c_void_p, c_void_p, c_uint32]),
        "xpu_pages_own": (c_int, [c_void_p, c_void_p, c_uint32, c_void_p, c_void_p, POINTER(c_uint32)]),
        "xpu_pages_compact": (c_int, [c_void_p, c_void_p, c_void_p, POINTER(c_uint32)]),
        "xpu_pages_renumber": (c_int, [c_void_p, c_void_p, c_uint32, c_void_p, c_uint32]),
        "xpu_peak_mfma": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_uint32, c_uint32]),
        "xpu_peak_read": (c_int, [c_void_p, c_void_p, c_uint64, c_void_p, c_uint32]),
        "run_peak_compute": (c_int, [c_int, POINTER(c_char_p)]),
        "run_peak_mem": (c_int, [c_int, POINTER(c_char_p)]),
        "run_qwen3": (c_int, [c_int, POINTER(c_char_p)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    for name, (res, args) in optional.items():
        fn = getattr(lib, name, None)
        if fn is not None:
            fn.restype = res
            fn.argtypes = args
    return lib


def library():
    """Load build/libxpu_playground.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIBRARY_PATH):
            raise RuntimeError(
                f"{LIBRARY_PATH} is missing: run __graft_entry__.build() (the HIP path has no fallback)"
            )
        _lib = _declare(ctypes.CDLL(LIBRARY_PATH))
    return _lib


def check(code: int) -> None:
    if code != XPU_OK:
        raise XpuError(code, library().xpu_last_error().decode(errors="replace"))


def module_kernel_names(path: str | None = None) -> list[str]:
    buf = ctypes.create_string_buffer(1 << 16)
    check(library().xpu_module_kernel_names(path.encode() if path else None, buf, len(buf)))
    return buf.value.decode().split()


class Args:
    """Builds an xpu_kernel_arg array and keeps the argument values alive."""

    def __init__(self):
        self._values = []
        self._sizes = []

    def ptr(self, p):
        self._values.append(c_void_p(p if isinstance(p, int) or p is None else p.value))
        self._sizes.append(8)
        return self

    def u32(self, v):
        self._values.append(c_uint32(v))
        self._sizes.append(4)
        return self

    def u64(self, v):
        self._values.append(c_uint64(v))
        self._sizes.append(8)
        return self

    def f32(self, v):
        self._values.append(c_float(v))
        self._sizes.append(4)
        return self

    def array(self):
        arr = (KernelArg * len(self._values))()
        for i, (v, s) in enumerate(zip(self._values, self._sizes)):
            arr[i].size = s
            arr[i].value = ctypes.cast(ctypes.pointer(v), c_void_p)
        return arr, len(self._values)


class Runtime:
    """Owner of one gfx950 device, stream, code object and allocations."""

    def __init__(self, module_path: str | None = None, device: int = -1):
        self.lib = library()
        self._dependents = weakref.WeakSet()
        handle = c_void_p()
        check(self.lib.xpu_rt_create(module_path.encode() if module_path else None, device, ctypes.byref(handle)))
        self.handle = handle

    def add_dependent(self, obj) -> None:
        """Register an object holding allocations of this runtime (an engine);
        close() closes it first, so it never frees through a destroyed
        runtime."""
        self._dependents.add(obj)

    def close(self):
        if self.handle:
            for dep in list(self._dependents):
                dep.close()
            self.lib.xpu_rt_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _string(self, fn):
        buf = ctypes.create_string_buffer(256)
        check(fn(self.handle, buf, len(buf)))
        return buf.value.decode()

    @property
    def device_name(self) -> str:
        return self._string(self.lib.xpu_rt_device_name)

    @property
    def arch(self) -> str:
        return self._string(self.lib.xpu_rt_device_arch)

    @property
    def compute_units(self) -> int:
        v = c_uint32()
        check(self.lib.xpu_rt_compute_units(self.handle, ctypes.byref(v)))
        return v.value

    @property
    def device_memory(self) -> int:
        v = c_uint64()
        check(self.lib.xpu_rt_device_memory(self.handle, ctypes.byref(v)))
        return v.value

    def kernel_names(self) -> list[str]:
        n = c_uint32()
        check(self.lib.xpu_rt_kernel_count(self.handle, ctypes.byref(n)))
        out = []
        for i in range(n.value):
            buf = ctypes.create_string_buffer(256)
            check(self.lib.xpu_rt_kernel_name(self.handle, i, buf, len(buf)))
            out.append(buf.value.decode())
        return out

    def alloc(self, nbytes: int, alignment: int = 256) -> int:
        p = c_void_p()
        check(self.lib.xpu_rt_alloc(self.handle, nbytes, alignment, ctypes.byref(p)))
        return p.value

    def free(self, ptr: int) -> None:
        check(self.lib.xpu_rt_free(self.handle, c_void_p(ptr)))

    def upload(self, array) -> int:
        """Allocate device memory and copy a contiguous numpy array into it."""
        import numpy as np

        a = np.ascontiguousarray(array)
        ptr = self.alloc(max(a.nbytes, 1))
        check(self.lib.xpu_rt_copy_to_device(self.handle, c_void_p(ptr), a.ctypes.data_as(c_void_p), a.nbytes))
        return ptr

    def copy_to(self, ptr: int, array) -> None:
        import numpy as np

        a = np.ascontiguousarray(array)
        check(self.lib.xpu_rt_copy_to_device(self.handle, c_void_p(ptr), a.ctypes.data_as(c_void_p), a.nbytes))

    def download(self, ptr: int, count: int, dtype) -> "np.ndarray":  # noqa: F821
        import numpy as np

        out = np.empty(count, dtype=dtype)
        check(self.lib.xpu_rt_copy_from_device(self.handle, out.ctypes.data_as(c_void_p), c_void_p(ptr), out.nbytes))
        return out

    def memset(self, ptr: int, value: int, nbytes: int) -> None:
        check(self.lib.xpu_rt_memset(self.handle, c_void_p(ptr), value, nbytes))

    def synchronize(self) -> None:
        check(self.lib.xpu_rt_synchronize(self.handle))

    def launch(self, fragment: str, work_items: int, args: Args) -> None:
        """Blocking launch with the reference's work-item convention."""
        arr, n = args.array()
        check(self.lib.xpu_rt_launch(self.handle, fragment.encode(), work_items, arr, n))

    def launch_grid(self, name: str, grid: int, block: int, shared: int, args: Args, grid_y: int = 1) -> None:
        arr, n = args.array()
        check(self.lib.xpu_rt_launch_grid(self.handle, name.encode(), grid, grid_y, block, shared, arr, n))

    def event(self) -> "Event":
        return Event(self)

    # ---- hot-path entry points
    def gemv(self, dtype: int, a: int, x: int, y: int, m: int, k: int, lda: int | None = None) -> None:
        check(self.lib.xpu_gemv(self.handle, dtype, c_void_p(a), c_void_p(x), c_void_p(y), m, k, lda or k))

    def gemm(self, dtype: int, a: int, b: int, c: int, m: int, n: int, k: int) -> None:
        check(self.lib.xpu_gemm(self.handle, dtype, c_void_p(a), c_void_p(b), c_void_p(c), m, n, k))

    def gemm_tile(self, m: int, n: int) -> tuple[int, int]:
        """The block tile (rows, cols) that gemm() uses for an m x n output."""
        rows, cols = ctypes.c_uint32(), ctypes.c_uint32()
        check(self.lib.xpu_gemm_tile(self.handle, m, n, ctypes.byref(rows), ctypes.byref(cols)))
        return rows.value, cols.value

    # ---- the paged cache and the attention over it (include/xpu_cache.h);
    # row operands are device addresses, dense rows without a stride
    def cache_append(self, cache: Cache, batch: Batch, layer: int, k: int, v: int, k_stride: int | None = None,
                     v_stride: int | None = None) -> None:
        dense = cache.kv_heads * cache.head_dim
        check(self.lib.xpu_cache_append(self.handle, cache, batch, layer, k, dense if k_stride is None else k_stride,
                                        v, dense if v_stride is None else v_stride))

    def tree_attention_workspace(self, cache: Cache, batch: Batch, heads: int) -> int:
        """Bytes of workspace that tree_attention needs for these shapes."""
        v = c_uint64()
        check(self.lib.xpu_tree_attention_workspace(self.handle, cache, batch, heads, ctypes.byref(v)))
        return v.value

    def tree_attention(self, cache: Cache, batch: Batch, layer: int, heads: int, q: int, out: int,
                       workspace: int | None, workspace_bytes: int, visible: int | None = None,
                       scale: float | None = None, q_stride: int | None = None, out_stride: int | None = None) -> None:
        dense = heads * cache.head_dim
        check(self.lib.xpu_tree_attention(self.handle, cache, batch, layer, heads,
                                          cache.head_dim ** -0.5 if scale is None else scale, q,
                                          dense if q_stride is None else q_stride, visible, out,
                                          dense if out_stride is None else out_stride, workspace, workspace_bytes))

    def cache_keep(self, cache: Cache, batch: Batch, kept: int, counts: int, new_context: int | None = None) -> None:
        check(self.lib.xpu_cache_keep(self.handle, cache, batch, kept, counts, new_context))

    def cache_copy(self, cache: Cache, src, dst) -> None:
        """src, dst: page ids on the host (arrays or lists of one length)."""
        s, d = page_ids(src), page_ids(dst)
        if len(s) != len(d):
            raise ValueError("src and dst must be of one length")
        check(self.lib.xpu_cache_copy(self.handle, cache, s.ctypes.data, d.ctypes.data, len(s)))

    def cache_append_rotary(self, cache: Cache, batch: Batch, layer: int, k: int, v: int, rotary: Rotary,
                            heads: int = 0, q: int | None = None, q_out: int | None = None,
                            k_stride: int | None = None, v_stride: int | None = None, q_stride: int | None = None,
                            out_stride: int | None = None) -> None:
        """cache_append with K, and with `heads` Q on its way to q_out, turned."""
        self._append_turned(self.lib.xpu_cache_append_rotary, cache, batch, layer, k, v, rotary, heads, q, q_out,
                            k_stride, v_stride, q_stride, out_stride)

    def _append_turned(self, call, cache, batch, layer, k, v, rotary, heads, q, q_out, k_stride, v_stride, q_stride,
                       out_stride):
        dense, q_dense = cache.kv_heads * cache.head_dim, heads * cache.head_dim
        check(call(self.handle, cache, batch, layer, rotary, heads, q, q_dense if q_stride is None else q_stride, q_out,
                   q_dense if out_stride is None else out_stride, k, dense if k_stride is None else k_stride, v,
                   dense if v_stride is None else v_stride))

    def cache8_page_bytes(self, cache: Cache8) -> int:
        """Bytes of a page, codes and scales."""
        v = c_uint64()
        check(self.lib.xpu_cache8_page_bytes(cache, ctypes.byref(v)))
        return v.value

    def cache8_append(self, cache: Cache8, batch: Batch, layer: int, k: int, v: int, rotary: Rotary | None = None,
                      heads: int = 0, q: int | None = None, q_out: int | None = None, k_stride: int | None = None,
                      v_stride: int | None = None, q_stride: int | None = None, out_stride: int | None = None) -> None:
        self._append_turned(self.lib.xpu_cache8_append, cache, batch, layer, k, v, rotary, heads, q, q_out, k_stride,
                            v_stride, q_stride, out_stride)

    def tree_attention8_workspace(self, cache: Cache8, batch: Batch, heads: int) -> int:
        """Bytes of workspace that tree_attention8 needs for these shapes."""
        v = c_uint64()
        check(self.lib.xpu_tree_attention8_workspace(self.handle, cache, batch, heads, ctypes.byref(v)))
        return v.value

    def tree_attention8(self, cache: Cache8, batch: Batch, layer: int, heads: int, q: int, out: int,
                        workspace: int | None, workspace_bytes: int, visible: int | None = None,
                        scale: float | None = None, q_stride: int | None = None, out_stride: int | None = None) -> None:
        dense = heads * cache.head_dim
        check(self.lib.xpu_tree_attention8(self.handle, cache, batch, layer, heads,
                                           cache.head_dim ** -0.5 if scale is None else scale, q,
                                           dense if q_stride is None else q_stride, visible, out,
                                           dense if out_stride is None else out_stride, workspace, workspace_bytes))

    def cache8_keep(self, cache: Cache8, batch: Batch, kept: int, counts: int, new_context: int | None = None) -> None:
        check(self.lib.xpu_cache8_keep(self.handle, cache, batch, kept, counts, new_context))

    def cache8_copy(self, cache: Cache8, src, dst) -> None:
        """src, dst: page ids on the host (arrays or lists of one length)."""
        s, d = page_ids(src), page_ids(dst)
        if len(s) != len(d):
            raise ValueError("src and dst must be of one length")
        check(self.lib.xpu_cache8_copy(self.handle, cache, s.ctypes.data, d.ctypes.data, len(s)))

    # ---- tokens from logits (include/xpu_sample.h)
    def sample_workspace(self, sampling: Sampling) -> int:
        """Bytes of workspace that sample needs for these shapes."""
        v = c_uint64()
        check(self.lib.xpu_sample_workspace(self.handle, sampling, ctypes.byref(v)))
        return v.value

    def sample(self, sampling: Sampling, logits: int, tokens: int, workspace: int | None = None,
               workspace_bytes: int = 0, probability: int | None = None) -> None:
        """A token of every row (uint32), and its share of the kept weight (FP32)."""
        check(self.lib.xpu_sample(self.handle, sampling, logits, tokens, probability, workspace, workspace_bytes))

    def prompt_attention(self, packed: Packed, q: int, k: int, v: int, out: int) -> None:
        check(self.lib.xpu_prompt_attention(self.handle, packed, q, k, v, out))

    def fill_uniform(self, dtype: int, ptr: int, count: int, seed: int) -> None:
        check(self.lib.xpu_fill_uniform(self.handle, dtype, c_void_p(ptr), count, seed))

    def fill_reference_gemv(self, dtype: int, matrix: int, vector: int, m: int, k: int, ld: int) -> None:
        check(self.lib.xpu_fill_reference_gemv(self.handle, dtype, c_void_p(matrix), c_void_p(vector), m, k, ld))


class Event:
    def __init__(self, rt: Runtime):
        self.rt = rt
        self.handle = c_void_p()
        check(rt.lib.xpu_rt_event_create(rt.handle, ctypes.byref(self.handle)))

    def record(self) -> None:
        check(self.rt.lib.xpu_rt_event_record(self.rt.handle, self.handle))

    def elapsed_ms(self, stop: "Event") -> float:
        ms = c_float()
        check(self.rt.lib.xpu_rt_event_elapsed_ms(self.handle, stop.handle, ctypes.byref(ms)))
        return ms.value

    def __del__(self):
        try:
            if self.handle:
                self.rt.lib.xpu_rt_event_destroy(self.handle)
        except Exception:
            pass
