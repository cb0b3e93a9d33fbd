"""Shared by the tests of the paged cache and its attention: 16-bit codes,
device buffers with guards, and attention in 64 bits with the error that the
kernels' arithmetic allows.

Error bound. With weights w_j = softmax_j, the kernels form sum_j p_j v_j /
sum_j p_j from p_j = 2^((s_j - m) log2 e), where
  - the FP32 score of D products is off by at most (D + 2) 2^-23 scale sum |q k|
    (the MFMA may round each product and partial sum), and the exponent's
    argument |s_j - m| log2 e by that times 2^-23 more; with 2^-21 for exp2:
    a relative error e_j of p_j,
  - p_j is rounded to the storage type (u = half a step relative), in fp16 with
    an absolute 2^-25 below its normal range, and the rounded values P_j are
    what both sums take: sum P v / sum P - o = sum (P - p) (v - o) / sum P, where
    sum P >= 1 in the scale of p, since the reference m is the score of some key
    (p = 1); so it is at most u sum w |v - o| / (1 - u) <= u (sum w |v| + |o|) /
    (1 - u), and in fp16 2^-25 (sum |v| + n |o|) more,
  - the FP32 sums of n terms are off by n 2^-23 relative to sum w |v|,
  - the result is rounded once (u).
Hence |error| <= (u + 2 max e + n 2^-22) sum w |v| + u |o| + 2^-25 (sum |v| + n
|o|) (fp16) + u |o|, all with a factor 1 + 3 u for the products of these, and a
subnormal result half its step more. Merging partial results adds a few 2^-22
per merge, counted with e.
"""
import numpy as np
import torch

import xpu_playground_amd as xpu

TORCH = {xpu.BF16: torch.bfloat16, xpu.FP16: torch.float16}
HALF_STEP = {xpu.BF16: 2.0 ** -8, xpu.FP16: 2.0 ** -11}
TINY = {xpu.BF16: 2.0 ** -134, xpu.FP16: 2.0 ** -25}  # half a subnormal step
GUARD = 0x7E7E
NAN = {xpu.BF16: 0x7FC0, xpu.FP16: 0x7E00}
INF = {xpu.BF16: 0x7F80, xpu.FP16: 0x7C00}


def codes(values, dtype):
    return torch.as_tensor(np.asarray(values, np.float32)).to(TORCH[dtype]).view(torch.int16).numpy().view(np.uint16)


def values(code, dtype):
    return torch.from_numpy(np.ascontiguousarray(code).view(np.int16)).view(TORCH[dtype]).double().numpy()


def normal(shape, seed, dtype, scale=1.0):
    return codes(np.random.RandomState(seed).randn(*shape) * scale, dtype)


def u32(values_):
    return np.asarray(values_, np.uint32)


class Buffers:
    """Device copies of host arrays, freed together."""

    def __init__(self, rt):
        self.rt, self.held = rt, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.rt.synchronize()
        for p in self.held:
            self.rt.free(p)

    def up(self, array, pad=0):
        """The array on the device, `pad` bytes into its block."""
        a = np.ascontiguousarray(array)
        p = self.rt.alloc(max(a.nbytes, 1) + pad)
        self.held.append(p)
        if a.nbytes:
            self.rt.copy_to(p + pad, a)
        return p + pad

    def alloc(self, nbytes):
        p = self.rt.alloc(max(nbytes, 1))
        self.held.append(p)
        return p


def attend(q, k, v, seen, scale, dtype, merges=4):
    """One head in 64 bits: (result, bound on the kernel's error). A row that
    sees nothing is 0; unseen keys take no part."""
    n, d = q.shape
    out, tol = np.zeros((n, d)), np.zeros((n, d))
    u = HALF_STEP[dtype]
    for i in range(n):
        at = np.flatnonzero(seen[i])
        if not len(at):
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (k[at] @ q[i])
            w = np.exp(s - s.max())
            w /= w.sum()
            o = w @ v[at]
            size, total = w @ np.abs(v[at]), np.abs(v[at]).sum(0)
            e = ((d + 2) * scale * (np.abs(k[at]) @ np.abs(q[i])).max() + np.abs(s - s.max()).max()) * 2.0 ** -23
            e += (2 + merges) * 2.0 ** -22
            out[i] = o
            small = 2.0 ** -25 * (total + len(at) * np.abs(o)) if dtype == xpu.FP16 else 0
            tol[i] = (u + 2 * e + len(at) * 2.0 ** -22) * size + 2 * u * np.abs(o) + small + TINY[dtype]
            tol[i] *= 1 + 3 * u
    return out, tol


def check(got, want, tol, what=""):
    with np.errstate(invalid="ignore"):  # infinities
        bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want))
    if bad.any():
        i = tuple(int(x[0]) for x in np.nonzero(bad))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} values outside the bound, first at {i}: "
                             f"{got[i]} for {want[i]} +- {tol[i]}")
