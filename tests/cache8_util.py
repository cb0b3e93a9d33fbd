"""Shared by the tests of the 8-bit paged cache: its pages on the host and on
the device, and what the calls make of them, worked out from their definition
(codes with torch's conversion, which rounds to the nearest, ties to even)."""
import numpy as np
import torch

import xpu_playground_amd as xpu
from cache_util import TORCH, u32

BLOCK, LEAST = 16, 27
PAD = 0x5A  # bytes of a page behind its scales


def codes8(x):
    """float32 -> e4m3 codes; infinities become NaN."""
    x = np.where(np.isinf(x), np.nan, np.asarray(x, np.float32)).astype(np.float32)
    return torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def values8(codes):
    return torch.from_numpy(np.ascontiguousarray(codes)).view(torch.float8_e4m3fn).double().numpy()


def scale_byte(top):
    """The smallest byte with which a value of `top` is at most 448."""
    if not top > 0:
        return LEAST
    m, e = np.frexp(np.float64(top))
    return int(max(e - 9 + (m > 0.875) + 127, LEAST))


def rescaled(codes, by):
    """Codes times 2^by, rounded."""
    return codes8(np.ldexp(values8(codes), by).astype(np.float32))


class Pool8:
    """An 8-bit cache on the device and what it should hold."""

    def __init__(self, rt, b, n_pages, kv=2, d=64, page=16, layers=2, dtype=xpu.BF16, seed=1, stride=None):
        self.rt, self.kv, self.d, self.page, self.layers, self.n_pages, self.dtype = rt, kv, d, page, layers, n_pages, dtype
        rng = np.random.RandomState(seed)
        self.codes = {n: codes8(np.clip(rng.randn(layers, n_pages, kv, page, d) * 100, -440, 440)) for n in "kv"}
        self.scales = {n: rng.randint(110, 130, (layers, n_pages, kv, page // BLOCK)) for n in "kv"}
        self.bytes = -(-(kv * page * d + kv * page // BLOCK) // 16) * 16
        self.stride = stride or -(-self.bytes // 128) * 128
        self.status = b.up(u32([0]))
        self.ptr = {n: b.up(self.raw(n)) for n in "kv"}
        self.cache = xpu.Cache8(dtype, layers, kv, d, page, n_pages, self.ptr["k"], self.ptr["v"], self.status,
                                page_stride=self.stride)

    def raw(self, n):
        out = np.full((self.layers, self.n_pages, self.stride), PAD, np.uint8)
        at = self.kv * self.page * self.d
        out[:, :, :at] = self.codes[n].reshape(self.layers, self.n_pages, -1)
        out[:, :, at: at + self.kv * self.page // BLOCK] = self.scales[n].reshape(self.layers, self.n_pages, -1)
        return out

    def load(self, n):
        got = self.rt.download(self.ptr[n], self.layers * self.n_pages * self.stride, np.uint8)
        return got.reshape(self.layers, self.n_pages, self.stride)

    def parts(self, raw):
        at = self.kv * self.page * self.d
        codes = raw[:, :, :at].reshape(self.layers, self.n_pages, self.kv, self.page, self.d)
        scales = raw[:, :, at: at + self.kv * self.page // BLOCK]
        return codes, scales.reshape(self.layers, self.n_pages, self.kv, -1).astype(int)

    def verify(self, status=0):
        self.rt.synchronize()
        for n in "kv":
            got, want = self.load(n), self.raw(n)
            end = self.kv * self.page * self.d
            for raw in (got, want):  # a NaN is a NaN with either sign
                raw[:, :, :end][raw[:, :, :end] == 0xFF] = 0x7F
            bad = np.argwhere(got != want)
            assert not len(bad), f"{len(bad)} bytes of {n} differ, first {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"
        assert int(self.rt.download(self.status, 1, np.uint32)[0]) == status

    def place(self, table, pos):
        return int(table[pos // self.page]), pos % self.page

    def read(self, n, layer, table, positions, head):
        """What positions of a kv head stand for, in the rows' type, as float64."""
        out = np.zeros((len(positions), self.d))
        for i, pos in enumerate(positions):
            p, slot = self.place(table, pos)
            out[i] = np.ldexp(values8(self.codes[n][layer, p, head, slot]),
                              int(self.scales[n][layer, p, head, slot // BLOCK]) - 127)
        with np.errstate(over="ignore"):
            return torch.from_numpy(out).to(TORCH[self.dtype]).double().numpy()

    def append(self, layer, table, context, rows, skip=()):
        """rows: {"k": float32 [n, kv, d], "v": ...}; rows `skip` are not written (of K)."""
        for n, x in rows.items():
            skipped = skip if n == "k" else ()
            for start in range(context // BLOCK * BLOCK, context + len(x), BLOCK):
                low, high = max(start, context), min(start + BLOCK, context + len(x))
                p, slot = self.place(table, start)
                if p >= self.n_pages:
                    continue
                at = [i for i in range(low, high) if i - context not in skipped]
                for h in range(self.kv):
                    new = np.array([x[i - context, h] for i in at], np.float32).reshape(-1, self.d)
                    finite = np.abs(new[np.isfinite(new)])
                    now = scale_byte(finite.max() if finite.size else 0)
                    if low > start:
                        old = int(self.scales[n][layer, p, h, slot // BLOCK])
                        now = max(now, old)
                        if now > old:
                            held = self.codes[n][layer, p, h, slot: slot + low - start]
                            held[:] = rescaled(held, old - now)
                    self.scales[n][layer, p, h, slot // BLOCK] = now
                    for i, row in zip(at, new):
                        self.codes[n][layer, p, h, slot + i - start] = codes8(np.ldexp(row, 127 - now))

    def keep(self, table, context, kept, rows):
        """The kept nodes of a sequence with so many rows; those without a place are left."""
        def there(pos):
            return pos // self.page < len(table) and int(table[pos // self.page]) < self.n_pages

        for n in "kv":
            for layer in range(self.layers):
                for h in range(self.kv):
                    def scale(pos):
                        p, slot = self.place(table, pos)
                        return int(self.scales[n][layer, p, h, slot // BLOCK])

                    moves = [(context + j, context + i) for j, i in enumerate(kept)
                             if i < min(rows, 64) and there(context + j) and there(context + i)]
                    if not moves:
                        continue
                    old = {to // BLOCK: scale(to) for pair in moves for to in pair}
                    now = dict(old)
                    for to, of in moves:
                        now[to // BLOCK] = max(now[to // BLOCK], old[of // BLOCK])
                    new = [rescaled(self.codes[n][layer, self.place(table, of)[0], h, self.place(table, of)[1]],
                                    old[of // BLOCK] - now[to // BLOCK]) for to, of in moves]
                    first = context // BLOCK
                    for pos in range(first * BLOCK, context) if first in now and first in {t // BLOCK for t, _ in moves} else ():
                        p, slot = self.place(table, pos)
                        row = self.codes[n][layer, p, h, slot]
                        row[:] = rescaled(row, old[first] - now[first])
                    for (to, _), row in zip(moves, new):
                        p, slot = self.place(table, to)
                        self.codes[n][layer, p, h, slot] = row
                        self.scales[n][layer, p, h, slot // BLOCK] = now[to // BLOCK]
