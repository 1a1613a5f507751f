"""A ragged batch over pages, on the host and on the device, for the tests of the operators over a KV cache in pages."""
import numpy as np

from helpers import draw

F16, F32 = np.float16, np.float32


class Handle:
    """Device memory at an offset, as what _capi's argument builders take."""

    def __init__(self, buf, shape, dtype, offset=0):
        self.buf, self.ptr, self.shape = buf, buf.ptr + offset, tuple(shape)
        self.dtype = np.dtype(dtype)
        self.code = {2: 1, 4: 0}[self.dtype.itemsize]


class Batch:
    """new[s] rows and held[s] positions before them; the pools start as NaN, the table's unused entries as no page.

    gap: elements between one page and the next (K's and V's pages then lie in one buffer, in turns); shift: elements
    by which the pools start off their buffer's alignment."""

    def __init__(self, gpu, rng, new, held, hkv, d, page, dt=F16, pad=0, gap=None, shift=0, spare=3, lead=0):
        self.gpu, self.new, self.held = gpu, list(new), list(held)
        self.hkv, self.d, self.page, self.dt = hkv, d, page, np.dtype(dt)
        self.starts = np.concatenate([[lead], lead + np.cumsum(self.new)]).astype(np.uint32)
        self.rows = int(self.starts[-1]) + pad
        used = [-(-(h + n) // page) for h, n in zip(held, new)]
        self.num_pages = sum(used) + spare
        order = rng.permutation(self.num_pages)
        self.table = np.full((len(new), max(max(used), 1) + 1), 0xffffffff, np.uint32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u]
            at += u
        one = hkv * page * d
        self.stride = one if gap is None else 2 * one + gap
        self.gap, self.shift = gap, shift
        self.k, self.v = (np.full((self.num_pages, hkv, page, d), np.nan, dt) for _ in range(2))
        self.upload_tables()

    def upload_tables(self, counts=None):
        D = self.gpu.DeviceArray.from_numpy
        self.d_table, self.d_start = D(self.table), D(self.starts)
        self.d_counts = D(np.array(self.held if counts is None else counts, np.uint32))

    def fill(self, rng, rows_too=True, loud=True):
        """Positions with values: K [L, hkv, d] and V of every sequence."""
        self.K, self.V = [], []
        for s, (n, h) in enumerate(zip(self.new, self.held)):
            L = h + (n if rows_too else 0)
            k, v = (draw((L, self.hkv, self.d), rng, F32).astype(self.dt) for _ in range(2))
            if loud:
                k[:, :, ::7] *= 3
            self.K.append(k)
            self.V.append(v)
            self.store(s, k, v)

    def store(self, s, k, v, first=0):
        for j in range(len(k)):
            page, slot = self.table[s, (first + j) // self.page], (first + j) % self.page
            if page < self.num_pages:
                self.k[page, :, slot], self.v[page, :, slot] = k[j], v[j]

    def upload(self):
        """The pools to the device; pages() after it."""
        D, one = self.gpu.DeviceArray.from_numpy, self.hkv * self.page * self.d
        if self.gap is None:
            flat = [np.full(self.num_pages * one + self.shift, np.nan, self.dt) for _ in range(2)]
            for f, x in zip(flat, (self.k, self.v)):
                f[self.shift:] = x.reshape(-1)
            bufs = [D(f) for f in flat]
            offs = [self.shift * self.dt.itemsize] * 2
        else:
            f = np.full(self.num_pages * self.stride + self.shift, np.nan, self.dt)
            g = f[self.shift:].reshape(self.num_pages, self.stride)
            g[:, :one], g[:, one:2 * one] = self.k.reshape(self.num_pages, -1), self.v.reshape(self.num_pages, -1)
            bufs = [D(f)] * 2
            offs = [self.shift * self.dt.itemsize, (self.shift + one) * self.dt.itemsize]
        shape = (self.num_pages, self.hkv, self.page, self.d)
        self.d_k, self.d_v = (Handle(b, shape, self.dt, o) for b, o in zip(bufs, offs))

    def pages(self):
        return self.gpu.kv_pages(self.d_k, self.d_v, self.d_table, self.d_start, self.d_counts,
                                 page_stride=self.stride if self.gap is not None else 0)

    def download(self):
        """The pools as they are now: K and V [num_pages, hkv, page, d]."""
        one, out = self.hkv * self.page * self.d, []
        for i, h in enumerate((self.d_k, self.d_v)):
            f = h.buf.numpy()[self.shift:]
            if self.gap is not None:
                f = f.reshape(self.num_pages, self.stride)[:, i * one:(i + 1) * one]
            out.append(f.reshape(self.num_pages, self.hkv, self.page, self.d))
        return out
