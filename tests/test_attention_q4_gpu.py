"""Attention over a 4-bit KV cache against its definition in 64 bits: the codes
exactly (through vai_attention_cache_read), the attention of the values they
stand for within the roundings of the kernels.

Tolerance of an output value sum_j p_j v_j: a score may be off by dS = 2^-11 *
scale * sum |q k| for each operand the matrix cores take rounded to fp16 (K as
stored always may be, an fp32 Q is), plus fp32 sums over the head dim; p then by
a factor of e^(2 dS) (its own score and the sum's), p and v are rounded to fp16
once each and so may be a partial result, and fp32 sums over the keys follow:
sum p |v| * (2 max dS + 3 * 2^-11 + 2^-16)."""
import ctypes

import numpy as np
import pytest

from helpers import draw

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32


def stored(x):
    """The values 4-bit rows [..., D] stand for, in 64 bits: NaN where a group is not finite in fp16."""
    with np.errstate(over="ignore"):
        x = x.astype(F16).astype(np.float64)
    out = np.empty_like(x)
    for g in range(0, x.shape[-1], 32):
        y = x[..., g:g + 32]
        ok = np.isfinite(y).all(-1, keepdims=True)
        y = np.where(ok, y, 0.0)
        lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
        s = ((hi - lo) / 15).astype(F16)
        s = np.where(15 * s.astype(np.float64) + lo > 65504, np.nextafter(s, F16(0)), s).astype(np.float64)
        n = np.where(s > 0, np.rint((y - lo) / np.where(s > 0, s, 1)), 0).clip(0, 15)
        out[..., g:g + 32] = np.where(ok, n * s + lo, np.nan)
    return out


def attend(q, k, v, see, q_rounded):
    """q [hq, T, D], k / v [hkv, L, D] as stored, see [T, L] -> (out [T, hq, D], tolerance before the output's)"""
    hq, T, D = q.shape
    grp = hq // k.shape[0]
    out, tol = np.zeros((T, hq, D)), np.zeros((T, hq, D))
    q = q.astype(np.float64)
    for h in range(hq):
        K, V = k[h // grp], v[h // grp]
        s = np.where(see, (q[h] @ K.T) / np.sqrt(D), -np.inf)
        ds = 2.0 ** -11 * (2 if q_rounded else 1) * (np.abs(q[h]) @ np.abs(K).T) / np.sqrt(D) * (1 + 2.0 ** -8)
        ds = np.where(see, ds, 0).max(-1, initial=0)[:, None]
        m = s.max(-1, keepdims=True, initial=-np.inf)
        p = np.exp(s - np.where(np.isfinite(m), m, 0))
        l = p.sum(-1, keepdims=True)
        p = np.where(l > 0, p / np.where(l > 0, l, 1), 0)
        out[:, h] = p @ V
        tol[:, h] = (p @ np.abs(V)) * (2 * ds + 3 * 2.0 ** -11 + 2.0 ** -16) + 1e-7
    return out, tol


def visible(count, tq, tkv, first, span, causal=True):
    """see [tq, positions first .. count + tkv)"""
    key = np.arange(first, count + tkv)
    i = np.arange(tq)
    end = count + np.clip(i + 1 + tkv - tq if causal else np.full(tq, tkv), 0, tkv)
    pos = count + np.maximum(i + tkv - tq, 0)
    see = key[None] < end[:, None]
    if span:
        see &= key[None] > (pos - span)[:, None]
    return see


class Cache:
    """Planes that start out as garbage, and the rows they should hold."""

    def __init__(self, gpu, hkv, size, d, ring):
        self.gpu, self.hkv, self.size, self.d, self.ring = gpu, hkv, size, d, ring
        self.k, self.v = (gpu.CachePlane(hkv, size, d, gpu.Q4) for _ in range(2))
        for p in (self.k, self.v):
            p.buf.fill_(0xFF)
        self.count = gpu.DeviceArray.from_numpy(np.zeros(1, np.uint32))
        self.n = 0
        self.rows = [np.zeros((hkv, 0, d)) for _ in range(2)]   # all positions, as stored

    def set_count(self, n):
        self.n = n
        self.gpu.check(self.gpu.lib().vai_memcpy_h2d(self.count.ptr, np.array([n], np.uint32).ctypes.data, 4, None), "h2d")

    def first(self, end):
        return max(0, end - self.size) if self.ring else 0

    def call(self, q, k, v, odt=F32, span=0, causal=True, blocks=None):
        """One call at the current count; then the count moves on."""
        g, D = self.gpu, self.gpu.DeviceArray.from_numpy
        hq, tq, _ = q.shape
        out = g.DeviceArray((1, tq, hq, self.d), odt)
        out.fill_(0xFF)
        g.attention(out, D(q[None]), None if k is None else D(k[None]), None if v is None else D(v[None]),
                    causal=causal and blocks is None, span=span, blocks=blocks,
                    cache=(self.k, self.v, self.count, self.ring))
        if k is not None:
            self.rows = [np.concatenate([r[:, :self.n], stored(x)], 1) for r, x in zip(self.rows, (k, v))]
            self.set_count(self.n + k.shape[1])
        return out.numpy()[0]

    def append(self, rng, n, dt=F16, piece=None):
        """n rows through calls of one query."""
        while n:
            m = min(n, piece or self.size)
            q = draw((self.hkv, 1, self.d), rng, F16)
            self.call(q, draw((self.hkv, m, self.d), rng, dt), draw((self.hkv, m, self.d), rng, dt), span=1)
            n -= m

    def check_rows(self):
        end, first = self.n, self.first(self.n)
        n = end - first
        if n == 0:
            return
        outs = [self.gpu.DeviceArray((self.hkv, n, self.d), F32) for _ in range(2)]
        self.gpu.attention_cache_read(*outs, self.k, self.v, first % self.size if self.ring else first)
        for o, r in zip(outs, self.rows):
            np.testing.assert_array_equal(o.numpy(), r[:, first:end].astype(F32))


def check(got, want, tol):
    if got.dtype == F16:
        tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"max error {err.max()}, {(err / tol).max()} of what is allowed"


CASES = [
    # d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt
    (64, 1, 1, 1, 1, 0, 32, False, 0, F16, F32),          # the first token of all
    (64, 8, 2, 1, 1, 31, 4096, False, 0, F16, F16),       # the new row ends a tile
    (64, 8, 2, 1, 1, 32, 4096, False, 0, F16, F16),       # ... starts one
    (128, 32, 8, 1, 1, 3000, 4096, False, 0, F16, F16),   # a decode step
    (128, 4, 4, 1, 1, 255, 256, False, 0, F32, F32),      # the cache filled to its last row, fp32
    (128, 8, 1, 4, 4, 1021, 2000, False, 0, F16, F16),    # 32 rows of one head, over a tile's end
    (128, 17, 1, 1, 1, 500, 512, False, 0, F16, F32),     # 17 rows
    (64, 4, 1, 16, 16, 700, 1024, False, 0, F16, F32),    # 64 rows
    (64, 4, 1, 17, 17, 700, 1024, False, 0, F16, F32),    # 68 rows
    (256, 8, 2, 5, 5, 900, 1280, False, 0, F16, F16),     # D = 256
    (256, 16, 1, 2, 2, 3000, 4096, False, 300, F32, F16),  # ... a window, fp32
    (32, 4, 2, 3, 3, 100, 128, False, 0, F16, F16),       # one group a row
    (80, 10, 2, 1, 1, 333, 400, False, 0, F16, F32),      # a short last group, a size that is no whole tile
    (96, 6, 2, 2, 2, 64, 99, False, 0, F32, F32),
    (17, 2, 1, 3, 3, 50, 64, False, 0, F16, F32),         # odd head dim
    (1, 2, 1, 2, 2, 5, 64, False, 0, F32, F32),
    (200, 4, 2, 3, 3, 90, 128, False, 50, F16, F32),
    (64, 4, 2, 8, 8, 252, 256, True, 60, F16, F16),       # the new rows wrap the ring
    (128, 4, 2, 5, 5, 1000, 64, True, 30, F32, F32),      # the smallest ring, wrapped many times
    (128, 8, 2, 1, 1, 700, 256, True, 0, F16, F16),       # a ring without a window: what it holds
    (256, 4, 2, 3, 3, 130, 128, True, 126, F16, F16),     # the widest window the ring allows
    (64, 4, 4, 2, 32, 100, 512, False, 0, F16, F16),      # more new keys than queries
    (64, 4, 4, 9, 4, 0, 512, False, 0, F16, F32),         # more queries than keys: the first see none
    (64, 2, 2, 200, 200, 100, 512, False, 0, F16, F16),   # a chunk of a prompt
    (128, 8, 2, 130, 130, 1000, 2048, False, 0, F16, F16),
    (128, 4, 1, 300, 300, 0, 300, False, 100, F32, F32),  # a whole prompt into a cache of its size, window
    (256, 4, 2, 70, 70, 200, 320, True, 200, F16, F16),
    (72, 4, 2, 100, 100, 30, 256, False, 0, F16, F32),
    (20, 4, 2, 90, 90, 30, 256, False, 0, F16, F32),
]


@pytest.mark.parametrize("d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt", CASES)
def test_attention_q4(gpu, d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt):
    rng = np.random.default_rng(d + size + count)
    c = Cache(gpu, hkv, size, d, ring)
    print(f"q4 d={d} hq={hq} hkv={hkv} tq={tq} tkv={tkv} count={count} size={size} ring={ring} span={span}", flush=True)
    c.append(rng, count)
    q, k, v = draw((hq, tq, d), rng, xdt), draw((hkv, tkv, d), rng, xdt), draw((hkv, tkv, d), rng, xdt)
    got = c.call(q, k, v, odt, span)
    c.check_rows()
    first = c.first(count + tkv)
    held = size - tkv + 1
    eff = (min(span, held) if span else held) if ring else span
    see = visible(count, tq, tkv, first, eff)
    want, tol = attend(q, *(r[:, first:] for r in c.rows), see, xdt == F32)
    check(got, want, tol)


@pytest.mark.parametrize("tq, span", [(1, 0), (4, 3), (40, 0), (130, 64)])
@pytest.mark.parametrize("d", [64, 128])
def test_without_new_rows_and_without_a_mask(gpu, d, tq, span):
    """Tkv = 0 attends the cache alone; an empty one gives zeros."""
    rng = np.random.default_rng(tq)
    c = Cache(gpu, 2, 200, d, False)
    q = draw((4, tq, d), rng, F16)
    print(f"q4 cache alone d={d} tq={tq}", flush=True)
    assert (c.call(q, None, None, F32, span) == 0).all()
    c.append(rng, 101)
    got = c.call(q, None, None, F32, span, causal=False)
    want, tol = attend(q, *c.rows, visible(101, tq, 0, 0, span, causal=False), False)
    check(got, want, tol)


def test_block_mask(gpu):
    """A full prefix of 3, then causal: the reference's prefix-LM mask, over cached rows."""
    rng = np.random.default_rng(6)
    for tq in (8, 70):
        c = Cache(gpu, 2, 256, 64, False)
        c.append(rng, 40)
        q, k, v = (draw((h, tq, 64), rng, F16) for h in (4, 2, 2))
        got = c.call(q, k, v, F32, blocks=(1, [3]))
        see = visible(40, tq, tq, 0, 0)
        see[:3, 40:43] = True
        want, tol = attend(q, *c.rows, see, False)
        check(got, want, tol)


@pytest.mark.parametrize("d, xdt", [(64, F16), (128, F32), (80, F16), (256, F16)])
def test_cut_into_calls_the_cache_is_the_same(gpu, d, xdt):
    """The same rows in one call, in pieces and one by one leave the same bytes."""
    rng = np.random.default_rng(d)
    n, hkv = 75, 3
    k, v = draw((hkv, n, d), rng, xdt), draw((hkv, n, d), rng, xdt)
    q = draw((hkv, 1, d), rng, F16)
    planes = []
    for pieces in ([n], [32, 33, 10], [1] * n):
        c = Cache(gpu, hkv, 96, d, False)
        for b in (c.k.buf, c.v.buf):
            b.fill_(0)
        at = 0
        for m in pieces:
            c.call(q, np.ascontiguousarray(k[:, at:at + m]), np.ascontiguousarray(v[:, at:at + m]))
            at += m
        c.check_rows()
        planes.append((c.k.buf.numpy(), c.v.buf.numpy()))
    for p in planes[1:]:
        for a, b in zip(p, planes[0]):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("d", [64, 128, 80])
def test_rows_with_nan_and_infinity(gpu, d):
    """A group that is not finite is NaN for the queries that see its row and nothing for those it is hidden from,
    one token or many; constant groups, halves and fp16's far ends keep their values."""
    rng = np.random.default_rng(3)
    for tq, count in ((1, 60), (4, 60), (70, 10)):
        for what in ("k", "v"):
            c = Cache(gpu, 2, 256, d, False)
            c.append(rng, count)
            q, k, v = draw((4, tq, d), rng, F16), draw((2, tq, d), rng, F32), draw((2, tq, d), rng, F32)
            x = k if what == "k" else v
            late = tq - 1
            x[0, 0, :16] = 0.25
            x[1, 0, :2] = (65504, -65504)
            if what == "k":
                x[1, 0] *= 2.0 ** -12
            x[0, late, 3] = np.nan
            x[1, late, d - 1] = 1e6
            print(f"q4 nan d={d} tq={tq} in {what}", flush=True)
            got = c.call(q, k, v, F32)
            c.check_rows()
            assert np.isnan(got[late]).all()
            if tq > 1:
                ks, vs = (r[:, :-1] for r in c.rows)
                see = visible(count, tq, tq, 0, 0)[:late, :-1]
                want, tol = attend(q[:, :late], ks, vs, see, False)
                check(got[:late], want, tol)
            # out of its window the row is as good as gone
            c.append(rng, 5)
            q1, k1, v1 = draw((4, 1, d), rng, F16), draw((2, 1, d), rng, F16), draw((2, 1, d), rng, F16)
            got = c.call(q1, k1, v1, F32, span=5)
            want, tol = attend(q1, *(r[:, -5:] for r in c.rows), np.ones((1, 5), bool), False)
            check(got, want, tol)


def test_cache_read_of_every_dtype(gpu):
    rng = np.random.default_rng(12)
    D = gpu.DeviceArray.from_numpy
    for dt in (F16, F32):
        k, v = draw((2, 40, 20), rng, dt), draw((2, 40, 20), rng, dt)
        for odt in (F16, F32):
            ko, vo = gpu.DeviceArray((2, 25, 20), odt), gpu.DeviceArray((2, 25, 20), odt)
            gpu.attention_cache_read(ko, vo, D(k), D(v), 30)
            rows = (30 + np.arange(25)) % 40
            np.testing.assert_array_equal(ko.numpy(), k[:, rows].astype(odt))
            np.testing.assert_array_equal(vo.numpy(), v[:, rows].astype(odt))


@pytest.mark.parametrize("hq, tq, d", [(8, 1, 64), (8, 4, 128), (4, 80, 128)])
def test_replayed_graph_follows_the_count(gpu, hq, tq, d):
    rng = np.random.default_rng(9)
    D, lib, hkv, size = gpu.DeviceArray.from_numpy, gpu.lib(), 2, 1024
    c = Cache(gpu, hkv, size, d, False)
    c.append(rng, 900)
    hist = [r.copy() for r in c.rows]
    q, k, v = draw((hq, tq, d), rng, F16), draw((hkv, tq, d), rng, F16), draw((hkv, tq, d), rng, F16)
    out = gpu.DeviceArray((1, tq, hq, d), F16)
    a = gpu.attention_args(out, D(q[None]), D(k[None]), D(v[None]), causal=True, cache=(c.k, c.v, c.count, False))
    need = lib.vai_attention_workspace_size(ctypes.byref(a))
    ws = gpu.DeviceArray((max(need, 1),), np.uint8)
    a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
    gpu.synchronize()
    stream = gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.check(lib.vai_attention_launch(ctypes.byref(a), stream.ptr), "step"))
    new = [stored(k), stored(v)]
    for count in (0, 5, 127, 128, 600, 900, 40):
        c.set_count(count)
        graph.launch()
        stream.synchronize()
        for h, n in zip(hist, new):
            h[:, count:count + tq] = n[:, :max(0, h.shape[1] - count)]
        rows = [np.concatenate([h[:, :count], n], 1) for h, n in zip(hist, new)]
        want, tol = attend(q, *rows, visible(count, tq, tq, 0, 0), False)
        check(out.numpy()[0], want, tol)


@pytest.mark.parametrize("d, hq, hkv, tq, xdt", [(64, 8, 2, 1, F16), (128, 8, 2, 3, F16), (128, 4, 4, 1, F32),
                                                 (96, 16, 1, 2, F32), (256, 4, 2, 2, F16), (256, 4, 2, 1, F32)])
def test_queries_of_any_magnitude(gpu, d, hq, hkv, tq, xdt):
    """A query times a power of two under a scale divided by it: the same result bit
    for bit (nothing under- or overflows: |q| >= 2^-6 or 0). A query of zeros: the mean of V."""
    rng = np.random.default_rng(d + hq)
    c = Cache(gpu, hkv, 320, d, False)
    c.append(rng, 300)
    q = draw((hq, tq, d), rng, xdt)
    q = np.where(np.abs(q) < 2.0 ** -6, 0, q).astype(xdt)
    q[1, 0] = 0
    print(f"q4 magnitudes d={d} hq={hq} tq={tq} {xdt.__name__}", flush=True)
    D = gpu.DeviceArray.from_numpy

    def run(e):
        out = gpu.DeviceArray((1, tq, hq, d), F32)
        gpu.attention(out, D((q * xdt(2.0 ** e))[None]), None, None, causal=True, scale=2.0 ** -e / np.sqrt(d),
                      cache=(c.k, c.v, c.count, False))
        return out.numpy()[0]

    got = run(0)
    check(got, *attend(q, *c.rows, visible(300, tq, 0, 0, 0), xdt == F32))
    for e in (-4, 8) if xdt == F16 else (-60, -20, 30, 100):
        np.testing.assert_array_equal(run(e), got)


@pytest.mark.parametrize("tq", [1, 40])
def test_planes_past_32_bit_offsets(gpu, tq):
    """The last rows of planes of 5 GB, behind a window."""
    rng = np.random.default_rng(tq)
    size, d, hkv = (1 << 26) + 64, 32, 2
    c = Cache(gpu, hkv, size, d, False)
    assert c.k.nbytes > 1 << 32
    n0 = size - 300
    c.set_count(n0)
    print(f"q4 far rows tq={tq}", flush=True)
    for m in (1, 200):   # appended by the attention itself, and by the append of a longer call
        k, v = (draw((hkv, m, d), rng, F16) for _ in range(2))
        c.call(draw((2, 1 if m == 1 else 20, d), rng, F16), k, v, span=1)
    q, k, v = draw((4, tq, d), rng, F16), draw((hkv, tq, d), rng, F16), draw((hkv, tq, d), rng, F16)
    got = c.call(q, k, v, F32, span=100)
    n = 201 + tq
    assert c.n == n0 + n
    see = visible(201, tq, tq, 0, 100)
    want, tol = attend(q, *c.rows, see, False)
    check(got, want, tol)
    outs = [gpu.DeviceArray((hkv, n, d), F32) for _ in range(2)]
    gpu.attention_cache_read(*outs, c.k, c.v, n0)
    for o, r in zip(outs, c.rows):
        np.testing.assert_array_equal(o.numpy(), r.astype(F32))


@pytest.mark.parametrize("d, tq", [(64, 1), (128, 5), (256, 2)])
def test_ring_at_far_positions(gpu, d, tq):
    """Positions past 2^31 in a ring of 256."""
    rng = np.random.default_rng(d)
    n0, hkv = 3_000_000_019, 2
    c = Cache(gpu, hkv, 256, d, True)
    c.set_count(n0)
    print(f"q4 far ring d={d} tq={tq}", flush=True)
    for _ in range(30):
        k, v = (draw((hkv, 10, d), rng, F16) for _ in range(2))
        c.call(draw((4, 1, d), rng, F16), k, v, span=1)   # (one query sees the last of them)
    q, k, v = draw((4, tq, d), rng, F16), draw((hkv, tq, d), rng, F16), draw((hkv, tq, d), rng, F16)
    got = c.call(q, k, v, F32, span=200)
    assert c.n == n0 + 300 + tq
    want, tol = attend(q, *c.rows, visible(300, tq, tq, 0, 200), False)
    check(got, want, tol)


def test_two_streams(gpu):
    """Decode steps of two sequences, each on a stream of its own, in turn."""
    rng = np.random.default_rng(3)
    D, lib, d, hkv = gpu.DeviceArray.from_numpy, gpu.lib(), 128, 2
    caches, calls, outs = [], [], []
    for n in (2000, 77):
        c = Cache(gpu, hkv, 2048, d, False)
        c.append(rng, n)
        q, k, v = (draw((h, 1, d), rng, F16) for h in (8, hkv, hkv))
        out = gpu.DeviceArray((1, 1, 8, d), F32)
        a = gpu.attention_args(out, D(q[None]), D(k[None]), D(v[None]), causal=True, cache=(c.k, c.v, c.count, False))
        ws = gpu.DeviceArray((max(lib.vai_attention_workspace_size(ctypes.byref(a)), 1),), np.uint8)
        a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
        caches.append((c, q, k, v, ws))
        calls.append(a)
        outs.append(out)
    streams = [gpu.Stream(), gpu.Stream()]
    gpu.synchronize()
    print("q4 two streams", flush=True)
    for _ in range(20):   # (the count stands: the same step each time)
        for a, s in zip(calls, streams):
            gpu.check(lib.vai_attention_launch(ctypes.byref(a), s.ptr), "step")
    for s in streams:
        s.synchronize()
    for (c, q, k, v, _), out in zip(caches, outs):
        rows = [np.concatenate([r, stored(x)], 1) for r, x in zip(c.rows, (k, v))]
        want, tol = attend(q, *rows, visible(c.n, 1, 1, 0, 0), False)
        check(out.numpy()[0], want, tol)


# Groups whose step or codes lie next to a rounding's border: fp32 alone, rounding max - min, the quotient or the
# difference x - m on the way, would land on the border itself. (low, values between, high)
BORDERS = [
    (3.045797348022461e-05, (0.5,), 1.00390625), (6.091594696044922e-05, (), 2.0078125), (9.161233901977539e-05, (), 1.0048828125),
    (6.097555160522461e-05, (), 1.8759765625), (0.00012183189392089844, (), 4.015625), (0.00012195110321044922, (1.0,), 3.751953125),
    (0.0009746551513671875, (), 32.125), (0.0077972412109375, (100.0,), 257.0), (0.015594482421875, (), 514.0),
    (-10.015625, (-3.0,), 0.00024366378784179688), (-17.703125, (), -0.00048732757568359375),
    (2.0 ** -24, (1.5, 3.5, 2.5, 14.5, 0.5), 15.0), (-2.0 ** -24, (2.5, 4.5, 1.5, 0.5, 8.5), 15.0),
    (3 * 2.0 ** -24, (1.5, 5.5, 13.5), 15.0), (2.0 ** -14, (48.0, 80.0, 112.0), 480.0), (-2.0 ** -20, (5.0, 9.0, 29.0), 30.0),
    (-65504.0, (2.0 ** -24, 0.0, -2.0 ** -24), 65504.0), (65472.0, (), 65504.0), (0.0, (2.0 ** -24,), 2.0 ** -24),
    (0.0, (7 * 2.0 ** -24, 8 * 2.0 ** -24), 22 * 2.0 ** -24),
]


@pytest.mark.parametrize("d", [64, 40, 20])
@pytest.mark.parametrize("together", [True, False])
def test_steps_and_codes_next_to_a_border(gpu, d, together):
    """Step and codes as the definition's exact arithmetic rounds them: rows appended with few queries, and a prompt's."""
    rows = np.zeros((1, len(BORDERS), d), F16)
    for i, (lo, between, hi) in enumerate(BORDERS):
        row = np.full(d, lo, F16)
        row[1:1 + len(between)] = between
        row[1 + len(between)] = hi
        row[32:] = row[:max(d - 32, 0)]
        rows[0, i] = row
    c = Cache(gpu, 1, 64, d, False)
    q = np.ones((1, 1, d), F16)
    print(f"q4 borders d={d} {together}", flush=True)
    if together:
        rows = np.concatenate([rows, rows[:, :20]], 1)      # more than 32 rows: the append of a longer call
        c.call(q, rows, np.ascontiguousarray(rows[:, ::-1]))
    else:
        for i in range(rows.shape[1]):
            c.call(q, rows[:, i:i + 1], -rows[:, i:i + 1])
    c.check_rows()


@pytest.mark.parametrize("d, tq, xdt, n", [(64, 1, F16, 8000), (128, 4, F32, 3000), (256, 2, F16, 3000)])
@pytest.mark.parametrize("down", [4, 20, 26, 30])
def test_many_keys_of_little_weight(gpu, d, tq, xdt, n, down):
    """One key in twenty outweighs the others by 2^down, but its value is zero: the result is what the others bring."""
    rng = np.random.default_rng(d + down)
    c = Cache(gpu, 1, 8192, d, False)
    k, v = np.zeros((1, n, d), F16), np.full((1, n, d), 64, F16)
    v[0, :, 1::3] = -32
    k[0, ::20, 0] = 15.0
    v[0, ::20] = 0
    q = np.zeros((4, tq, d), xdt)
    q[:, :, 0] = down * np.log(2.0) * np.sqrt(d) / 15
    q[1, :, 0] *= 0.75
    for a in range(0, n, 1000):
        c.call(np.zeros((1, 1, d), F16), np.ascontiguousarray(k[:, a:a + 1000]), np.ascontiguousarray(v[:, a:a + 1000]), span=1)
    print(f"q4 little weight d={d} tq={tq} down={down}", flush=True)
    got = c.call(q, None, None, F32)
    check(got, *attend(q, *c.rows, visible(n, tq, 0, 0, 0), xdt == F32))


MANY = [
    # d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt: up to 128 rows of a KV head, 256 over 4096 positions, from the codes
    (128, 4, 4, 33, 33, 1000, 2048, False, 0, F16, F32),     # 33 rows: the second block has one
    (64, 4, 4, 200, 200, 100, 4096, False, 0, F16, F16),     # blocks that see different tiles
    (64, 8, 2, 64, 64, 0, 4096, False, 0, F32, F32),         # a prompt
    (64, 4, 4, 128, 128, 0, 128, False, 0, F16, F32),        # ... into a cache of its size
    (128, 8, 1, 32, 32, 3000, 4096, False, 0, F32, F16),
    (128, 4, 2, 100, 100, 1000, 4100, False, 40, F16, F16),  # a window that moves with the blocks
    (128, 2, 2, 200, 200, 500, 5000, False, 7, F32, F32),    # ... of which the first blocks' is over before the last's
    (64, 4, 2, 60, 60, 1000, 256, True, 100, F16, F32),      # in a ring
    (128, 4, 2, 50, 250, 1000, 256, True, 0, F16, F16),      # nearly the whole ring anew
    (128, 8, 2, 50, 50, 5000, 4096, True, 0, F16, F16),
    (256, 4, 2, 60, 60, 700, 1024, False, 0, F32, F32),
    (256, 4, 2, 3, 3, 700, 1024, False, 0, F16, F32),        # appended apart, few rows
    (64, 4, 4, 2, 17, 100, 512, False, 0, F16, F16),         # ... and more new keys than queries
    (64, 4, 4, 90, 20, 0, 512, False, 0, F16, F32),          # more queries than keys: the first blocks see none
    (80, 6, 2, 40, 40, 333, 400, False, 0, F16, F32),
    (200, 4, 2, 70, 70, 90, 4500, False, 50, F16, F32),
    # past them: over the copies
    (64, 8, 2, 65, 65, 700, 4096, False, 0, F16, F32),
    (256, 8, 2, 40, 40, 200, 320, True, 200, F16, F16),
    (128, 4, 2, 129, 129, 1000, 2048, False, 40, F32, F16),
    (72, 8, 2, 100, 100, 30, 256, False, 0, F16, F32),
    (64, 8, 1, 40, 10, 300, 512, False, 0, F16, F32),
]


@pytest.mark.parametrize("d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt", MANY)
def test_many_rows(gpu, d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt):
    test_attention_q4(gpu, d, hq, hkv, tq, tkv, count, size, ring, span, xdt, odt)


@pytest.mark.parametrize("tq", [20, 100, 200])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_rows_of_a_block_mask(gpu, d, tq):
    """A full prefix that ends inside a block of rows, then causal; a full block after it."""
    rng = np.random.default_rng(tq)
    c = Cache(gpu, 2, 512 if tq < 200 else 4096, d, False)
    c.append(rng, 70)
    q, k, v = (draw((h, tq, d), rng, F16) for h in (2, 2, 2))
    print(f"q4 block mask d={d} tq={tq}", flush=True)
    got = c.call(q, k, v, F32, blocks=(0b010, [7, 15]))
    see = visible(70, tq, tq, 0, 0)
    see[:7, 70:77] = True
    see[15:, 85:] = True
    want, tol = attend(q, *c.rows, see, False)
    check(got, want, tol)


@pytest.mark.parametrize("hq, tq, d", [(2, 40, 64), (2, 100, 128), (4, 60, 256), (2, 150, 64), (4, 150, 128), (4, 150, 256)])
def test_rows_with_nan_among_many(gpu, hq, tq, d):
    """As for few rows: a row that is not finite reaches the queries that see it alone, from the codes and over the copies."""
    rng = np.random.default_rng(tq)
    for what in ("k", "v"):
        c = Cache(gpu, 2, 512, d, False)
        c.append(rng, 100)
        q, k, v = draw((hq, tq, d), rng, F16), draw((2, tq, d), rng, F32), draw((2, tq, d), rng, F32)
        late = tq - 7
        (k if what == "k" else v)[0, late, 3] = np.nan
        (k if what == "k" else v)[1, late, d - 1] = -np.inf
        print(f"q4 nan among many d={d} tq={tq} in {what}", flush=True)
        got = c.call(q, k, v, F32)
        c.check_rows()
        assert np.isnan(got[late:]).all()
        want, tol = attend(q[:, :late], *(r[:, :100 + late] for r in c.rows), visible(100, tq, tq, 0, 0)[:late, :100 + late], False)
        check(got[:late], want, tol)


@pytest.mark.parametrize("hq, tq, d, xdt", [(8, 80, 128, F16), (4, 60, 64, F32), (4, 100, 64, F16), (8, 5, 256, F16)])
def test_replayed_graph_of_many_rows(gpu, hq, tq, d, xdt):
    """Recorded once, replayed at other counts: an append and attention from the codes, or the copies."""
    rng = np.random.default_rng(tq)
    D, lib, hkv, size = gpu.DeviceArray.from_numpy, gpu.lib(), 2, 1024
    c = Cache(gpu, hkv, size, d, False)
    c.append(rng, 900)
    hist = [r.copy() for r in c.rows]
    q, k, v = draw((hq, tq, d), rng, xdt), draw((hkv, tq, d), rng, xdt), draw((hkv, tq, d), rng, xdt)
    out = gpu.DeviceArray((1, tq, hq, d), F32)
    a = gpu.attention_args(out, D(q[None]), D(k[None]), D(v[None]), causal=True, cache=(c.k, c.v, c.count, False))
    ws = gpu.DeviceArray((max(lib.vai_attention_workspace_size(ctypes.byref(a)), 1),), np.uint8)
    ws.fill_(0xFF)
    a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
    gpu.synchronize()
    stream = gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.check(lib.vai_attention_launch(ctypes.byref(a), stream.ptr), "step"))
    new = [stored(k), stored(v)]
    print(f"q4 graph of many rows d={d} tq={tq}", flush=True)
    for count in (0, 33, 900, 127):
        c.set_count(count)
        graph.launch()
        stream.synchronize()
        for h, n in zip(hist, new):
            h[:, count:count + tq] = n[:, :max(0, h.shape[1] - count)]
        rows = [np.concatenate([h[:, :count], n], 1) for h, n in zip(hist, new)]
        want, tol = attend(q, *rows, visible(count, tq, tq, 0, 0), xdt == F32)
        check(out.numpy()[0], want, tol)


def test_planes_past_32_bit_offsets_over_copies(gpu):
    """260 rows of a KV head at the end of planes of 5 GB: rows of fp32 copies of 17 GB each."""
    rng = np.random.default_rng(1)
    size, d, hkv, tq = (1 << 26) + 64, 32, 2, 130
    c = Cache(gpu, hkv, size, d, False)
    n0 = size - 400
    c.set_count(n0)
    print("q4 far rows over copies", flush=True)
    k, v = (draw((hkv, 200, d), rng, F16) for _ in range(2))
    c.call(draw((2, 20, d), rng, F16), k, v, span=1)
    q, k, v = draw((4, tq, d), rng, F16), draw((hkv, tq, d), rng, F16), draw((hkv, tq, d), rng, F16)
    got = c.call(q, k, v, F32, span=100)
    assert c.n == n0 + 200 + tq
    want, tol = attend(q, *c.rows, visible(200, tq, tq, 0, 100), False)
    check(got, want, tol)


@pytest.mark.parametrize("d, hq, tq, xdt, odt", [(64, 8, 1, F16, F16), (128, 4, 3, F32, F32), (128, 4, 30, F16, F16), (256, 4, 20, F32, F16),
                                                 (64, 4, 50, F16, F32), (128, 4, 140, F16, F16), (20, 4, 5, F16, F16)])
def test_operands_anywhere(gpu, d, hq, tq, xdt, odt):
    """Q, K, V and the output one element off any boundary; what lies before and behind the output stays. The same
    call gives the same bits again; a scale below zero is the query's sign turned."""
    rng = np.random.default_rng(d + tq)
    hkv, count = 2, 333
    D = gpu.DeviceArray.from_numpy
    c = Cache(gpu, hkv, 1024, d, False)
    c.append(rng, count)
    q, k, v = draw((hq, tq, d), rng, xdt), draw((hkv, tq, d), rng, xdt), draw((hkv, tq, d), rng, xdt)
    off = lambda t: D(np.concatenate([np.full(1, np.nan, t.dtype), t.ravel()]))  # noqa: E731
    rows = [np.concatenate([r, stored(x)], 1) for r, x in zip(c.rows, (k, v))]
    want, tol = attend(q, *rows, visible(count, tq, tq, 0, 0), xdt == F32)
    outs = []
    for sign in (1, 1, -1):
        dq, dk, dv = off(q * xdt(sign)), off(k), off(v)
        do = D(np.full(1 + want.size + 32, 3.0, odt))
        a = gpu.attention_args(gpu.DeviceArray((1, tq, hq, d), odt), D(q[None]), D(k[None]), D(v[None]), causal=True,
                               scale=sign / np.sqrt(d), cache=(c.k, c.v, c.count, False))
        for name, x in (("q", dq), ("k", dk), ("v", dv), ("out", do)):
            setattr(a, name, x.ptr + np.dtype(odt if name == "out" else xdt).itemsize)
        ws = gpu.DeviceArray((max(gpu.lib().vai_attention_workspace_size(ctypes.byref(a)), 1),), np.uint8)
        ws.fill_(0xFF)
        a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
        print(f"q4 anywhere d={d} tq={tq} sign={sign}", flush=True)
        gpu.check(gpu.lib().vai_attention_launch(ctypes.byref(a), None), "attention")
        gpu.synchronize()
        got = do.numpy()
        assert got[0] == 3.0 and (got[1 + want.size:] == 3.0).all()
        outs.append(got[1:1 + want.size].reshape(tq, hq, d))
        check(outs[-1], want, tol)
    np.testing.assert_array_equal(*outs[:2])


@pytest.mark.parametrize("d, hq, tq", [(64, 2, 60), (128, 4, 50), (128, 4, 140)])
def test_many_rows_of_a_ring_at_far_positions(gpu, d, hq, tq):
    """Positions past 2^31 in a ring of 512, from the codes and over the copies."""
    rng = np.random.default_rng(d)
    n0, hkv = 3_000_000_019, 2
    c = Cache(gpu, hkv, 512, d, True)
    c.set_count(n0)
    print(f"q4 far ring of many rows d={d} tq={tq}", flush=True)
    for _ in range(6):
        k, v = (draw((hkv, 100, d), rng, F16) for _ in range(2))
        c.call(draw((2, 1, d), rng, F16), k, v, span=1)
    q, k, v = draw((hq, tq, d), rng, F16), draw((hkv, tq, d), rng, F16), draw((hkv, tq, d), rng, F16)
    got = c.call(q, k, v, F32, span=300)
    want, tol = attend(q, *c.rows, visible(600, tq, tq, 0, 300), False)
    check(got, want, tol)
