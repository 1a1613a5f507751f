"""Attention over a KV cache in pages (vai_paged_attention_launch) against its
definition in 64 bits.

Tolerance of sum_j p_j v_j. A score: fp32 sums of D products, at most (D + 4)
half steps (2^-24) of sum |q k| * scale, 2^-21 of it more where an fp32 q enters
as two fp16 numbers; its exponent in log2 units is rounded at |s| + the largest
|s|, 2^-23 each. The weight follows by twice that (its own score's and the
largest's or the sum's), is rounded to one fp16 number for fp16 out over fp16
pages (2^-11), or to two (2^-21) or none; the sums over L keys are fp32, in the
numerator and below it, at most L / 16 + 64 steps deep each. All relative to
sum p |v|; then the output's own rounding."""
import ctypes

import numpy as np
import pytest

from helpers import draw
from paged import Batch, F16, F32, Handle

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def attend(q, k, v, see, pdt, odt, scale=None):
    """q [n, hq, D], k / v [L, hkv, D], see [n, L] -> (out [n, hq, D], tolerance)"""
    n, hq, D = q.shape
    L = len(k)
    scale = 1 / np.sqrt(D) if scale is None else scale
    out, tol = np.zeros((n, hq, D)), np.zeros((n, hq, D))
    two = pdt == F16 and q.dtype == F32
    pe = 2.0 ** -11 if pdt == F16 and odt == F16 else 2.0 ** -21
    k, v, x = k.astype(np.float64), v.astype(np.float64), q.astype(np.float64)
    for h in range(hq):
        K, V = k[:, h // (hq // k.shape[1])], v[:, h // (hq // k.shape[1])]
        s = np.where(see, x[:, h] @ K.T * scale, -np.inf)
        ds = np.abs(x[:, h]) @ np.abs(K).T * abs(scale) * ((D + 4) * U + (2.0 ** -21 if two else 0))
        top = np.where(see, np.abs(s), 0).max(-1, initial=0)
        ds = np.where(see, ds, 0).max(-1, initial=0) + 2.0 ** -22 * (top + 1)
        m = s.max(-1, keepdims=True, initial=-np.inf)
        p = np.exp(s - np.where(np.isfinite(m), m, 0))
        l = p.sum(-1, keepdims=True)
        p = np.where(l > 0, p / np.where(l > 0, l, 1), 0)
        out[:, h] = p @ V
        tol[:, h] = (p @ np.abs(V)) * (2 * ds + pe + 2 * (L / 16 + 64) * U)[:, None] + 1e-30
    if odt == F16:
        tol = tol + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
    else:
        tol = tol + np.abs(out) * 2 * U
    return out, tol


def visible(held, n, span, causal=True):
    pos, key = held + np.arange(n)[:, None], np.arange(held + n)[None]
    see = (key <= pos) if causal else np.ones((n, held + n), bool)
    return see & (key > pos - span) if span else see


def near(got, want, tol, what=""):
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), f"{what}: max error {np.nanmax(err)}, {np.nanmax(err / tol)} of what is allowed"


def check(b, q, got, odt, span=0, causal=True, scale=None, only=None):
    for s, (n, h) in enumerate(zip(b.new, b.held)):
        if n == 0 or (only is not None and s not in only):
            continue
        at = int(b.starts[s])
        want, tol = attend(q[at:at + n], b.K[s], b.V[s], visible(h, n, span, causal), b.dt, odt, scale)
        near(got[at:at + n], want, tol, f"sequence {s}")


def call(gpu, b, q, odt, out=None, shift=0, q_shift=0, q_stride=0, max_new=0, **kw):
    """q [rows, hq, d] (or rows of q_stride) -> out [rows, hq, d], 0xff where nothing was written"""
    D = gpu.DeviceArray.from_numpy
    hq = kw.pop("hq", None) or q.shape[1]
    obuf = gpu.DeviceArray((b.rows * hq * b.d + shift,), odt)
    obuf.fill_(0xFF)
    o = Handle(obuf, (b.rows, hq, b.d), odt, shift * np.dtype(odt).itemsize)
    qbuf = D(np.concatenate([np.zeros(q_shift, q.dtype), q.reshape(-1)]))
    x = Handle(qbuf, q.shape, q.dtype, q_shift * q.dtype.itemsize)
    a = gpu.paged_attention_args(o, x, b.pages(), q_stride=q_stride, max_new=max_new, **kw)
    need = gpu.lib().vai_paged_attention_workspace_size(ctypes.byref(a))
    ws = gpu.DeviceArray((need,), np.uint8)
    ws.fill_(0xFF)                         # what the workspace held does not matter
    a.workspace, a.workspace_bytes = ws.ptr, need
    gpu.check(gpu.lib().vai_paged_attention_launch(ctypes.byref(a), None), "attention")
    gpu.synchronize()
    return obuf.numpy()[shift:].reshape(b.rows, hq, b.d)


CASES = [
    # new, held, hq, hkv, d, page, pdt, qdt, odt, span
    ([1], [0], 1, 1, 64, 16, F16, F16, F16, 0), ([1], [0], 1, 1, 1, 1, F32, F32, F32, 0),
    ([1], [499], 32, 8, 64, 16, F16, F16, F16, 0), ([1], [3000], 32, 8, 128, 16, F16, F32, F32, 0),
    ([1, 1, 1, 1, 1], [0, 15, 16, 17, 4095], 8, 2, 128, 16, F16, F16, F16, 0),
    ([1, 1, 1], [31, 32, 33], 4, 4, 64, 32, F16, F16, F32, 0),
    ([1, 1], [700, 20000], 40, 8, 64, 64, F16, F32, F32, 4096), ([1], [20000], 16, 1, 256, 128, F16, F16, F16, 0),
    ([1, 1], [100, 2000], 17, 1, 128, 16, F16, F32, F16, 0), ([1, 1], [100, 2000], 5, 5, 80, 16, F16, F16, F16, 0),
    ([6, 1, 0, 3], [700, 5, 9, 0], 40, 8, 64, 32, F16, F32, F32, 0), ([5, 2], [900, 1250], 8, 2, 256, 16, F16, F16, F16, 300),
    ([4, 4, 4], [63, 64, 65], 16, 2, 128, 64, F16, F32, F32, 3), ([8], [1000], 8, 1, 96, 48, F16, F16, F16, 5),
    ([3, 1, 2], [700, 30, 0], 9, 3, 50, 24, F32, F32, F32, 0), ([3, 1, 2], [700, 30, 0], 9, 3, 50, 24, F16, F16, F16, 0),
    ([1, 2], [400, 33], 6, 2, 64, 16, F32, F32, F32, 0), ([1, 2], [400, 33], 6, 2, 128, 16, F32, F16, F16, 17),
    ([1, 1], [77, 300], 4, 1, 64, 7, F16, F16, F32, 0), ([2, 1], [77, 300], 4, 1, 17, 5, F16, F16, F16, 50),
    ([2, 2], [77, 3], 4, 2, 255, 5, F32, F32, F32, 0), ([1, 3], [10, 90], 2, 2, 256, 3, F32, F32, F32, 0),
    ([100], [0], 4, 2, 64, 16, F16, F16, F16, 0), ([129, 1, 40], [0, 1000, 17], 8, 2, 128, 16, F16, F16, F16, 0),
    ([300, 2], [333, 600], 4, 1, 128, 64, F16, F32, F32, 0), ([200, 100], [50, 0], 6, 2, 80, 32, F16, F16, F16, 64),
    ([70, 1, 33], [20, 900, 0], 16, 2, 256, 16, F16, F16, F16, 0), ([64], [4], 4, 4, 64, 8, F16, F16, F16, 0),
    ([50, 3], [7, 200], 3, 3, 33, 16, F16, F32, F32, 0), ([61], [0], 8, 4, 72, 16, F32, F32, F32, 9),
    ([2, 1], [30, 600], 4, 2, 8, 16, F16, F16, F16, 0), ([2, 40], [30, 600], 4, 2, 16, 16, F16, F32, F32, 0),
    ([3, 70], [100, 9], 6, 3, 40, 48, F16, F16, F32, 20), ([1, 33], [100, 300], 4, 2, 248, 16, F16, F16, F16, 0),
    ([1, 2], [1000, 70], 128, 1, 64, 16, F16, F16, F16, 0), ([3, 200], [900, 70], 4, 1, 128, 4096, F16, F16, F16, 0),
    ([1, 5], [3000, 0], 4, 2, 128, 1, F16, F16, F16, 0), ([7, 1], [2100, 90], 8, 2, 192, 64, F16, F32, F32, 0),
    ([2100, 1], [10, 70], 4, 1, 64, 16, F16, F16, F16, 0), ([700], [10], 8, 1, 32, 16, F32, F32, F32, 0),
    ([513], [1030], 8, 8, 64, 128, F16, F16, F16, 0), ([1] * 40, [37 * i for i in range(40)], 8, 2, 64, 16, F16, F16, F16, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{c[0][0]}-{c[4]}-{c[5]}-{c[9]}")
def test_attention(gpu, case):
    new, held, hq, hkv, d, page, pdt, qdt, odt, span = case
    rng = np.random.default_rng(d + sum(held))
    b = Batch(gpu, rng, new, held, hkv, d, page, pdt, pad=2, lead=1)
    b.fill(rng)
    b.upload()
    q = draw((b.rows, hq, d), rng, qdt)
    q[:1] = np.nan
    for hint in (max(new), 0, 1):          # (a hint that sequences exceed is only slower)
        print(f"paged attention {case} max_new={hint}", flush=True)
        got = call(gpu, b, q, odt, span=span, max_new=hint)
        check(b, q, got, odt, span)
        keep = np.r_[0:1, int(b.starts[-1]):b.rows]      # rows of no sequence stay as they were
        assert (got[keep].view(np.uint8) == 0xFF).all()
        np.testing.assert_array_equal(call(gpu, b, q, odt, span=span, max_new=hint), got)


@pytest.mark.parametrize("d, page, pdt", [(64, 16, F16), (128, 32, F16), (50, 12, F32)])
@pytest.mark.parametrize("new", [[2, 5], [40, 3], [300, 1]])
def test_without_a_mask_and_with_a_scale(gpu, d, page, pdt, new):
    """Every query over every position of its sequence (what an encoder holds, say)."""
    rng = np.random.default_rng(d)
    b = Batch(gpu, rng, new, [90, 333], 2, d, page, pdt)
    b.fill(rng)
    b.upload()
    q = draw((b.rows, 6, d), rng, F16)
    for span, scale in ((0, 0.3), (60, -0.1)):
        print(f"paged attention without a mask d={d} new={new}", flush=True)
        got = call(gpu, b, q, F32, causal=False, span=span, scale=scale)
        check(b, q, got, F32, span, False, np.float32(scale))


def test_batches_of_nothing(gpu):
    rng = np.random.default_rng(0)
    b = Batch(gpu, rng, [0, 0, 0], [5, 0, 90], 2, 64, 16, pad=4)
    b.fill(rng)
    b.upload()
    print("paged attention of nothing", flush=True)
    got = call(gpu, b, draw((b.rows, 4, 64), rng, F16), F16)
    assert (got.view(np.uint8) == 0xFF).all()


@pytest.mark.parametrize("d, page, pdt, qdt", [(64, 16, F16, F16), (128, 32, F16, F32), (50, 12, F32, F32)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 4, 2], [70, 1, 40]])
def test_entries_that_are_no_page(gpu, d, page, pdt, qdt, new):
    """Their positions are not seen; a query that sees none gives zeros."""
    rng = np.random.default_rng(d)
    hq, hkv, held = 6, 2, [200, 150, 30]
    b = Batch(gpu, rng, new, held, hkv, d, page, pdt)
    b.fill(rng)
    b.table[0, 1] = b.num_pages
    b.table[0, 3:5] = 0xffffffff
    b.table[1, :] = b.num_pages + 7
    b.upload_tables()
    b.upload()
    q = draw((b.rows, hq, d), rng, qdt)
    odt = qdt
    print(f"paged attention without some pages d={d} new={new}", flush=True)
    got = call(gpu, b, q, odt)
    see = visible(held[0], new[0], 0)
    see[:, page:2 * page] = False
    see[:, 3 * page:5 * page] = False
    near(got[:new[0]], *attend(q[:new[0]], b.K[0], b.V[0], see, pdt, odt))
    assert (got[new[0]:new[0] + new[1]] == 0).all()
    check(b, q, got, odt, only=[2])


@pytest.mark.parametrize("d, page, pdt", [(64, 16, F16), (128, 64, F16), (256, 16, F16), (50, 12, F32)])
@pytest.mark.parametrize("new, span", [([5, 1], 0), ([5, 3], 40), ([100, 1], 0), ([90, 2], 50)])
def test_values_that_are_not_finite(gpu, d, page, pdt, new, span):
    """NaN and infinity in K reach the queries that see their position, those in V at least their column of those
    queries, and no other query: not those before it, not those whose window it has left."""
    rng = np.random.default_rng(d)
    hq, hkv, held = 4, 2, [160, 77]
    b = Batch(gpu, rng, new, held, hkv, d, page, pdt)
    b.fill(rng)
    mid = held[0] + new[0] // 2
    k, v = [x.copy() for x in b.K], [x.copy() for x in b.V]
    v[0][mid, 0, 3] = np.inf
    v[0][mid, 1, 5 % d] = np.nan
    v[0][held[0] + new[0] - 1, 1, 7] = -np.inf
    k[1][held[1] + new[1] - 1, 0, 1] = np.nan
    if span:                               # positions that the windows of the first queries alone reach
        v[0][held[0] - span + 1, 0, 4] = np.nan
        k[0][held[0] - span + 2, 1, 0] = np.nan
        k[0][5, 0, 0] = v[0][6, 1, 1] = np.inf    # out of every window
    for s in range(2):
        b.store(s, k[s], v[s])
    b.upload()
    q = draw((b.rows, hq, d), rng, F16)
    odt = F16 if pdt == F16 else F32
    print(f"paged attention not finite d={d} new={new} span={span}", flush=True)
    got = call(gpu, b, q, odt, span=span).astype(np.float64)
    for s, n in enumerate(new):
        at = int(b.starts[s])
        see = visible(held[s], n, span)
        want, tol = attend(q[at:at + n], b.K[s], b.V[s], see, pdt, odt)
        for h in range(hq):
            badk = ~np.isfinite(k[s][:, h // 2]).all(-1)
            badv = ~np.isfinite(v[s][:, h // 2])
            row = (see & badk[None]).any(-1)
            bad = (see.astype(int) @ badv > 0) | row[:, None]
            assert (~np.isfinite(got[at:at + n, h][bad])).all(), f"sequence {s} head {h}"
            good = ~bad.any(-1)
            near(got[at:at + n, h][good], want[:, h][good], tol[:, h][good], f"sequence {s} head {h}")


@pytest.mark.parametrize("d, page, gap, shift, q_gap, o_shift", [
    (64, 16, 0, 0, 0, 0), (64, 16, 8, 0, 24, 0), (64, 32, 24, 1, 7, 3), (128, 16, 5, 0, 64, 1), (80, 16, 16, 8, 1, 8),
    (50, 9, 3, 1, 5, 1)])
@pytest.mark.parametrize("new", [[2, 1], [90, 1]])
def test_strides_and_alignment(gpu, d, page, gap, shift, q_gap, o_shift, new):
    """K and V in one buffer page about, queries read out of a wider row, operands off 16-byte boundaries."""
    rng = np.random.default_rng(d)
    hq, hkv = 6, 2
    b = Batch(gpu, rng, new, [200, 31], hkv, d, page, F16, gap=gap, shift=shift)
    b.fill(rng)
    b.upload()
    for qdt, odt in ((F16, F16), (F32, F32)):
        wide = np.full((b.rows, hq * d + q_gap), np.nan, qdt)
        wide[:, :hq * d] = draw((b.rows, hq * d), rng, qdt)
        print(f"paged attention strides d={d} shift={shift}", flush=True)
        got = call(gpu, b, wide, odt, shift=o_shift, q_shift=shift, q_stride=hq * d + q_gap, hq=hq)
        check(b, wide[:, :hq * d].reshape(b.rows, hq, d), got, odt)


@pytest.mark.parametrize("new", [[1, 1], [60, 1]])
def test_sequences_may_share_pages(gpu, new):
    """Two sequences over one prefix, in the same pages."""
    rng = np.random.default_rng(8)
    hq, hkv, d, page, held = 8, 2, 64, 16, [160, 160]
    b = Batch(gpu, rng, new, held, hkv, d, page, F16)
    b.fill(rng)
    b.table[1, :10] = b.table[0, :10]
    for x in (b.K, b.V):
        x[1] = np.concatenate([x[0][:160], x[1][160:]])
    b.upload_tables()
    b.store(1, b.K[1], b.V[1])
    b.upload()
    q = draw((b.rows, hq, d), rng, F16)
    print("paged attention shared", flush=True)
    check(b, q, call(gpu, b, q, F16), F16)


@pytest.mark.parametrize("d, pdt, most", [(64, F16, 1), (64, F16, 0), (256, F16, 0), (50, F32, 1)])
def test_many_sequences(gpu, d, pdt, most):
    """As many as a call takes, most of one position, with gaps (and, without a hint, one of a whole prompt)."""
    rng = np.random.default_rng(9)
    n = 4096
    new = [int(i % 3 != 1) for i in range(n)]
    new[2000] = 1 if most else 150
    held = [int(x) for x in rng.integers(0, 40, n)]
    b = Batch(gpu, rng, new, held, 1, d, 16, pdt)
    b.fill(rng)
    b.upload()
    q = draw((b.rows, 2, d), rng, F16)
    print(f"paged attention of {n}", flush=True)
    check(b, q, call(gpu, b, q, F32, max_new=most), F32)


@pytest.mark.parametrize("d, page, pdt", [(64, 16, F16), (128, 16, F16), (50, 12, F32)])
@pytest.mark.parametrize("new", [[3, 1], [80, 1]])
def test_a_query_of_nan_is_alone(gpu, d, page, pdt, new):
    rng = np.random.default_rng(d)
    b = Batch(gpu, rng, new, [70, 33], 2, d, page, pdt)
    b.fill(rng)
    b.upload()
    for qdt in (F16, F32):
        q = draw((b.rows, 4, d), rng, qdt)
        bad = q.copy()
        bad[1, 2, 3] = np.nan
        bad[0, 1] = np.inf
        print(f"paged attention nan query d={d} new={new}", flush=True)
        got = call(gpu, b, bad, F32)
        assert np.isnan(got[1, 2]).all() and not np.isfinite(got[0, 1]).any()
        good = call(gpu, b, q, F32)
        got[1, 2], got[0, 1] = good[1, 2], good[0, 1]
        check(b, q, got, F32)


@pytest.mark.parametrize("d, hq, pdt, qdt", [(64, 8, F16, F16), (128, 4, F16, F32), (50, 4, F32, F32)])
def test_replayed_graph_follows_the_tables(gpu, d, hq, pdt, qdt):
    """A recorded launch follows lengths, starts and pages; two graphs may share a workspace as they run in turn."""
    rng = np.random.default_rng(d)
    hkv, page = 2, 16
    D = gpu.DeviceArray.from_numpy
    b = Batch(gpu, rng, [30, 4], [300, 900], hkv, d, page, pdt, pad=2)
    b.k[:], b.v[:] = draw(b.k.shape, rng, F32), draw(b.v.shape, rng, F32)
    b.upload()
    q = draw((b.rows, hq, d), rng, qdt)
    out = [gpu.DeviceArray((b.rows, hq, d), F32) for _ in range(2)]
    stream, x = gpu.Stream(), D(q)
    calls = [gpu.paged_attention_args(o, x, b.pages(), max_new=30, span=span) for o, span in zip(out, (0, 100))]
    ws = gpu.DeviceArray((max(gpu.lib().vai_paged_attention_workspace_size(ctypes.byref(a)) for a in calls),), np.uint8)
    graphs = []
    for a in calls:
        a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
        graphs.append(gpu.Graph(stream, lambda: gpu.check(gpu.lib().vai_paged_attention_launch(ctypes.byref(a), stream.ptr), "x")))
    h2d = lambda d, h: gpu.check(gpu.lib().vai_memcpy_h2d(d.ptr, h.ctypes.data, h.nbytes, None), "h2d")  # noqa: E731
    for new, held in (([30, 4], [300, 900]), ([1, 1], [0, 903]), ([0, 34], [7, 500]), ([20, 0], [310, 1]), ([2, 2], [50, 60])):
        b.new, b.held = new, held
        b.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        b.table = rng.integers(0, b.num_pages, b.table.shape).astype(np.uint32)
        h2d(b.d_start, b.starts), h2d(b.d_table, b.table), h2d(b.d_counts, np.array(held, np.uint32))
        at = [np.arange(h + n) for n, h in zip(new, held)]
        b.K, b.V = ([pool[b.table[s, p // page], :, p % page] for s, p in enumerate(at)] for pool in (b.k, b.v))
        print(f"paged attention replay {new} {held}", flush=True)
        for g in graphs:
            g.launch()
        stream.synchronize()
        for o, span in zip(out, (0, 100)):
            check(b, q, o.numpy(), F32, span)


def test_two_streams(gpu):
    """Calls at once on two streams, a workspace each, over the same pages."""
    rng = np.random.default_rng(11)
    hq, hkv, d = 8, 2, 128
    D = gpu.DeviceArray.from_numpy
    b = Batch(gpu, rng, [1, 3, 1], [5000, 800, 90], hkv, d, 16, F16)
    b.fill(rng)
    b.upload()
    runs = []
    for i in range(2):
        q = draw((b.rows, hq, d), rng, F16)
        out = gpu.DeviceArray((b.rows, hq, d), F16)
        a = gpu.paged_attention_args(out, D(q), b.pages())
        n = gpu.lib().vai_paged_attention_workspace_size(ctypes.byref(a))
        ws = gpu.DeviceArray((n,), np.uint8)
        a.workspace, a.workspace_bytes = ws.ptr, n
        runs.append((gpu.Stream(), a, q, out, ws))
    print("paged attention on two streams", flush=True)
    for _ in range(10):
        for stream, a, *_ in runs:
            gpu.check(gpu.lib().vai_paged_attention_launch(ctypes.byref(a), stream.ptr), "x")
    for stream, a, q, out, ws in runs:
        stream.synchronize()
        check(b, q, out.numpy(), F16)


@pytest.mark.parametrize("tokens", [1, 40])
def test_pages_past_32_bit_offsets(gpu, tokens):
    """Pools of more than 2^32 elements: pages at both ends of them."""
    rng = np.random.default_rng(12)
    hq, hkv, d, page, n = 4, 1, 128, 64, 17
    stride = 1 << 28
    D = gpu.DeviceArray.from_numpy
    pools = [gpu.DeviceArray(((n - 1) * stride + hkv * page * d,), F16) for _ in range(2)]
    table = np.array([[16, 0, 15]], np.uint32)
    k, v = (draw((3 * page, hkv, d), rng, F16) for _ in range(2))
    for pool, x in zip(pools, (k, v)):
        for i, at in enumerate(table[0]):
            rows = np.ascontiguousarray(x[i * page:(i + 1) * page, 0])
            gpu.check(gpu.lib().vai_memcpy_h2d(pool.ptr + 2 * int(at) * stride, rows.ctypes.data, rows.nbytes, None), "h2d")
    held = 150
    hold = (D(table), D(np.array([0, tokens], np.uint32)), D(np.array([held], np.uint32)))
    pages = gpu.kv_pages(*(Handle(p, (n, hkv, page, d), F16) for p in pools), *hold, page_stride=stride)
    for qdt in (F16, F32):
        q = draw((tokens, hq, d), rng, qdt)
        out = gpu.DeviceArray((tokens, hq, d), qdt)
        print(f"paged attention past 2^32 tokens={tokens}", flush=True)
        gpu.paged_attention(out, D(q), pages)
        L = held + tokens
        near(out.numpy(), *attend(q, k[:L], v[:L], visible(held, tokens, 0), F16, qdt))


@pytest.mark.parametrize("d, qdt", [(64, F16), (128, F32), (50, F32)])
def test_queries_of_any_magnitude(gpu, d, qdt):
    """Scores far apart: one key takes all; tiny queries: every key counts alike."""
    rng = np.random.default_rng(d)
    b = Batch(gpu, rng, [4, 40], [500, 700], 2, d, 16, F16)
    b.fill(rng, loud=False)
    b.upload()
    for size in (1e-6, 1e-3, 30.0, 1000.0) + ((1e-30, 1e30) if qdt == F32 else ()):
        q = (draw((b.rows, 4, d), rng, F32) * F32(size)).astype(qdt)
        scale = None if size <= 1000 else 1e-30
        print(f"paged attention q of {size} d={d}", flush=True)
        check(b, q, call(gpu, b, q, F32, scale=scale), F32, scale=None if scale is None else np.float32(scale))
