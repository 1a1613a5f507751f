"""Appending to a KV cache in pages (vai_paged_append_launch): the formulas and
tolerances of the head norms and the rotation, and that nothing but the batch's
rows and slots is written."""
import ctypes

import numpy as np
import pytest

import test_qk_norm_rope_gpu as rope
from helpers import draw
from paged import Batch, F16, F32, Handle

pytestmark = pytest.mark.gpu


def positions(b, s):
    return b.held[s] + np.arange(b.new[s])


def bits(x):
    return x.view({2: np.uint16, 4: np.uint32}[x.dtype.itemsize])


def check(b, qkv, hq, q_out, q_was, pools_was, kw, drop=()):
    """q_out [rows, hq, d] (or None) and the pools after a call, against 64 bits; drop: (sequence, position) not kept."""
    k_was, v_was = pools_was
    k_now, v_now = b.download()
    k_rest, v_rest = k_now.copy(), v_now.copy()
    for s, n in enumerate(b.new):
        if n == 0:
            continue
        at, pos = int(b.starts[s]), positions(b, s)
        want, mag = rope.want64(qkv[None, at:at + n], hq, b.hkv, b.d, pos=pos[None], **kw)
        k, v = (np.zeros((1, b.hkv, n, b.d), b.dt) for _ in range(2))
        for i, p in enumerate(pos):
            if (s, p) in drop:
                k[0, :, i], v[0, :, i] = want[1][0, :, i], want[2][0, :, i]
                continue
            page, slot = b.table[s, p // b.page], p % b.page
            k[0, :, i], v[0, :, i] = k_now[page, :, slot], v_now[page, :, slot]
            k_rest[page, :, slot], v_rest[page, :, slot] = k_was[page, :, slot], v_was[page, :, slot]
        q = None if q_out is None else q_out[at:at + n].transpose(1, 0, 2)[None]
        rope.check((q, k, v), want, mag)
    np.testing.assert_array_equal(bits(k_rest), bits(k_was))
    np.testing.assert_array_equal(bits(v_rest), bits(v_was))
    if q_out is not None:
        keep = np.ones(b.rows, bool)
        keep[int(b.starts[0]):int(b.starts[-1])] = False
        np.testing.assert_array_equal(bits(q_out[keep]), bits(q_was[keep]))


def call(gpu, b, qkv, hq, odt, with_q=True, row_stride=0, shift=0, x_shift=0, **kw):
    """-> (q_out or None, what it held before)"""
    D = gpu.DeviceArray.from_numpy
    was = np.full(b.rows * hq * b.d + shift, np.nan, odt)
    qbuf = D(was)
    q = Handle(qbuf, (b.rows, hq, b.d), odt, shift * np.dtype(odt).itemsize)
    xbuf = D(np.concatenate([np.zeros(x_shift, qkv.dtype), qkv.reshape(-1)]))
    x = Handle(xbuf, qkv.shape, qkv.dtype, x_shift * qkv.dtype.itemsize)
    w = [None if x is None else D(x) for x in (kw.pop("q_weight", None), kw.pop("k_weight", None))]
    f = None if (f := kw.pop("inv_freq", None)) is None else D(f)
    a = gpu.paged_append_args(q, x, b.pages(), *w, inv_freq=f, row_stride=row_stride, **kw)
    if not with_q:
        a.q_out = None
    gpu.check(gpu.lib().vai_paged_append_launch(ctypes.byref(a), None), "append")
    gpu.synchronize()
    view = lambda x: x[shift:].reshape(b.rows, hq, b.d)  # noqa: E731
    return view(qbuf.numpy()) if with_q else None, view(was)


@pytest.mark.parametrize("new, held, hq, hkv, d, page, rot, pairs, norm, xdt, odt, pdt", [
    ([1], [0], 1, 1, 2, 1, 0, "HALVES", True, F32, F32, F32),
    ([1], [2999], 32, 8, 64, 16, 0, "HALVES", True, F16, F16, F16),
    ([1, 1, 1], [5, 0, 31], 4, 2, 64, 16, 0, "NEIGHBOURS", True, F16, F32, F16),
    ([3, 0, 7, 1], [14, 9, 0, 100000], 12, 4, 80, 24, 40, "NEIGHBOURS", False, F32, F32, F16),
    ([33, 2], [1, 70], 3, 1, 128, 64, 0, "HALVES", True, F32, F16, F32),
    ([5], [3], 8, 8, 128, 8, 64, "HALVES", True, F16, F16, F16),
    ([3, 4], [7, 2], 5, 1, 17, 3, 10, "HALVES", True, F16, F16, F16),
    ([3, 4], [7, 2], 5, 1, 17, 5, 10, "NEIGHBOURS", True, F32, F32, F32),
    ([2], [2], 2, 1, 1, 16, 0, "NONE", True, F32, F32, F32),
    ([2, 3], [1, 1], 2, 1, 512, 16, 0, "HALVES", True, F16, F16, F16),
    ([2, 3], [1, 1], 1, 2, 2048, 4, 0, "HALVES", True, F32, F32, F16),
    ([2, 1], [1, 4], 2, 1, 510, 16, 102, "NEIGHBOURS", True, F16, F16, F16),
    ([6], [90], 3, 3, 64, 32, 0, "NONE", False, F16, F32, F16),
    ([300, 1, 40], [0, 1000, 17], 40, 8, 128, 16, 0, "HALVES", True, F16, F16, F16),
    ([1] * 70, list(range(70)), 8, 2, 64, 16, 32, "HALVES", True, F16, F16, F16),
    ([0, 0, 5, 0], [1, 2, 3, 4], 4, 4, 256, 16, 0, "NEIGHBOURS", True, F16, F16, F16),
])
def test_append(gpu, new, held, hq, hkv, d, page, rot, pairs, norm, xdt, odt, pdt):
    rng = np.random.default_rng(d + len(new))
    b = Batch(gpu, rng, new, held, hkv, d, page, pdt, pad=3, lead=1)
    b.upload()
    was = b.download()
    qkv = draw((b.rows, (hq + 2 * hkv) * d), rng, xdt)
    qkv[:1] = np.nan                     # rows of no sequence are not read
    qkv[int(b.starts[-1]):] = np.nan
    kw = dict(norm=norm, eps=1e-5, pairs=pairs, theta=500000.0)
    w = [draw((d,), rng, F16) for _ in range(2)] if norm else [None, None]
    print(f"append new={new[:4]} d={d} page={page}", flush=True)
    got, q_was = call(gpu, b, qkv, hq, odt, q_weight=w[0], k_weight=w[1], rot_dim=rot, **kw)
    check(b, qkv, hq, got, q_was, was, dict(kw, qw=w[0], kw=w[1], rot=rot))


@pytest.mark.parametrize("d, gap, shift, stride, x_shift", [(64, 0, 0, 0, 0), (64, 24, 1, 5, 1), (128, 8, 3, 16, 2),
                                                          (72, 5, 1, 0, 1), (600, 3, 1, 7, 1)])
def test_strides_and_alignment(gpu, d, gap, shift, stride, x_shift):
    """K and V in one buffer, page about; projections further apart than their heads; nothing on a 16-byte boundary."""
    rng = np.random.default_rng(d)
    hq, hkv = 3, 2
    b = Batch(gpu, rng, [4, 1, 9], [3, 40, 0], hkv, d, 8, F16, gap=gap, shift=shift)
    b.upload()
    was = b.download()
    row = (hq + 2 * hkv) * d
    wide = np.full((b.rows, row + stride), np.nan, F16)
    wide[:, :row] = draw((b.rows, row), rng, F16)
    print(f"append strides d={d}", flush=True)
    got, q_was = call(gpu, b, wide, hq, F16, row_stride=row + stride, shift=shift, x_shift=x_shift, norm=False)
    check(b, wide[:, :row], hq, got, q_was, was, dict(norm=False, eps=1e-6, pairs="HALVES", rot=0))


@pytest.mark.parametrize("d", [64, 600])
def test_queries_may_stay_and_frequencies_be_given(gpu, d):
    rng = np.random.default_rng(d)
    hq, hkv = 5, 2
    b = Batch(gpu, rng, [4, 2], [30, 7], hkv, d, 16, F32)
    b.upload()
    was = b.download()
    qkv = draw((b.rows, (hq + 2 * hkv) * d), rng, F32)
    f = rng.uniform(0, 1, d // 2).astype(F32)
    print(f"append without queries d={d}", flush=True)
    call(gpu, b, qkv, hq, F32, with_q=False, norm=False, inv_freq=f)
    check(b, qkv, hq, None, None, was, dict(norm=False, pairs="HALVES", rot=0, theta=1.0, inv_freq=f))


@pytest.mark.parametrize("d", [64, 600])
def test_what_no_page_holds_is_dropped(gpu, d):
    """Entries that are no page, positions past the table and counts near 2^32: queries come, keys and values do not."""
    rng = np.random.default_rng(d)
    hq, hkv, page = 2, 2, 8
    b = Batch(gpu, rng, [20, 3, 4], [0, 5, 2], hkv, d, page, F16)
    b.table[0, 1] = b.num_pages            # one past the last
    room = b.table.shape[1] * page
    drop = {(0, p) for p in range(8, 16)} | {(2, p) for p in range(room, room + 9)}
    b.held[2] = room - 2                   # two of four rows fit; their entries are no pages either
    drop |= {(2, room - 2), (2, room - 1)}
    b.upload_tables()
    b.upload()
    was = b.download()
    qkv = draw((b.rows, (hq + 2 * hkv) * d), rng, F16)
    print(f"append dropped d={d}", flush=True)
    got, q_was = call(gpu, b, qkv, hq, F32, norm=False)
    check(b, qkv, hq, got, q_was, was, dict(norm=False, eps=1e-6, pairs="HALVES", rot=0), drop)
    b.held = [2 ** 32 - 2, 2 ** 32 - 1, 2 ** 30]   # (the last two of three positions pass 2^32: nothing wraps to 0)
    b.new, b.starts = [2, 1, 24], np.array([0, 2, 3, 27], np.uint32)
    b.upload_tables()
    drop = {(s, h + i) for s, (h, n) in enumerate(zip(b.held, b.new)) for i in range(n)}
    b.upload()
    got, q_was = call(gpu, b, qkv, hq, F32, norm=False)
    check(b, qkv, hq, got, q_was, was, dict(norm=False, eps=1e-6, pairs="HALVES", rot=0), drop)


def test_replayed_graph_follows_the_tables(gpu):
    """A recorded launch reads starts, counts and table when it runs."""
    rng = np.random.default_rng(3)
    hq, hkv, d, page = 4, 2, 64, 16
    b = Batch(gpu, rng, [3, 2], [5, 30], hkv, d, page, F16, spare=9, pad=2)
    b.upload()
    qkv = draw((b.rows, (hq + 2 * hkv) * d), rng, F16)
    D = gpu.DeviceArray.from_numpy
    q, x = D(np.zeros((b.rows, hq, d), F32)), D(qkv)
    stream = gpu.Stream()
    a = gpu.paged_append_args(q, x, b.pages(), norm=False)
    graph = gpu.Graph(stream, lambda: gpu.check(gpu.lib().vai_paged_append_launch(ctypes.byref(a), stream.ptr), "append"))
    h2d = lambda d, h: gpu.check(gpu.lib().vai_memcpy_h2d(d.ptr, h.ctypes.data, h.nbytes, None), "h2d")  # noqa: E731
    for new, held in (([3, 2], [5, 30]), ([1, 4], [8, 28]), ([0, 5], [0, 3]), ([5, 0], [17, 0])):
        b.new, b.held = new, held
        b.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        b.table = rng.permutation(b.num_pages)[:b.table.size].reshape(b.table.shape).astype(np.uint32)
        h2d(b.d_start, b.starts), h2d(b.d_table, b.table), h2d(b.d_counts, np.array(held, np.uint32))
        was, q_was = b.download(), q.numpy()
        print(f"append replay {new} {held}", flush=True)
        graph.launch()
        stream.synchronize()
        check(b, qkv, hq, q.numpy(), q_was, was, dict(norm=False, eps=1e-6, pairs="HALVES", rot=0))


def test_pages_past_32_bit_offsets(gpu):
    """Pools of more than 2^32 elements: the last page and the first."""
    rng = np.random.default_rng(4)
    hq, hkv, d, page = 2, 1, 128, 64
    stride = 1 << 28                       # 17 pages: 2^32 elements and a page
    n = 17
    D = gpu.DeviceArray.from_numpy
    pools = [gpu.DeviceArray(((n - 1) * stride + hkv * page * d,), F16) for _ in range(2)]
    table = np.array([[16, 0]], np.uint32)
    starts, counts = np.array([0, 4], np.uint32), np.array([62], np.uint32)
    hold = (D(table), D(starts), D(counts))
    pages = gpu.kv_pages(*(Handle(p, (n, hkv, page, d), F16) for p in pools), *hold, page_stride=stride)
    qkv = draw((4, (hq + 2 * hkv) * d), rng, F16)
    q = gpu.DeviceArray((4, hq, d), F32)
    print("append past 2^32", flush=True)
    gpu.paged_append(q, D(qkv), pages, norm=False)
    want, mag = rope.want64(qkv[None], hq, hkv, d, norm=False, pos=62 + np.arange(4)[None])
    got = []
    for p in pools:
        out = np.zeros((4, d), F16)
        for i, at in enumerate((16 * stride + 62 * d, 16 * stride + 63 * d, 0, d)):
            gpu.check(gpu.lib().vai_memcpy_d2h(out[i].ctypes.data, p.ptr + 2 * at, 2 * d, None), "d2h")
        got.append(out[None, None])
    rope.check((q.numpy().transpose(1, 0, 2)[None], *got), want, mag)
