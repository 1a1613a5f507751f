"""Head norms, rotation and layout (vai_qk_norm_rope_launch) against the
formulas in 64 bits.

Tolerance: the norm's factor carries the fp32 sum of D squares (pairwise over
lanes: at most 16 roundings deep for D <= 2048), a division, a root and a
reciprocal, and the product with the weight three more: 24 half steps of the
value. An angle's fraction of a turn is rounded to fp32 (2^-25 turns of it, 3.2
half steps as an angle), its cosine and sine to 2 steps each, the two products
and their sum three: 12 half steps of |a| + |e|."""
import ctypes

import numpy as np
import pytest

from helpers import draw

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32
U = 2.0 ** -24


def want64(qkv, hq, hkv, d, qw=None, kw=None, norm=True, eps=1e-6, offset=0.0, pairs="HALVES", rot=0, theta=10000.0,
           pos=None, inv_freq=None):
    """qkv [B, T, (hq + 2 hkv) d], pos [B, T] -> ((q, k, v), their magnitudes)"""
    B, T = qkv.shape[:2]
    x = qkv.astype(np.float64).reshape(B, T, hq + 2 * hkv, d).transpose(0, 2, 1, 3)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    rot = 0 if pairs == "NONE" else rot or d
    outs, mags = [], []
    for y, w in ((q, qw), (k, kw)):
        if norm:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
            if w is not None:
                y = y * (w.astype(np.float64) + offset)
        y, mag = y.copy(), np.abs(y)
        if rot:
            i = np.arange(rot // 2)
            f = theta ** (-2.0 * i / rot) if inv_freq is None else inv_freq.astype(np.float64)
            t = pos.astype(np.float64)[:, None, :, None] * f
            lo = i if pairs == "HALVES" else 2 * i
            hi = i + rot // 2 if pairs == "HALVES" else 2 * i + 1
            a, e = y[..., lo].copy(), y[..., hi].copy()
            y[..., lo], y[..., hi] = a * np.cos(t) - e * np.sin(t), e * np.cos(t) + a * np.sin(t)
            mag[..., lo] = mag[..., hi] = np.abs(a) + np.abs(e)
        outs.append(y)
        mags.append(mag)
    return (*outs, v), (*mags, np.abs(v))


def check(got, want, mag):
    for name, g, w, m in zip("qkv", got, want, mag):
        if g is None:
            continue
        tol = 40 * U * m
        if g.dtype == F16:
            tol = tol + np.abs(w) * 2.0 ** -11 + 2.0 ** -25
        if name == "v":
            tol = np.abs(w) * 2.0 ** -11 + 2.0 ** -25 if g.dtype == F16 else 0 * m
        err = np.abs(g.astype(np.float64) - w)
        assert (err <= tol).all(), f"{name}: max error {err.max()}, {(err / np.maximum(tol, 1e-30)).max()} of what is allowed"


def run(gpu, qkv, hq, hkv, d, odt, with_v=True, **kw):
    B, T = qkv.shape[:2]
    D = gpu.DeviceArray.from_numpy
    q, k = gpu.DeviceArray((B, hq, T, d), odt), gpu.DeviceArray((B, hkv, T, d), odt)
    v = gpu.DeviceArray((B, hkv, T, d), odt) if with_v else None
    for o in (q, k, v):
        if o is not None:
            o.fill_(0xFF)
    dev = {n: None if x is None else D(x) for n, x in kw.items() if n in ("positions", "count", "inv_freq")}
    qw, kw_ = (None if kw.get(n) is None else D(kw[n]) for n in ("q_weight", "k_weight"))
    rest = {n: x for n, x in kw.items() if n not in ("positions", "count", "inv_freq", "q_weight", "k_weight")}
    gpu.qk_norm_rope(q, k, v, D(qkv), qw, kw_, **dev, **rest)
    return tuple(None if o is None else o.numpy() for o in (q, k, v))


@pytest.mark.parametrize("B, T, hq, hkv, d, rot, pairs, norm, idt, odt", [
    (1, 1, 1, 1, 2, 0, "HALVES", True, F32, F32), (1, 1, 32, 8, 64, 0, "HALVES", True, F16, F16),
    (2, 7, 4, 2, 64, 0, "NEIGHBOURS", True, F16, F32), (1, 33, 3, 1, 128, 0, "HALVES", True, F32, F16),
    (1, 5, 8, 8, 128, 64, "HALVES", True, F16, F16), (3, 4, 2, 1, 256, 0, "NEIGHBOURS", True, F16, F16),
    (1, 9, 4, 1, 256, 128, "HALVES", False, F32, F32), (2, 11, 12, 4, 80, 40, "NEIGHBOURS", True, F32, F32),
    (1, 13, 2, 2, 72, 0, "HALVES", True, F16, F16), (1, 13, 2, 2, 96, 48, "HALVES", True, F16, F32),
    (1, 3, 5, 1, 17, 10, "HALVES", True, F16, F16), (1, 3, 5, 1, 17, 10, "NEIGHBOURS", True, F32, F32),
    (1, 2, 2, 1, 1, 0, "NONE", True, F32, F32), (1, 2, 2, 1, 512, 0, "HALVES", True, F16, F16),
    (1, 2, 1, 1, 2048, 0, "HALVES", True, F32, F32), (1, 6, 3, 3, 64, 0, "NONE", False, F16, F32),
    (1, 6, 3, 3, 32, 6, "NEIGHBOURS", True, F16, F16), (1, 300, 40, 8, 128, 0, "HALVES", True, F16, F16),
    (5, 1, 16, 2, 64, 32, "HALVES", True, F16, F16), (1, 4, 3, 1, 136, 0, "HALVES", True, F16, F16),
])
def test_norm_rope(gpu, B, T, hq, hkv, d, rot, pairs, norm, idt, odt):
    rng = np.random.default_rng(T * d)
    qkv = draw((B, T, (hq + 2 * hkv) * d), rng, idt)
    qw, kw = (draw((d,), rng, F16) for _ in range(2)) if norm else (None, None)
    pos = rng.integers(0, 100000, (B, T)).astype(np.uint32)
    print(f"norm_rope B={B} T={T} hq={hq} hkv={hkv} d={d} rot={rot} {pairs}", flush=True)
    got = run(gpu, qkv, hq, hkv, d, odt, q_weight=qw, k_weight=kw, norm=norm, eps=1e-5, pairs=pairs, rot_dim=rot,
              theta=500000.0, positions=pos)
    check(got, *want64(qkv, hq, hkv, d, qw, kw, norm, 1e-5, 0.0, pairs, rot, 500000.0, pos))


@pytest.mark.parametrize("d, pairs", [(64, "HALVES"), (128, "NEIGHBOURS"), (72, "HALVES")])
@pytest.mark.parametrize("first", [0, 1, 12345, 2 ** 20 + 1, 2 ** 32 - 3])
def test_positions_from_the_counter(gpu, d, pairs, first):
    """Positions count + token, far ones included: fp32 angles would be off by radians at 2^32."""
    rng = np.random.default_rng(d)
    T, hq, hkv = 3, 4, 2
    qkv = draw((1, T, (hq + 2 * hkv) * d), rng, F32)
    print(f"norm_rope from {first} d={d}", flush=True)
    got = run(gpu, qkv, hq, hkv, d, F32, norm=False, pairs=pairs, count=np.array([first], np.uint32))
    pos = (first + np.arange(T, dtype=np.uint64))[None]
    check(got, *want64(qkv, hq, hkv, d, norm=False, pairs=pairs, pos=pos))
    none = run(gpu, qkv, hq, hkv, d, F32, norm=False, pairs=pairs)
    check(none, *want64(qkv, hq, hkv, d, norm=False, pairs=pairs, pos=np.arange(T)[None]))


@pytest.mark.parametrize("d, rot", [(64, 0), (128, 64), (40, 20)])
def test_given_frequencies_offset_and_weights(gpu, d, rot):
    """Frequencies of the caller's, weights around zero with an offset, one weight only, and values left alone."""
    rng = np.random.default_rng(d)
    T, hq, hkv = 21, 4, 2
    qkv = draw((2, T, (hq + 2 * hkv) * d), rng, F16)
    f = (rng.uniform(0.0, 1.0, (rot or d) // 2)).astype(F32)
    qw = draw((d,), rng, F32)
    pos = rng.integers(0, 8192, (2, T)).astype(np.uint32)
    print(f"norm_rope frequencies d={d}", flush=True)
    got = run(gpu, qkv, hq, hkv, d, F32, with_v=False, q_weight=qw, weight_offset=1.0, rot_dim=rot, inv_freq=f,
              positions=pos)
    want, mag = want64(qkv, hq, hkv, d, qw, None, True, 1e-6, 1.0, "HALVES", rot, 1.0, pos, f)
    # (|w + 1| is rounded once more, at |w| + 1)
    mag = (mag[0] * 1.0 + np.abs(want[0]) + 8 * np.abs(qw).max(), *mag[1:])
    check(got, want, mag)


def test_rows_apart_and_off_alignment(gpu):
    """Rows further apart than their heads, and off 16-byte boundaries: what lies between is not read as heads."""
    rng = np.random.default_rng(2)
    D = gpu.DeviceArray.from_numpy
    B, T, hq, hkv = 2, 5, 3, 1
    for d, gap, off in ((64, 8, 0), (64, 3, 0), (64, 0, 1), (128, 16, 3), (72, 5, 1)):
        row = (hq + 2 * hkv) * d
        qkv = draw((B, T, row), rng, F16)
        wide = np.full((B * T, row + gap), np.nan, F16)
        wide[:, :row] = qkv.reshape(B * T, row)
        dx = D(np.concatenate([np.full(off, np.nan, F16), wide.ravel()]))
        q, k, v = (gpu.DeviceArray((B, h, T, d), F16) for h in (hq, hkv, hkv))
        a = gpu.qk_norm_rope_args(q, k, v, dx if False else D(qkv), row_stride=row + gap)
        a.qkv = dx.ptr + 2 * off
        print(f"norm_rope rows apart d={d} gap={gap} off={off}", flush=True)
        gpu.check(gpu.lib().vai_qk_norm_rope_launch(ctypes.byref(a), None), "norm_rope")
        gpu.synchronize()
        check((q.numpy(), k.numpy(), v.numpy()),
              *want64(qkv, hq, hkv, d, pos=np.broadcast_to(np.arange(T), (B, T))))


@pytest.mark.parametrize("d", [64, 72])
def test_heads_of_zeros_nan_and_infinity(gpu, d):
    """A head of zeros stays zero (eps > 0); a NaN or an infinity reaches its own head only."""
    rng = np.random.default_rng(1)
    T, hq, hkv = 4, 4, 2
    qkv = draw((1, T, (hq + 2 * hkv) * d), rng, F16)
    h = qkv.reshape(T, hq + 2 * hkv, d)
    h[0, 0], h[1, 1, 3], h[2, 4, 0] = 0, np.nan, np.inf
    clean = qkv.copy()
    clean.reshape(T, hq + 2 * hkv, d)[[1, 2], [1, 4]] = 1
    q, k, v = run(gpu, qkv, hq, hkv, d, F32)
    want, mag = want64(clean, hq, hkv, d, pos=np.arange(T)[None])
    assert (q[0, 0, 0] == 0).all() and np.isnan(q[0, 1, 1]).all() and np.isnan(k[0, 0, 2]).any()
    q[0, 1, 1], k[0, 0, 2] = want[0][0, 1, 1], want[1][0, 0, 2]
    check((q, k, v), want, mag)


def test_replayed_graph_follows_the_counter(gpu):
    rng = np.random.default_rng(4)
    D = gpu.DeviceArray.from_numpy
    lib, hq, hkv, d = gpu.lib(), 8, 2, 128
    qkv = draw((1, 1, (hq + 2 * hkv) * d), rng, F16)
    cnt, dx = D(np.zeros(1, np.uint32)), D(qkv)
    q, k, v = (gpu.DeviceArray((1, h, 1, d), F16) for h in (hq, hkv, hkv))
    a = gpu.qk_norm_rope_args(q, k, v, dx, count=cnt)
    gpu.synchronize()
    stream = gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.check(lib.vai_qk_norm_rope_launch(ctypes.byref(a), stream.ptr), "rec"))
    for c in (0, 1, 77, 4000, 3):
        gpu.check(lib.vai_memcpy_h2d(cnt.ptr, np.array([c], np.uint32).ctypes.data, 4, None), "h2d")
        graph.launch()
        stream.synchronize()
        check((q.numpy(), k.numpy(), v.numpy()), *want64(qkv, hq, hkv, d, pos=np.array([[c]])))


@pytest.mark.parametrize("d", [1, 2, 7, 18, 33, 66, 100, 127, 250, 495, 497])
@pytest.mark.parametrize("pairs", ["HALVES", "NEIGHBOURS"])
def test_odd_head_dims_and_rotated_parts(gpu, d, pairs):
    """Parts of a lane's eight values: every remainder of the rotated part, and of what follows it."""
    rng = np.random.default_rng(d)
    T, hq, hkv = 3, 3, 2
    qkv = draw((2, T, (hq + 2 * hkv) * d), rng, F16)
    qw, kw = (draw((d,), rng, F16) for _ in range(2))
    pos = rng.integers(0, 5000, (2, T)).astype(np.uint32)
    for rot in sorted({2, 4, 6, 10, 12, 14, 16, d // 2 * 2, d // 4 * 2, d // 3 * 2} & set(range(2, d + 1, 2))):
        print(f"norm_rope odd d={d} rot={rot} {pairs}", flush=True)
        got = run(gpu, qkv, hq, hkv, d, F16, q_weight=qw, k_weight=kw, pairs=pairs, rot_dim=rot, positions=pos)
        check(got, *want64(qkv, hq, hkv, d, qw, kw, pairs=pairs, rot=rot, pos=pos))
    got = run(gpu, qkv, hq, hkv, d, F16, q_weight=qw, k_weight=kw, pairs="NONE", positions=pos)
    check(got, *want64(qkv, hq, hkv, d, qw, kw, pairs="NONE", pos=pos))


@pytest.mark.parametrize("d", [32, 64, 72, 128, 17, 250, 640])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-5, 1e38])
def test_heads_of_any_magnitude(gpu, d, eps):
    """Heads whose squares leave fp32's range, alone or beside eps: the norm of what they hold, not 0 or infinity.
    (Below 2^-126 the inputs themselves are subnormal; the formula takes them as they stand.)"""
    rng = np.random.default_rng(d)
    scales = [-147, -140, -126, -100, -75, -66, -63, -62, -40, -20, 0, 40, 62, 63, 64, 100, 124]
    T, hq, hkv = len(scales), 3, 1
    x = draw((1, T, hq + 2 * hkv, d), rng, F32)
    x = np.clip(x, -7, 7)
    x[:, :, 1] = np.where(rng.uniform(size=(1, T, d)) < 0.5, 0, x[:, :, 1])   # a head with zeros in it
    x[:, :, 1, 0] = 2.0                                                      # (not of zeros: 0 / 0 where eps is 0)
    for t, e in enumerate(scales):
        x[:, t] = np.ldexp(x[:, t], e)
        x[:, t, :, 0] = np.where(x[:, t, :, 0] == 0, F32(np.ldexp(1.0, e)), x[:, t, :, 0])
    qkv = np.ascontiguousarray(x.reshape(1, T, -1))
    qw, kw = (draw((d,), rng, F32) for _ in range(2))
    pairs = "HALVES" if d % 2 == 0 else "NONE"
    pos = rng.integers(0, 1000, (1, T)).astype(np.uint32)
    print(f"norm_rope magnitudes d={d} eps={eps}", flush=True)
    got = run(gpu, qkv, hq, hkv, d, F32, q_weight=qw, k_weight=kw, eps=eps, pairs=pairs, positions=pos)
    want, mag = want64(qkv, hq, hkv, d, qw, kw, True, float(F32(eps)), 0.0, pairs, 0, 10000.0, pos)
    # (a result below fp32's normal range is rounded to a step of 2^-149, and so is each of its three parts)
    for g, w, m in zip(got[:2], want, mag):
        assert np.isfinite(g).all()
        assert (np.abs(g.astype(np.float64) - w) <= 40 * U * m + 2.0 ** -147).all()
    np.testing.assert_array_equal(got[2], x.transpose(0, 2, 1, 3)[:, hq + hkv:])


@pytest.mark.parametrize("d, rot", [(32, 6), (64, 10), (64, 20), (17, 10), (80, 36), (250, 12), (640, 6)])
@pytest.mark.parametrize("pairs", ["HALVES", "NEIGHBOURS"])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_what_is_not_rotated_stays(gpu, d, rot, pairs, what):
    """Values past rot_dim are only moved: one that is not finite leaves its neighbours alone."""
    rng = np.random.default_rng(d)
    T, hq, hkv = 3, 2, 1
    qkv = draw((1, T, (hq + 2 * hkv) * d), rng, F16)
    h = qkv.reshape(T, hq + 2 * hkv, d)
    clean = qkv.copy()
    for t in range(T):
        h[t, :hq + hkv, min(rot + t, d - 1)] = what
    pos = rng.integers(1, 1000, (1, T)).astype(np.uint32)
    print(f"norm_rope not rotated d={d} rot={rot} {pairs}", flush=True)
    q, k, v = run(gpu, qkv, hq, hkv, d, F32, norm=False, pairs=pairs, rot_dim=rot, positions=pos)
    want, mag = want64(clean, hq, hkv, d, norm=False, pairs=pairs, rot=rot, pos=pos)
    for o, w in ((q, want[0]), (k, want[1])):
        for t in range(T):
            at = o[0, :, t, min(rot + t, d - 1)]
            np.testing.assert_array_equal(at, np.full_like(at, what))
            o[0, :, t, min(rot + t, d - 1)] = w[0, :, t, min(rot + t, d - 1)]
    check((q, k, v), want, mag)
