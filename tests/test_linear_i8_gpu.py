"""Linear over 8-bit weights (vai_linear_i8_launch, vai_quantize_i8_launch)
against the operator's definition in 64 bits. The codes and the sums are
integers, so they are compared exactly; what follows them is fp32: the sum's
conversion, two scales, bias, scale and residual are one rounding each."""
import ctypes

import numpy as np
import pytest

from helpers import TRANS, draw, normal, np_epilogue

pytestmark = pytest.mark.gpu
F16, F32 = np.float16, np.float32
U = 2.0 ** -24   # half a step of fp32


def codes64(x):
    """(codes, scale): scale fp32 of max |x| / 127, codes the nearest integers of the exact quotients."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore"):
        amax = np.abs(x).max(-1)
        scale = (amax / 127).astype(np.float32)
        scale = np.where(scale < np.finfo(np.float32).tiny, np.float32(0), scale)
        scale = np.where(np.isfinite(x).all(-1), scale, np.float32(np.nan))
        s = scale.astype(np.float64)[:, None]
        n = np.where(s > 0, np.rint(x / np.where(s > 0, s, 1)), 0)
    return n.astype(np.int64), scale


def want64(x, w, w_scale, bias=None, residual=None, epi="NONE", order="AFTER_EPILOGUE", scale=1.0):
    """(O, the magnitude its roundings work at)"""
    n, s = codes64(x)
    a = (n @ w.astype(np.int64).T).astype(np.float64) * s.astype(np.float64)[:, None] * w_scale.astype(np.float64)
    y, mag = a, np.abs(a)
    r = 0.0
    if bias is not None:
        y, mag = y + bias.astype(np.float64), mag + np.abs(bias)
    if residual is not None:
        r = residual.astype(np.float64)
        mag = mag + np.abs(r)
    if order == "BEFORE_EPILOGUE":
        return scale * np_epilogue(epi, y + r), abs(scale) * mag
    return scale * np_epilogue(epi, y) + r, abs(scale) * mag + np.abs(r)


def check(got, want, mag, epi):
    """Six roundings at most between the integer sum and the result, each at most U of a magnitude of at most
    mag; an activation (slope below 1.13) adds its own tier; an fp16 result one rounding of its own."""
    tol = 8 * U * mag
    if epi not in ("NONE", "RELU"):
        tol = 1.13 * tol + TRANS[0] * np.abs(want) + TRANS[1]
    if got.dtype == F16:
        tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), f"max error {err.max()}, {(err / tol).max()} of what is allowed"


def weight(rng, n, k):
    w = rng.integers(-127, 128, (n, k)).astype(np.int8)
    w[0, 0] = -128
    return w, (0.01 * rng.uniform(0.5, 1.5, n)).astype(F32)


def on_gpu(gpu, w):
    rows = np.full((w.shape[0], gpu.i8_stride(w.shape[1])), 77, np.int8)   # what lies past K does not count
    rows[:, :w.shape[1]] = w
    return gpu.DeviceArray.from_numpy(rows)


@pytest.mark.parametrize("rows, k, dt", [(1, 1, F32), (1, 16, F16), (3, 17, F16), (5, 1000, F32), (2, 4096, F16),
                                         (4, 8193, F32), (1, 131072, F16), (700, 33, F16)])
def test_quantize(gpu, rows, k, dt):
    rng = np.random.default_rng(rows * k)
    x = draw((rows, k), rng, dt)
    print(f"quantize {rows} x {k} {dt.__name__}", flush=True)
    codes, scale = gpu.quantize_i8(gpu.DeviceArray.from_numpy(x))
    want, s = codes64(x)
    np.testing.assert_array_equal(scale.numpy(), s)
    got = codes.numpy()
    np.testing.assert_array_equal(got[:, :k], want)
    assert (got[:, k:] == 0).all()


def test_quantize_halves_zeros_and_what_is_not_finite(gpu):
    """Quotients that are halves go to the even integer, in exact arithmetic: with scale 3 * 2^-10 (not a power of
    two, so 1 / scale rounds) every (n + 1/2) * scale is an fp32 number."""
    s = 3 * 2.0 ** -10
    row = np.array([(n + 0.5) * s for n in range(-126, 126)] + [127 * s], F32)
    tiny = np.full_like(row, 1e-39)
    zero = np.zeros_like(row)
    nan, inf = row.copy(), row.copy()
    nan[7], inf[251] = np.nan, -np.inf
    x = np.stack([row, -row, tiny, zero, nan, inf, np.nextafter(row, F32(0)), np.full_like(row, 3e38)])
    print("quantize edges", flush=True)
    codes, scale = gpu.quantize_i8(gpu.DeviceArray.from_numpy(x))
    want, sc = codes64(x[[0, 1, 2, 3, 6, 7]])
    got = codes.numpy()[:, :x.shape[1]]
    np.testing.assert_array_equal(got[[0, 1, 2, 3, 6, 7]], want)
    np.testing.assert_array_equal(scale.numpy()[[0, 1, 2, 3, 6, 7]], sc)
    assert np.isnan(scale.numpy()[[4, 5]]).all() and (got[[4, 5]] == 0).all()


@pytest.mark.parametrize("m, n, k, xdt, odt", [
    (1, 1, 1, F16, F32), (1, 16, 64, F16, F16), (1, 8192, 2048, F16, F16), (2, 33, 100, F32, F32),
    (3, 1000, 4096, F16, F32), (7, 515, 1999, F32, F16), (8, 64, 11008, F16, F32), (9, 48, 16, F16, F32),
    (16, 100, 4097, F32, F32), (17, 31, 127, F16, F32), (33, 129, 128, F16, F32), (64, 256, 512, F16, F16),
    (100, 1003, 1000, F32, F32), (255, 257, 640, F16, F32), (256, 256, 256, F16, F16), (300, 512, 96, F16, F32),
    (513, 2049, 384, F16, F16), (1030, 4100, 200, F32, F32), (2, 64, 131072, F16, F32), (40, 40, 20000, F16, F32),
])
def test_linear_i8(gpu, m, n, k, xdt, odt):
    rng = np.random.default_rng(m + n + k)
    x, (w, ws) = draw((m, k), rng, xdt), weight(rng, n, k)
    D = gpu.DeviceArray.from_numpy
    out = gpu.DeviceArray((m, n), odt)
    out.fill_(0xFF)
    print(f"linear_i8 {m} x {n} x {k} {xdt.__name__} {odt.__name__}", flush=True)
    got = gpu.linear_i8(out, D(x), on_gpu(gpu, w), D(ws)).numpy()
    check(got, *want64(x, w, ws), "NONE")


@pytest.mark.parametrize("m, n, k", [(1, 40, 96), (5, 515, 300), (16, 64, 2048), (61, 1000, 500), (300, 768, 256),
                                     (2048, 1028, 128)])
@pytest.mark.parametrize("epi, order, scale, full_bias, bdt, odt", [
    ("NONE", "AFTER_EPILOGUE", 1.0, False, F32, F32), ("RELU", "BEFORE_EPILOGUE", 1.0, False, F16, F32),
    ("SILU", "AFTER_EPILOGUE", -0.5, True, F32, F16), ("GELU_TANH", "BEFORE_EPILOGUE", 2.0, False, F16, F16),
    ("GELU", "AFTER_EPILOGUE", 1.0, False, F32, F32), ("SIGMOID", "AFTER_EPILOGUE", 1.0, True, F16, F32)])
def test_linear_i8_epilogues(gpu, m, n, k, epi, order, scale, full_bias, bdt, odt):
    rng = np.random.default_rng(m * n)
    x, (w, ws) = draw((m, k), rng, F16), weight(rng, n, k)
    bias = draw((m, n) if full_bias else (n,), rng, bdt)
    res = draw((1, n) if m % 2 else (m, n), rng, odt)
    D = gpu.DeviceArray.from_numpy
    print(f"linear_i8 {m} x {n} x {k} {epi} {order}", flush=True)
    got = gpu.linear_i8(gpu.DeviceArray((m, n), odt), D(x), on_gpu(gpu, w), D(ws), D(bias), D(res), epi=epi,
                        order=order, scale=scale).numpy()
    want, mag = want64(x, w, ws, bias, res, epi, order, scale)
    check(got, want, mag, epi)


@pytest.mark.parametrize("m", [1, 4, 20, 300])
def test_linear_i8_rows_of_zeros_and_nan(gpu, m):
    """A row of zeros gives the bias, a row with a NaN or an infinity NaN, and neither touches the others."""
    rng = np.random.default_rng(m)
    n, k = 70, 200
    x, (w, ws), bias = draw((m, k), rng, F16), weight(rng, n, k), draw((n,), rng, F32)
    x[0] = 0
    bad = []
    if m > 1:
        x[1, 5] = np.nan
        x[m - 1, 7] = np.inf
        bad = [1, m - 1]
    D = gpu.DeviceArray.from_numpy
    print(f"linear_i8 zeros and nan m={m}", flush=True)
    got = gpu.linear_i8(gpu.DeviceArray((m, n), F32), D(x), on_gpu(gpu, w), D(ws), D(bias)).numpy()
    np.testing.assert_array_equal(got[0], bias)
    assert np.isnan(got[bad]).all()
    rest = [i for i in range(m) if i not in bad]
    check(got[rest], *want64(x[rest], w, ws, bias), "NONE")


def test_linear_i8_offset_operands(gpu):
    """X, bias, residual and the output start anywhere their types may; rows behind the last stay as they were."""
    rng = np.random.default_rng(5)
    D = gpu.DeviceArray.from_numpy
    for m, n, k in ((1, 33, 70), (6, 33, 70), (40, 70, 129), (520, 515, 130)):
        x, (w, ws) = draw((m, k), rng, F16), weight(rng, n, k)
        bias, res = draw((n,), rng, F16), draw((m, n), rng, F16)
        pad = np.zeros(1, F16)
        dx, db, dr = (D(np.concatenate([pad, t.ravel()])) for t in (x, bias, res))
        do = D(np.full(1 + m * n + 64, 3.0, F16))
        dw, dws = on_gpu(gpu, w), D(ws)
        a = gpu.linear_i8_args(gpu.DeviceArray((m, n), F16), D(x), dw, dws, D(bias), D(res))
        a.inp, a.bias, a.residual, a.out = dx.ptr + 2, db.ptr + 2, dr.ptr + 2, do.ptr + 2
        need = gpu.lib().vai_linear_i8_workspace_size(ctypes.byref(a))
        wsp = gpu.DeviceArray((max(need, 1),), np.uint8)
        a.workspace, a.workspace_bytes = wsp.ptr, wsp.nbytes
        print(f"linear_i8 offset {m} x {n} x {k}", flush=True)
        gpu.check(gpu.lib().vai_linear_i8_launch(ctypes.byref(a), None), "linear_i8")
        gpu.synchronize()
        got = do.numpy()
        assert got[0] == 3.0 and (got[1 + m * n:] == 3.0).all()
        check(got[1:1 + m * n].reshape(m, n), *want64(x, w, ws, bias, res), "NONE")


def test_linear_i8_streams_and_graph(gpu):
    """Two streams with a workspace each, and a recorded call replayed over new rows of X: the same results."""
    rng = np.random.default_rng(8)
    D = gpu.DeviceArray.from_numpy
    lib = gpu.lib()
    for m, n, k in ((1, 512, 1024), (4, 512, 1024), (100, 512, 1024)):
        w, ws = weight(rng, n, k)
        dw, dws, streams, calls = on_gpu(gpu, w), D(ws), [gpu.Stream(), gpu.Stream()], []
        for _ in streams:
            x = draw((m, k), rng, F16)
            out, dx = gpu.DeviceArray((m, n), F32), D(x)
            a = gpu.linear_i8_args(out, dx, dw, dws)
            wsp = gpu.DeviceArray((max(lib.vai_linear_i8_workspace_size(ctypes.byref(a)), 1),), np.uint8)
            a.workspace, a.workspace_bytes = wsp.ptr, wsp.nbytes
            calls.append((a, x, dx, out, wsp))
        gpu.synchronize()
        print(f"linear_i8 streams {m} x {n} x {k}", flush=True)
        for _ in range(20):
            for s, c in zip(streams, calls):
                gpu.check(lib.vai_linear_i8_launch(ctypes.byref(c[0]), s.ptr), "linear_i8")
        for s, c in zip(streams, calls):
            s.synchronize()
            check(c[3].numpy(), *want64(c[1], w, ws), "NONE")
        a, x, dx, out, _ = calls[0]
        graph = gpu.Graph(streams[0], lambda: gpu.check(lib.vai_linear_i8_launch(ctypes.byref(a), streams[0].ptr), "rec"))
        for _ in range(3):
            x = draw((m, k), rng, F16)
            gpu.check(lib.vai_memcpy_h2d(dx.ptr, x.ctypes.data, x.nbytes, None), "h2d")
            graph.launch()
            streams[0].synchronize()
            check(out.numpy(), *want64(x, w, ws), "NONE")


def test_quantized_weight_serves_linear(gpu):
    """quantize_i8 of a weight makes what linear_i8 takes; the product stays within the two roundings of the float one."""
    rng = np.random.default_rng(11)
    m, n, k = 9, 300, 1000
    x, w = draw((m, k), rng, F16), draw(normal((n, k), 0.02), rng, F16)
    D = gpu.DeviceArray.from_numpy
    codes, scale = gpu.quantize_i8(D(w))
    got = gpu.linear_i8(gpu.DeviceArray((m, n), F32), D(x), codes, scale).numpy()
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    hx, hw = np.abs(x64).max(1, keepdims=True) / 254, np.abs(w64).max(1, keepdims=True) / 254
    # |ab - a'b'| <= |a| hb + |b| ha + ha hb, ha, hb half a step each
    bound = np.abs(x64).sum(1)[:, None] * hw.T + hx * np.abs(w64).sum(1)[None, :] + k * hx * hw.T
    assert (np.abs(got - x64 @ w64.T) <= 1.001 * bound).all()


@pytest.mark.parametrize("n, k, xdt", [(300, 2048, F16), (300, 2049, F16), (515, 2730, F32), (16384, 96, F16),
                                       (16400, 96, F16), (77, 8192, F32)])
def test_rows_do_not_depend_on_their_number(gpu, n, k, xdt):
    """The sums are integers, so a row's outputs are the same bits in calls of 1 to 200
    rows: one launch or two, split over waves or in tiles."""
    rng = np.random.default_rng(n + k)
    x, (w, ws) = draw((200, k), rng, xdt), weight(rng, n, k)
    D, lib = gpu.DeviceArray.from_numpy, gpu.lib()
    dw, dws, outs = on_gpu(gpu, w), D(ws), {}
    for m in (1, 2, 3, 4, 5, 16, 17, 40, 64, 70, 200):
        out = gpu.DeviceArray((m, n), F32)
        out.fill_(0xFF)
        dx = D(x[:m])
        need = lib.vai_linear_i8_workspace_size(ctypes.byref(gpu.linear_i8_args(out, dx, dw, dws)))
        assert (need == 0) == (m <= 4 and m * k <= 8192 and n <= 16384 and n * k < 1 << 26)
        print(f"linear_i8 rows {m} x {n} x {k}", flush=True)
        outs[m] = gpu.linear_i8(out, dx, dw, dws).numpy()
    check(outs[200], *want64(x, w, ws), "NONE")
    for m, o in outs.items():
        np.testing.assert_array_equal(o, outs[200][:m])


@pytest.mark.parametrize("m, n, k", [(1, 70, 1000), (5, 70, 1000), (20, 600, 300), (64, 70, 1000), (100, 300, 700),
                                     (1000, 4096, 700), (3900, 4020, 900)])
def test_linear_i8_far_scales(gpu, m, n, k):
    """Scales of row and channel that only together lie in fp32's range: neither half of the product overflows."""
    rng = np.random.default_rng(m)
    large = np.arange(m) % 2 == 0       # rows from either end of the range in turn
    x = np.ldexp(np.clip(draw((m, k), rng, F32), -7, 7), np.where(large, 120, -110)[:, None])
    w, ws = weight(rng, n, k)
    D = gpu.DeviceArray.from_numpy
    print(f"linear_i8 far scales {m} x {n} x {k}", flush=True)
    dx, dw = D(x), on_gpu(gpu, w)
    for rows, e in ((large, -110), (~large, 100)):
        s = np.ldexp(ws, e)
        got = gpu.linear_i8(gpu.DeviceArray((m, n), F32), dx, dw, D(s)).numpy()
        codes, xs = codes64(x[rows])
        sums = codes.astype(np.float64) @ w.astype(np.float64).T      # exact: far below 2^53
        want = sums * xs.astype(np.float64)[:, None] * s.astype(np.float64)
        assert (np.abs(got[rows] - want) <= 4 * U * np.abs(want)).all()


@pytest.mark.parametrize("m, n, k, xdt, odt, biased, residual, epi", [
    # wave rings over rounded rows: 16 columns a workgroup, 32, then 32 and 64 rows
    (7, 4095, 2999, F32, F16, True, False, "NONE"), (3, 5003, 4096, F16, F32, False, True, "NONE"),
    (7, 5120, 4096, F32, F32, True, False, "NONE"), (16, 8190, 1500, F16, F16, True, True, "SILU"),
    (20, 8000, 700, F16, F32, True, True, "NONE"), (32, 4999, 2100, F32, F16, False, False, "GELU_TANH"),
    (61, 5003, 1999, F16, F16, True, False, "GELU_TANH"), (64, 4100, 1300, F32, F32, True, True, "NONE"),
    # tiles of 64
    (500, 2048, 2048, F32, F32, False, True, "NONE"), (333, 1999, 900, F16, F16, True, False, "SILU"),
    (70, 8191, 1100, F16, F32, True, True, "NONE"), (1, 16500, 2100, F16, F16, True, False, "NONE"),
    # of 128: one tile a workgroup, then two
    (1000, 4096, 700, F16, F16, True, False, "NONE"), (1000, 4091, 1100, F32, F32, True, True, "SILU"),
    (2000, 8190, 300, F16, F16, False, False, "NONE"), (1999, 8190, 290, F16, F32, True, False, "NONE"),
    # of 256: one tile a workgroup, then two; whole tiles, and rows, columns and K that end inside one
    (4096, 4096, 1024, F16, F16, False, False, "NONE"), (3900, 4020, 900, F16, F16, True, False, "GELU_TANH"),
    (3900, 4019, 1001, F32, F32, True, False, "NONE"), (3841, 3843, 900, F16, F16, True, True, "NONE"),
    (3900, 8192, 1100, F16, F32, True, False, "NONE"), (4000, 8000, 1100, F32, F16, True, True, "SILU"),
])
def test_every_kernel_over_several_stages_of_k(gpu, m, n, k, xdt, odt, biased, residual, epi):
    """Each of the kernels and epilogues the sizes choose between, over more than two 128-byte stages of K."""
    rng = np.random.default_rng(m + n + k)
    x, (w, ws) = draw((m, k), rng, xdt), weight(rng, n, k)
    bias = draw((n,), rng, F16) if biased else None
    res = draw((m, n), rng, odt) if residual else None
    D = gpu.DeviceArray.from_numpy
    out = gpu.DeviceArray((m + 1, n), odt)
    out.fill_(0xFF)
    a = gpu.linear_i8_args(gpu.DeviceArray((1, n), odt), D(x), on_gpu(gpu, w), D(ws), None if bias is None else D(bias),
                           None if res is None else D(res), epi=epi)
    a.out = out.ptr
    if biased:
        a.bias_repeat = n
    need = gpu.lib().vai_linear_i8_workspace_size(ctypes.byref(a))
    wsp = gpu.DeviceArray((max(need, 1),), np.uint8)
    wsp.fill_(0xFF)                     # (NaN scales, codes of -1, were any of it read unwritten)
    a.workspace, a.workspace_bytes = wsp.ptr, wsp.nbytes
    print(f"linear_i8 stages {m} x {n} x {k} {xdt.__name__} {odt.__name__} {epi}", flush=True)
    gpu.check(gpu.lib().vai_linear_i8_launch(ctypes.byref(a), None), "linear_i8")
    gpu.synchronize()
    got = out.numpy()
    assert (got[m].view(np.uint8) == 0xFF).all()
    codes, xs = codes64(x)
    sums = codes.astype(np.float64) @ w.astype(np.float64).T          # exact: far below 2^53
    y = sums * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    mag = np.abs(y)
    if biased:
        y, mag = y + bias.astype(np.float64), mag + np.abs(bias.astype(np.float64))
    y = np_epilogue(epi, y)
    if residual:
        y, mag = y + res.astype(np.float64), mag + np.abs(res.astype(np.float64))
    check(got[:m], y, mag, epi)
