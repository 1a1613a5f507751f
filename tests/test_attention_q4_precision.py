"""How exact attention over a 4-bit cache is, and that these tests would notice if it were not.

From the codes (up to 128 rows of a KV head, 256 over 4096 positions), per value. Queries with two values each that are not 0 and V whose stored values are fp16 numbers leave only
the roundings that the kernel means to be small. With A = scale * sum_d |q_d| (|k_d - m| + |m|), m the group's minimum,
a score is off by at most A times
    2^-22   an fp32 q as two fp16 numbers (fp16 ones are exact)
    2^-22   a group's sum of q as two fp16 numbers
    10 * 2^-23   fp32: the products' sums (at most 4 parts that are not 0), the step, the minima, the scale
which is below 2^-19; its weight by that, by 2^-19 for the fp32 difference to the reference (below 64) and 2^-23 for the
power, and by 2^-22 as two fp16 numbers, the largest at 2^14 or above; the sums over at most 24 tiles a wave, the waves
and the shares are fp32 (128 steps of 2^-24 at most, 2^-17). So a value is off by sum p |v| times
    2 max (2^-19 A + 2^-19 + 2^-22) + 2^-17.

Any number of rows, by the norm. One rounding to fp16 is off by 2^-11 / sqrt(3) of a value at most in the root mean
square (a uniform error of half a step of a value just above a power of two): 2.82e-4. Errors of single values are
independent, so a rounded V gives that much of the output's norm: 2.9e-4 with the fp32 part, and 1.5 times that for one
row of 64 or more values, its norm's own spread. Through the fp16 copies V, the weights, K (scores of a size about 1) and an fp32 Q are
rounded once each, and partial results of the key splits not at all: the square root of 4 times as much, 5.7e-4, and
1.5 times that for one row; both taken with a third to spare."""
import numpy as np
import pytest

from helpers import draw
from test_attention_q4_gpu import Cache, stored, visible

F16, F32 = np.float16, np.float32

FINE = [
    # d, hq, hkv, tq, count, size, ring, span, xdt
    (64, 8, 2, 1, 3000, 4096, False, 0, F16), (64, 32, 8, 1, 3000, 4096, False, 0, F32),
    (64, 16, 1, 2, 700, 1024, False, 0, F32), (64, 16, 1, 2, 700, 1024, False, 3, F16),
    (128, 32, 8, 1, 2999, 4096, False, 0, F16), (128, 8, 1, 4, 1021, 2000, False, 4, F32),
    (128, 17, 1, 1, 500, 512, False, 0, F32), (128, 4, 4, 1, 255, 256, False, 0, F32),
    (256, 8, 2, 5, 900, 1280, False, 300, F16), (256, 16, 1, 2, 2500, 4096, False, 3, F32),
    (80, 10, 2, 1, 333, 400, False, 4, F16), (96, 16, 1, 2, 64, 99, False, 5, F32),
    (32, 4, 2, 3, 100, 128, False, 0, F32), (200, 4, 2, 3, 90, 128, False, 6, F16),
    (64, 4, 2, 8, 252, 256, True, 60, F16), (128, 4, 2, 5, 1000, 64, True, 4, F32),
    (128, 4, 2, 40, 900, 1024, False, 0, F16), (64, 4, 2, 60, 300, 512, False, 5, F32), (128, 4, 2, 50, 500, 256, True, 6, F32),
    (256, 2, 1, 30, 200, 256, False, 4, F32), (64, 8, 2, 64, 30, 4096, False, 0, F16), (96, 4, 4, 200, 100, 4096, False, 6, F16),
]


def fine_inputs(d, hq, hkv, tq, count, size, ring, span, xdt):
    """q [hq, tq, d], k and v [hkv, count + tq, d], the positions the cache holds, see [tq, those positions]"""
    rng = np.random.default_rng(d + hq + count)
    n = count + tq
    k = draw((hkv, n, d), rng, F16)
    codes = rng.integers(0, 16, (hkv, n, d))
    codes[..., 0::32], codes[..., 1::32] = 0, 15        # every group from its minimum to its maximum
    codes[..., (d - 1) // 32 * 32 + 1] = 15
    v = (0.25 * codes - 2).astype(F16)
    assert (stored(v) == v).all()
    q = np.zeros((hq, tq, d), xdt)
    size_q = rng.uniform(0.6, 1.2, (hq, tq)) * np.sqrt(d) * rng.choice((-1, 1), (hq, tq))
    at = rng.integers(0, d, (hq, tq))
    other = at // 32 * 32 + rng.integers(0, np.minimum(32, d - at // 32 * 32))
    h, t = np.indices((hq, tq))
    q[h, t, other] = (size_q * rng.uniform(0.003, 0.01, (hq, tq))).astype(xdt)
    q[h, t, at] = size_q.astype(xdt)
    first = max(0, n - size) if ring else 0
    eff = min(span, size - tq + 1) if ring and span else span
    see = visible(count, tq, tq, first, eff)
    if not 0 < span <= 6:    # the keys at the ends of what a row sees: none of little weight, and all with large values
        ends = first + np.concatenate([see.argmax(1), see.argmax(1) - 1, n - first - 1 - see[:, ::-1].argmax(1)])
        ends = ends[ends >= first]
        k[:, ends] = 0
        v[:, ends] *= 8
        assert (stored(v) == v).all()
    return q, k, v, first, see


def fine_attend(q, k, v, see, q_as=None, p_as=None, sum_as=None):
    """(out [T, hq, D], what it may be off by) of rows as stored; q_as, p_as, sum_as: as if these were rounded so."""
    hq, T, D = q.shape
    K, V = stored(k), stored(v)
    low = np.concatenate([np.broadcast_to(K[..., g:g + 32].min(-1, keepdims=True), K[..., g:g + 32].shape)
                          for g in range(0, D, 32)], -1)      # (a group's smallest value is stored as it is)
    out, tol = np.zeros((T, hq, D)), np.zeros((T, hq, D))
    for h in range(hq):
        Kh, Vh, mh = (x[h // (hq // k.shape[0])] for x in (K, V, low))
        x = q[h].astype(np.float64)
        xr = q_as(x) if q_as else x
        s = (xr @ (Kh - mh).T)
        for g in range(0, D, 32):
            total = xr[:, g:g + 32].sum(-1)
            s += np.outer(sum_as(total) if sum_as else total, mh[:, g])
        s = np.where(see, s / np.sqrt(D), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        pn = p_as(p) if p_as else p
        out[:, h] = pn @ Vh / p.sum(-1, keepdims=True)
        A = np.where(see, np.abs(x) @ (np.abs(Kh - mh) + np.abs(mh)).T / np.sqrt(D), 0).max(-1, keepdims=True)
        rel = 2 * (2.0 ** -19 * A + 2.0 ** -19 + 2.0 ** -22) + 2.0 ** -17
        tol[:, h] = p @ np.abs(Vh) / p.sum(-1, keepdims=True) * rel
    return out, tol


def to16(x):
    return x.astype(F16).astype(np.float64)


def to16_at(x):   # (the largest at 2^14)
    return to16(x * 2.0 ** 14) / 2.0 ** 14


@pytest.mark.parametrize("case", FINE, ids=str)
def test_a_coarser_result_would_be_noticed(case):
    """On the CPU: one number for an fp32 query, for a group's sum or for a weight, and the newest or oldest key seen
    dropped or the first hidden one let in, in every row, leave the tolerance."""
    d, hq, hkv, tq, count, size, ring, span, xdt = case
    q, k, v, first, see = fine_inputs(*case)
    k, v = k[:, first:], v[:, first:]
    want, tol = fine_attend(q, k, v, see)
    same, _ = fine_attend(q, k, v, see, q_as=lambda x: x.astype(F32).astype(np.float64))
    assert (np.abs(same - want) <= tol).all()
    wrong = {}
    if xdt == F32:
        wrong["q"] = fine_attend(q, k, v, see, q_as=to16)
    if 0 < span <= 6:            # (over many keys these roundings average out)
        wrong["p"] = fine_attend(q, k, v, see, p_as=to16_at)
        wrong["sum"] = fine_attend(q, k, v, see, sum_as=to16)
    rows = np.arange(tq)
    newest, oldest = see.shape[1] - 1 - see[:, ::-1].argmax(1), see.argmax(1)
    for name, at in (("newest", newest), ("oldest", oldest)):
        less = see.copy()
        less[rows, at] = False
        wrong[name] = fine_attend(q, k, v, less)
    for name, at in (("after", newest + 1), ("before", oldest - 1)):
        ok = (at >= 0) & (at < see.shape[1])
        more = see.copy()
        more[rows[ok], at[ok]] = True
        if ok.any():
            wrong[name] = fine_attend(q, k, v, more)
    for name, (got, _) in wrong.items():
        if name in ("sum", "q", "p"):
            assert (np.abs(got - want) > tol).any(), name
        else:                    # in every row that the change reaches
            hit = (np.abs(got - want) > tol).any(-1)
            reached = {"after": newest + 1 < see.shape[1], "before": oldest > 0}.get(name, np.ones(tq, bool))
            assert hit[reached].all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("case", FINE, ids=str)
def test_exact_but_for_v(gpu, case):
    d, hq, hkv, tq, count, size, ring, span, xdt = case
    q, k, v, first, see = fine_inputs(*case)
    c = Cache(gpu, hkv, size, d, ring)
    print(f"q4 fine {case}", flush=True)
    scrap = np.ones((hkv, 1, d), F16)
    for a in range(0, count, size):
        b = min(count, a + size)
        c.call(scrap, np.ascontiguousarray(k[:, a:b]), np.ascontiguousarray(v[:, a:b]), span=1)
    got = c.call(q, np.ascontiguousarray(k[:, count:]), np.ascontiguousarray(v[:, count:]), F32, span)
    want, tol = fine_attend(q, k[:, first:], v[:, first:], see)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), f"{(err / tol).max()} of what is allowed"


NORM = [
    # d, hq, hkv, tq, count, size, span, xdt: few rows
    (64, 32, 8, 1, 3000, 4096, 0, F16), (128, 32, 8, 1, 3000, 4096, 0, F32), (256, 8, 2, 5, 900, 1280, 0, F16),
    (64, 16, 1, 4, 700, 1024, 0, F32), (96, 6, 2, 2, 2000, 2048, 900, F32),
    (64, 4, 1, 17, 700, 1024, 0, F16), (128, 16, 1, 5, 2000, 2048, 0, F32), (256, 4, 2, 64, 200, 320, 150, F32),
    (64, 4, 4, 40, 3000, 4096, 0, F16), (128, 8, 2, 64, 500, 5000, 0, F32),
    # past that, over the copies
    (128, 8, 2, 130, 1000, 2048, 0, F16), (64, 4, 1, 65, 700, 1024, 0, F16), (256, 8, 2, 70, 200, 320, 150, F32),
    (64, 4, 4, 300, 1000, 2048, 0, F32),
]


def from_codes(d, hq, hkv, tq, size):
    return d % 8 == 0 and hq // hkv * tq <= (256 if size >= 4096 else 128)


def dense(q, k, v, see):
    hq, T, D = q.shape
    K, V = stored(k), stored(v)
    out = np.zeros((T, hq, D))
    for h in range(hq):
        s = np.where(see, q[h].astype(np.float64) @ K[h * k.shape[0] // hq].T / np.sqrt(D), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = p @ V[h * k.shape[0] // hq] / p.sum(-1, keepdims=True)
    return out


def norms(got, want):
    """error of the whole, and of the worst row"""
    e = got.astype(np.float64) - want
    return np.linalg.norm(e) / np.linalg.norm(want), (np.linalg.norm(e, axis=-1) / np.linalg.norm(want, axis=-1)).max()


def bounds(case):
    return (2.9e-4, 4.4e-4) if from_codes(*case[:4], case[5]) else (7.6e-4, 1.14e-3)


def norm_inputs(d, hq, hkv, tq, count, size, span, xdt):
    rng = np.random.default_rng(d + tq)
    q, k, v = draw((hq, tq, d), rng, xdt), draw((hkv, count + tq, d), rng, xdt), draw((hkv, count + tq, d), rng, xdt)
    return q, k, v, visible(count, tq, tq, 0, span)


@pytest.mark.parametrize("case", NORM, ids=str)
def test_a_lost_key_would_be_noticed(case):
    q, k, v, see = norm_inputs(*case)
    want = dense(q, k, v, see)
    rows = np.arange(see.shape[0])
    for at in (see.shape[1] - 1 - see[:, ::-1].argmax(1), see.argmax(1)):
        less = see.copy()
        less[rows, at] = False
        whole, worst = norms(dense(q, k, v, less), want)
        assert whole > bounds(case)[0] and worst > bounds(case)[1]


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM, ids=str)
def test_error_by_the_norm(gpu, case):
    d, hq, hkv, tq, count, size, span, xdt = case
    q, k, v, see = norm_inputs(*case)
    c = Cache(gpu, hkv, size, d, False)
    print(f"q4 norm {case}", flush=True)
    c.call(np.ones((hkv, 1, d), F16), np.ascontiguousarray(k[:, :count]), np.ascontiguousarray(v[:, :count]), span=1)
    got = c.call(q, np.ascontiguousarray(k[:, count:]), np.ascontiguousarray(v[:, count:]), F32, span)
    c.check_rows()
    whole, worst = norms(got, dense(q, k, v, see))
    print(f"error {whole:.3g}, worst row {worst:.3g}", flush=True)
    assert whole <= bounds(case)[0] and worst <= bounds(case)[1]


@pytest.mark.gpu
@pytest.mark.parametrize("d, hq, hkv, tq, count, size, ring, span, xdt", [
    (20, 4, 2, 3, 30, 64, False, 0, F32), (17, 4, 1, 1, 60, 64, False, 0, F16), (250, 4, 2, 2, 30, 64, False, 0, F32),
    (100, 2, 2, 20, 9, 64, False, 0, F16), (1, 2, 1, 5, 40, 64, False, 0, F32), (65, 4, 2, 20, 400, 128, True, 20, F32),
    (12, 4, 2, 20, 20, 64, False, 0, F16), (30, 2, 1, 300, 500, 1024, False, 9, F16)])
def test_other_head_dims_are_exact(gpu, d, hq, hkv, tq, count, size, ring, span, xdt):
    """Head dims the matrix cores do not take: every value in fp32 as it is stored, so a result is off by what fp32
    leaves of the scores (the head dim's chain of sums and the scale: (d + 4) 2^-24 of scale * sum |q k|, twice), of the
    powers (2^-21) and of the sum over the keys (a chain of each, 2 n 2^-24)."""
    rng = np.random.default_rng(d + tq)
    n = count + tq
    q, k, v = draw((hq, tq, d), rng, xdt), draw((hkv, n, d), rng, xdt), draw((hkv, n, d), rng, xdt)
    c = Cache(gpu, hkv, size, d, ring)
    print(f"q4 exact d={d} tq={tq}", flush=True)
    for a in range(0, count, size):
        b = min(count, a + size)
        c.call(np.ones((hkv, 1, d), F16), np.ascontiguousarray(k[:, a:b]), np.ascontiguousarray(v[:, a:b]), span=1)
    got = c.call(q, np.ascontiguousarray(k[:, count:]), np.ascontiguousarray(v[:, count:]), F32, span)
    c.check_rows()
    first = max(0, n - size) if ring else 0
    see = visible(count, tq, tq, first, min(span, size - tq + 1) if ring and span else span)
    K, V = stored(k[:, first:]), stored(v[:, first:])
    for h in range(hq):
        Kh, Vh, x = K[h * hkv // hq], V[h * hkv // hq], q[h].astype(np.float64)
        s = np.where(see, x @ Kh.T / np.sqrt(d), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        ds = np.where(see, np.abs(x) @ np.abs(Kh).T / np.sqrt(d), 0).max(-1, keepdims=True) * (d + 4) * 2.0 ** -24
        tol = p @ np.abs(Vh) * (4 * ds + 2.0 ** -21 + 4 * see.sum(1).max() * 2.0 ** -24)
        assert (np.abs(got[:, h] - p @ Vh) <= tol).all()
