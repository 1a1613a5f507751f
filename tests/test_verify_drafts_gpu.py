"""Drafted tokens against the target's probabilities (vai_verify_drafts_launch),
token for token against the definition in 64 bits.

A result could differ only where a random number falls within the roundings of
64 bits of a border: 2^-45 of the running sum over 50000 tokens at most, which a
random number given in fp32 meets by chance once in 10^9 draws, or on purpose
(those cases are exact in 64 bits: probabilities that are powers of two)."""
import ctypes

import numpy as np
import pytest

from helpers import draw
from paged import F16, F32, Handle

pytestmark = pytest.mark.gpu
NO = 0xffffffff


def spread(x, t):
    """None: no distribution"""
    x = x.astype(np.float64)
    if not (x < np.inf).all() or not (x > -np.inf).any():
        return None
    if not t > 0:
        return (np.arange(len(x)) == x.argmax()).astype(np.float64)
    e = np.where(x == -np.inf, 0.0, np.exp((x - x.max()) / float(t)))
    return e / e.sum()


def verify(target, draft, tokens, uniform, starts, temps):
    """-> (out_tokens with None where nothing is written, accepted)"""
    out, kept = [None] * len(target), []
    for s in range(len(starts) - 1):
        a, b = int(starts[s]), int(starts[s + 1])
        t = 1.0 if temps is None else temps[s]
        if b <= a:
            kept.append(None)
            continue
        r, token = a, NO
        while True:
            p = spread(target[r], t)
            if p is None:
                break
            w = p
            if r < b - 1:
                x = int(tokens[r + 1])
                q = (np.arange(len(p)) == x).astype(np.float64) if draft is None else spread(draft[r], t)
                if q is None:
                    break
                px = p[x] if x < len(p) else 0.0
                qx = 1.0 if draft is None else q[x] if x < len(p) else 0.0
                if float(uniform[r]) * qx < px:
                    r += 1
                    continue
                rest = np.maximum(p - q, 0)
                w = rest if rest.sum() > 0 else p
            c = np.cumsum(w)
            past = np.flatnonzero((c > float(uniform[b - 1]) * c[-1]) & (w > 0))
            token = int(past[0]) if len(past) else int(np.flatnonzero(w)[-1])
            break
        for i in range(a, b):
            out[i] = int(tokens[i + 1]) if i < r else token if i == r else NO
        kept.append(r - a)
    return out, kept


def run(gpu, target, draft, tokens, uniform, starts, temps=None, counts=None, alias=False, stride=0):
    D = gpu.DeviceArray.from_numpy
    rows, vocab = target.shape
    n = len(starts) - 1

    def wide(x):
        if x is None:
            return None
        y = np.full((rows, vocab + stride), np.nan, x.dtype)
        y[:, :vocab] = x
        return Handle(D(y), x.shape, x.dtype)

    out, kept = D(np.full(rows, 7777, np.uint32)), D(np.full(n, 7777, np.uint32))
    c = None if counts is None else D(np.array(counts, np.uint32))
    new = c if alias else None if counts is None else D(np.full(n, 7777, np.uint32))
    a = gpu.verify_drafts_args(out, kept, wide(target), D(np.array(tokens, np.uint32)), D(np.array(uniform, F32)),
                               D(np.array(starts, np.uint32)), draft=wide(draft),
                               temperature=None if temps is None else D(np.array(temps, F32)), counts=c, new_counts=new)
    if stride:
        a.target_stride = a.draft_stride = vocab + stride
    need = gpu.lib().vai_verify_drafts_workspace_size(ctypes.byref(a))
    ws = gpu.DeviceArray((need,), np.uint8)
    ws.fill_(0xFF)
    a.workspace, a.workspace_bytes = ws.ptr, need
    gpu.check(gpu.lib().vai_verify_drafts_launch(ctypes.byref(a), None), "verify")
    gpu.synchronize()
    return out.numpy(), kept.numpy(), None if new is None else new.numpy()


def check(gpu, target, draft, tokens, uniform, starts, temps=None, **kw):
    n = len(starts) - 1
    counts = [100 * s + 3 for s in range(n)]
    out, kept, new = run(gpu, target, draft, tokens, uniform, starts, temps, counts, **kw)
    temps32 = None if temps is None else np.array(temps, F32)
    want, acc = verify(target, draft, tokens, np.array(uniform, F32), starts, temps32)
    np.testing.assert_array_equal(out, [7777 if x is None else x for x in want])
    np.testing.assert_array_equal(kept, [x or 0 for x in acc])
    np.testing.assert_array_equal(new, [c if x is None else c + x + 1 for c, x in zip(counts, acc)])
    return out, kept


def batch(rng, vocab, lens, dt, with_draft, temps, pad=2, lead=1):
    starts = np.concatenate([[lead], lead + np.cumsum(lens)])
    rows = int(starts[-1]) + pad
    target = (2.5 * draw((rows, vocab), rng, F32)).astype(dt)
    d = (target.astype(F32) + 0.7 * draw((rows, vocab), rng, F32)).astype(dt) if with_draft else None
    tokens = rng.integers(0, vocab, rows)
    for s in range(len(lens)):
        for r in range(int(starts[s]), int(starts[s + 1]) - 1):
            p = spread((d if with_draft else target)[r], temps[s])
            tokens[r + 1] = rng.choice(vocab, p=p)
    return target, d, tokens, rng.uniform(0, 1, rows).astype(F32), starts


@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 4095, 4096, 4097, 50021])
@pytest.mark.parametrize("dt, with_draft", [(F16, True), (F32, True), (F32, False)])
def test_verify(gpu, vocab, dt, with_draft):
    rng = np.random.default_rng(vocab)
    lens = [1, 4, 0, 6, 9, 2, 1]
    temps = [1.0, 0.7, 1.0, 0.0, 0.9, 1.5, 0.0]
    for turn in range(3):
        args = batch(rng, vocab, lens, dt, with_draft, temps)
        print(f"verify vocab={vocab} turn={turn}", flush=True)
        check(gpu, *args, temps)
        check(gpu, *args)


@pytest.mark.parametrize("stride", [1, 24])
def test_rows_apart_and_counts_in_place(gpu, stride):
    rng = np.random.default_rng(stride)
    args = batch(rng, 1000, [3, 5, 2], F16, True, [1.0] * 3)
    print("verify strides", flush=True)
    check(gpu, *args, stride=stride)
    check(gpu, *args, alias=True)


def test_what_is_drafted_from_the_same_model_is_kept(gpu):
    rng = np.random.default_rng(0)
    target, _, _, u, starts = batch(rng, 5000, [8, 8], F32, False, [0.8, 0.8])
    tokens = np.zeros(len(target), int)
    for r in range(len(target) - 1):
        tokens[r + 1] = rng.choice(5000, p=spread(target[r], 0.8))
    print("verify equal", flush=True)
    _, kept = check(gpu, target, target.copy(), tokens, u, starts, [0.8, 0.8])
    assert list(kept) == [7, 7]


def test_borders(gpu):
    """Probabilities of 1/4 each (exact): u q < p decides at equality, and a running sum that equals u * total is not
    past it. u = 0 keeps whatever has a probability and draws the first that has."""
    vocab, ninf = 8, -np.inf
    target = np.full((4, vocab), ninf, F32)
    target[:, [1, 3, 4, 6]] = 0.0
    starts = [0, 2, 4]
    print("verify borders", flush=True)
    for u, kept, token in ((0.0, 1, 1), (0.2499, 1, 1), (0.25, 0, 3), (0.5, 0, 4), (0.75, 0, 6), (0.99999994, 0, 6)):
        # a draft of token 3 without probabilities of its own: kept below 1/4
        uniform = [u, 0.25, u, u]
        out, acc = check(gpu, target, None, [0, 3, 0, 3], uniform, starts)
        assert acc[0] == kept
    # a refused draft's replacement: w = p without the draft, 1/4 each of 1, 4, 6, of 3/4 in all
    for u, token in ((0.0, 1), (0.3, 1), (0.34, 4), (0.66, 4), (0.67, 6), (0.99999994, 6)):
        out, acc = check(gpu, target, None, [0, 3, 0, 3], [0.9, u, 0.9, u], starts)
        assert acc[0] == 0 and out[0] == token


def test_ties_and_greedy(gpu):
    """T = 0: the lowest index of the largest logit, -0 and 0 alike, in whatever part of the row they are."""
    vocab = 9000
    target = np.zeros((6, vocab), F16)
    target[:, ::2] = -0.0
    target[1, [70, 5000, 8999]] = 3
    target[2, [4096, 4097]] = 3
    target[3] = -np.inf
    target[3, 8000] = -65504
    tokens = [0, 0, 70, 4096, 8000, 5]
    print("verify ties", flush=True)
    out, kept = check(gpu, target, None, tokens, [0.5] * 6, [0, 6], [0.0])
    assert kept[0] == 4 and out[4] == 0
    out, kept = check(gpu, target, np.roll(target, 0, 0), tokens, [0.5] * 6, [0, 6], [0.0])
    assert kept[0] == 4


@pytest.mark.parametrize("vocab", [6, 5000])
def test_rows_without_a_distribution(gpu, vocab):
    """NaN, +infinity or nothing above -infinity ends a sequence without a token, where the row is needed."""
    rng = np.random.default_rng(vocab)
    for dt in (F16, F32):
        target, d, tokens, u, starts = batch(rng, vocab, [3, 3, 3, 3, 3], dt, True, [1.0] * 5, pad=0, lead=0)
        u[:] = 0                            # every draft of some probability is kept
        target[1, vocab // 2] = np.nan
        target[5, vocab - 1] = np.inf
        target[6] = -np.inf
        d[10, 0] = np.nan
        d[14, 0] = np.nan                   # a last row's draft is not read
        target[12:15, :2] = -np.inf
        tokens[13], tokens[14] = 0, 1       # a draft without a probability: refused; what follows does not matter
        target[13, 3] = np.nan
        print(f"verify without a distribution vocab={vocab}", flush=True)
        out, kept = check(gpu, target, d, tokens, u, starts)
        assert out[1] == NO and out[5] == NO and out[6] == NO and out[10] == NO and list(kept) == [1, 2, 0, 1, 0]
        check(gpu, target, d, tokens, u, starts, [0.0] * 5)


def test_odd_inputs(gpu):
    """Tokens past the vocabulary, drafts that their own distribution rules out, extreme temperatures and logits."""
    rng = np.random.default_rng(1)
    vocab = 700
    target, d, tokens, u, starts = batch(rng, vocab, [3, 4, 2, 3, 3, 3], F32, True, [1.0] * 6, pad=0, lead=0)
    tokens[1], tokens[4] = vocab, 2 ** 32 - 1
    d[7, 5] = -np.inf
    tokens[8] = 5
    target[9:12] *= 1e30
    d[9:12] *= 1e30
    print("verify odd inputs", flush=True)
    temps = [1.0, 1.0, 1.0, 1.0, 1e-30, 1e30]
    check(gpu, target, d, tokens, u, starts, temps)
    check(gpu, target, None, tokens, u, starts, temps)
    # p and q alike, and a draft outside both: nothing is left of p - q, so from p
    d[0] = target[0]
    check(gpu, target, d, tokens, u, starts, temps)


def test_replayed_graph(gpu):
    """A recorded launch follows starts, tokens, random numbers and counts; counts advance in place."""
    rng = np.random.default_rng(5)
    vocab, D = 5000, gpu.DeviceArray.from_numpy
    target, d, tokens, u, _ = batch(rng, vocab, [5, 5], F16, True, [1.0] * 2, pad=0, lead=0)
    dev = [D(x) for x in (target, d, tokens.astype(np.uint32), u)]
    starts, counts = D(np.array([0, 5, 10], np.uint32)), D(np.array([11, 50], np.uint32))
    out, kept = D(np.zeros(10, np.uint32)), D(np.zeros(2, np.uint32))
    a = gpu.verify_drafts_args(out, kept, dev[0], dev[2], dev[3], starts, draft=dev[1], counts=counts, new_counts=counts)
    n = gpu.lib().vai_verify_drafts_workspace_size(ctypes.byref(a))
    ws = gpu.DeviceArray((n,), np.uint8)
    a.workspace, a.workspace_bytes = ws.ptr, n
    stream = gpu.Stream()
    graph = gpu.Graph(stream, lambda: gpu.check(gpu.lib().vai_verify_drafts_launch(ctypes.byref(a), stream.ptr), "x"))
    held = np.array([11, 50])
    for begin in ([0, 5, 10], [0, 1, 10], [0, 0, 7], [2, 6, 9]):
        u = rng.uniform(0, 1, 10).astype(F32)
        for dst, src in ((starts, np.array(begin, np.uint32)), (dev[3], u)):
            gpu.check(gpu.lib().vai_memcpy_h2d(dst.ptr, src.ctypes.data, src.nbytes, None), "h2d")
        print(f"verify replay {begin}", flush=True)
        graph.launch()
        stream.synchronize()
        want, acc = verify(target, d, tokens, u, begin, None)
        got = out.numpy()
        for g, w in zip(got, want):
            assert w is None or g == w
        held = [h if x is None else h + x + 1 for h, x in zip(held, acc)]
        np.testing.assert_array_equal(counts.numpy(), held)
