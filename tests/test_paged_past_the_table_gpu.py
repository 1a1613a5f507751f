"""Attention over pages where counts are past what the table holds (drafts that were kept advance them without regard
to it): a query is at counts[s] + t, its window is counted from there, and positions past the table hold nothing."""
import numpy as np
import pytest

import test_paged_attention_gpu as att
from helpers import draw
from paged import Batch, F16, F32

pytestmark = pytest.mark.gpu


def full(gpu, rng, new, room, hkv, d, page, pdt):
    """A batch whose table has room positions, all of them with values."""
    b = Batch(gpu, rng, new, [room - n for n in new], hkv, d, page, pdt, pad=1)
    b.fill(rng)
    b.table = np.ascontiguousarray(b.table[:, :room // page])
    assert (b.table < b.num_pages).all()
    b.upload()
    return b


def seen(room, count, n, span, causal):
    """In Python's integers: [n, room]"""
    return np.array([[j < count + n and (not causal or j <= count + t) and (span == 0 or j > count + t - span)
                      for j in range(room)] for t in range(n)])


def check(gpu, b, q, room, counts, span, causal, odt, **kw):
    b.upload_tables(counts)
    got = att.call(gpu, b, q, odt, span=span, causal=causal, **kw)
    for s, n in enumerate(b.new):
        at, see = int(b.starts[s]), seen(room, counts[s], n, span, causal)
        want, tol = att.attend(q[at:at + n], b.K[s], b.V[s], see, b.dt, odt)
        att.near(got[at:at + n], want, tol, f"sequence {s} counts {counts[s]} span {span} causal {causal}")
        assert (got[at:at + n][~see.any(-1)] == 0).all()


@pytest.mark.parametrize("d, page, room, pdt", [(64, 16, 192, F16), (128, 32, 192, F16), (256, 16, 160, F16), (50, 12, 180, F32),
                                                (33, 6, 90, F16)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 1, 2, 4], [70, 3, 40, 34]])
def test_counts_past_the_table(gpu, d, page, room, pdt, new):
    """Windows that end before, at and inside what the table holds; sequences on both sides of its end in one call."""
    rng = np.random.default_rng(d)
    b = full(gpu, rng, new, room, 2, d, page, pdt)
    for qdt, odt in ((F16, F16), (F32, F32)):
        q = draw((b.rows, 8, d), rng, qdt)
        for counts in ([room + 36, room, room - 1, room + 7], [room - 20, 2 ** 31 - 1, 2 ** 31 + 5, room + 2 ** 30]):
            for span, causal in ((10, True), (37, True), (0, True), (60, False), (room, True), (room + 36, False)):
                print(f"past the table d={d} new={new} counts={counts} span={span} causal={causal}", flush=True)
                check(gpu, b, q, room, counts, span, causal, odt, max_new=max(new))


@pytest.mark.parametrize("d, page, room, pdt", [(64, 16, 192, F16), (50, 12, 180, F32)])
@pytest.mark.parametrize("new", [[1, 2], [70, 33]])
def test_positions_past_32_bits(gpu, d, page, room, pdt, new):
    """A position and a window at the end of what 32 bits hold, or past it by the call's own rows."""
    rng = np.random.default_rng(d)
    b = full(gpu, rng, new, room, 2, d, page, pdt)
    q = draw((b.rows, 8, d), rng, F16)
    for counts, span in (([2 ** 32 - 1, 2 ** 32 - 40], 2 ** 32 - 1), ([2 ** 32 - 2, 2 ** 32 - 60], 2 ** 32 - 100),
                         ([2 ** 31 + 50, 2 ** 31 - 20], 2 ** 31)):
        print(f"past 32 bits d={d} new={new} counts={counts} span={span}", flush=True)
        check(gpu, b, q, room, counts, span, True, F32)
