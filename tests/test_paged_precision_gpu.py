"""How exact fp16 rows of attention over fp16 pages are. Values of +1 and -1 nearly cancel in every row, so that the
output's own rounding is small beside sum p |v| = 1 and a probability rounded to one fp16 number (2^-11) would show: the
tolerance is that of two (2^-21), the scores' and the sums', then the output's rounding."""
import numpy as np
import pytest

import test_paged_attention_gpu as att
from helpers import draw
from paged import Batch, F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d, page", [(64, 16), (80, 16), (128, 32), (256, 16)])
@pytest.mark.parametrize("new, held", [([130, 1, 3], [2, 30, 5]), ([1, 300], [70, 0]), ([1, 4, 1], [1, 2, 40])])
def test_probabilities_keep_their_bits(gpu, d, page, new, held):
    rng = np.random.default_rng(d)
    b = Batch(gpu, rng, new, held, 2, d, page, F16)
    b.fill(rng, loud=False)
    for s in range(len(new)):
        b.V[s][:] = np.where((np.arange(len(b.V[s]))[:, None, None] + np.arange(d)) % 2 == 0, 1, -1)
        b.store(s, b.K[s], b.V[s])
    b.upload()
    for qdt in (F16, F32):
        q = (draw((b.rows, 8, d), rng, F32) * F32(0.05)).astype(qdt)
        print(f"paged precision d={d} new={new}", flush=True)
        got = att.call(gpu, b, q, F16, max_new=max(new))
        for s, (n, h) in enumerate(zip(new, held)):
            at = int(b.starts[s])
            want, tol = att.attend(q[at:at + n], b.K[s], b.V[s], att.visible(h, n, 0), F16, F32)
            att.near(got[at:at + n], want, tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25, f"sequence {s}")


@pytest.mark.parametrize("d, page, pdt", [(64, 16, F16), (128, 32, F16), (256, 16, F16), (50, 12, F32)])
@pytest.mark.parametrize("new, held", [([1, 3], [400, 300]), ([80, 40], [400, 300])])
@pytest.mark.parametrize("at", [0, 299])
def test_probabilities_far_below_the_largest(gpu, d, page, pdt, new, held, at):
    """One position whose score is 16.5 above all others' and whose value is 0: the output is what the others, at
    probabilities of e^-16.5, make of it. (Two fp16 numbers after 2^14 hold them to 2^-25 of 2^-9.8, a tenth of the
    tolerance that a score of 16.5 has by itself.)"""
    rng = np.random.default_rng(d)
    b = Batch(gpu, rng, new, held, 2, d, page, pdt)
    b.fill(rng, loud=False)
    for s in range(len(new)):
        b.K[s][:, :, 0] = 0
        b.K[s][at, :, 0] = 16.5 * d ** 0.5
        b.V[s][:] = np.abs(b.V[s]) + 1
        b.V[s][at] = 0
        b.store(s, b.K[s], b.V[s])
    b.upload()
    for qdt in (F16, F32):
        q = np.zeros((b.rows, 8, d), qdt)
        q[:, :, 0] = 1
        print(f"paged precision far below d={d} new={new} at={at}", flush=True)
        att.check(b, q, att.call(gpu, b, q, F32, max_new=max(new)), F32)
