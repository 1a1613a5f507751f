"""The check of drafted tokens: tokens drawn exactly at borders, and greedy sequences whose draft model wants another
token than the target."""
import numpy as np
import pytest

import test_verify_drafts_gpu as ver
from helpers import draw
from paged import F16, F32

pytestmark = pytest.mark.gpu


def test_tokens_at_borders(gpu):
    """Probabilities of 1/4 each of tokens 1, 3, 4 and 6 (exact). A draft of token 3 without probabilities of its own is
    kept below u = 1/4, and the token after it is the first whose running sum is past u; from 1/4 on it is replaced by
    the first of 1, 4 and 6 whose running sum is past 3/4 u."""
    target = np.full((2, 8), -np.inf, F32)
    target[:, [1, 3, 4, 6]] = 0.0
    print("verify borders", flush=True)
    for u, kept, token in ((0.0, 1, 1), (0.2499, 1, 1), (0.25, 0, 1), (0.33, 0, 1), (0.34, 0, 4), (0.5, 0, 4), (0.66, 0, 4),
                           (0.67, 0, 6), (0.75, 0, 6), (0.99999994, 0, 6)):
        out, acc = ver.check(gpu, target, None, [0, 3], [u, u], [0, 2])
        assert acc[0] == kept and out[kept] == token
    for u, token in ((0.0, 1), (0.25, 3), (0.4999, 3), (0.5, 4), (0.75, 6), (0.99999994, 6)):
        out, acc = ver.check(gpu, target[:1], None, [0], [u], [0, 1])        # no draft: from p
        assert out[0] == token


@pytest.mark.parametrize("dt", [F16, F32])
def test_greedy_with_a_draft_model(gpu, dt):
    """T = 0 with logits of a draft model: a draft is kept where it is the target's choice, whatever the draft model's
    is; else the target's choice takes its place, also where a tie of the draft model's hides its own."""
    rng = np.random.default_rng(3)
    vocab, rows = 9000, 7
    target = draw((rows, vocab), rng, F32).astype(dt)
    draft = np.roll(target, 1, 0)
    target[np.arange(rows), 100 * np.arange(rows) + 4090] = 9      # the target's choices
    target[2, [8000, 8500]] = 9                                    # ties behind it
    draft[:, 17] = draft[:, 8999] = 9                              # the draft model's: 17
    choice = 100 * np.arange(rows) + 4090
    print(f"verify greedy with a draft model {np.dtype(dt).name}", flush=True)
    for drafts, kept in (([4090, 4190, 4290, 4390, 4490, 4590], 6), ([4090, 17, 4290, 4390, 4490, 4590], 1),
                         ([17] * 6, 0), ([8999] * 6, 0), ([4090, 4190, 8000, 4390, 4490, 4590], 2)):
        for u in (0.0, 0.5, 0.99999994):
            out, acc = ver.check(gpu, target, draft, [5] + drafts, [u] * rows, [0, rows], [0.0])
            assert acc[0] == kept and out[kept] == choice[kept]


def test_temperatures_that_are_not_above_zero(gpu):
    """They are 0: greedy. An infinite one makes every logit above -infinity equally likely."""
    rng = np.random.default_rng(4)
    temps = [-1.0, np.nan, -0.0, -np.inf, np.inf, 1e-45]
    args = ver.batch(rng, 5000, [3, 3, 3, 3, 3, 3], F32, True, [0.0] * 4 + [1e30, 0.0])
    args[0][:, 40:50] = -np.inf
    print("verify temperatures", flush=True)
    ver.check(gpu, *args, temps)
