"""How many rows of logits the check of drafted tokens takes: argument checks that need no GPU."""
import ctypes

import pytest

from test_paged_checks import UNSUPPORTED, verify_args
from vai_amd import _capi


@pytest.mark.parametrize("rows, vocab, taken", [
    ((1 << 24) - 1, 4096, True), ((1 << 23) - 1, 4097, True), (1 << 23, 4097, False), (1 << 22, 4 * 4096, False),
    ((1 << 22) - 1, 4 * 4096, True), (1 << 12, (1 << 24) - 1, False), ((1 << 12) - 1, (1 << 24) - 1, True),
])
def test_rows_of_logits(rows, vocab, taken):
    """A launch has fewer than 2^32 threads, 256 for each 4096 logits of a row."""
    a = verify_args(rows=rows, vocab=vocab)
    assert (_capi.lib().vai_verify_drafts_workspace_size(ctypes.byref(a)) > 0) == taken
    if not taken:
        assert _capi.lib().vai_verify_drafts_launch(ctypes.byref(a), None) == UNSUPPORTED
