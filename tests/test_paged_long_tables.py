"""How long a table attention over pages takes: argument checks that need no GPU, and a prompt near what they allow."""
import ctypes

import numpy as np
import pytest

from test_paged_checks import UNSUPPORTED, attention_args
from vai_amd import _capi

HEADS = dict(hq=32, hkv=8, head_dim=128)


@pytest.mark.parametrize("kw, taken", [
    # one prompt as long as its table, in units of 128 rows and 64 positions: up to 2^32 of their pairs
    (dict(tokens=1 << 18, sequences=1, max_pages=1 << 14, **HEADS), True),
    (dict(tokens=1 << 19, sequences=1, max_pages=1 << 15, **HEADS), True),
    (dict(tokens=1 << 20, sequences=1, max_pages=1 << 16, **HEADS), False),
    # the same rows over fp32 pages, and over pages of no whole 16s: units of 16 rows and 32 positions
    (dict(tokens=1 << 17, sequences=1, max_pages=1 << 13, page_dtype=0, **HEADS), True),
    (dict(tokens=1 << 18, sequences=1, max_pages=1 << 14, page_dtype=0, **HEADS), False),
    (dict(tokens=1 << 18, sequences=1, max_pages=1 << 15, page_size=8, **HEADS), False),
    # single tokens: a unit each
    (dict(tokens=64, sequences=64, max_new=1, max_pages=1 << 21, **HEADS), True),
    (dict(tokens=64, sequences=64, max_new=1, max_pages=1 << 26, **HEADS), False),
])
def test_lengths(kw, taken):
    a = attention_args(**{"page_size": 16, **kw})
    assert (_capi.lib().vai_paged_attention_workspace_size(ctypes.byref(a)) > 0) == taken
    if not taken:
        assert _capi.lib().vai_paged_attention_launch(ctypes.byref(a), None) == UNSUPPORTED


def test_a_line_of_almost_2_to_the_32():
    """Its shares are its length divided and rounded up in 32 bits: lengths that this would carry past 2^32 are refused."""
    def taken(max_pages):
        a = attention_args(tokens=1, sequences=1, hq=65535, hkv=65535, head_dim=8, max_pages=max_pages, page_size=32)
        return _capi.lib().vai_paged_attention_workspace_size(ctypes.byref(a)) > 0

    # 65535 units of max_pages + 1 tiles and the 10 that stand before them
    most = (2 ** 32 - 1 - 1024) // 65535 - 11
    assert taken(most) and not taken(most + 1)
    assert 65535 * (most + 1 + 11) + 1024 >= 2 ** 32 > 65535 * (most + 11) + 1024


@pytest.mark.gpu
def test_a_long_prompt_and_a_long_table(gpu):
    """32768 rows over a table of 2^22 positions; some of the rows against their definition."""
    import test_paged_attention_gpu as att
    from helpers import draw
    from paged import F16, F32, Handle

    rng = np.random.default_rng(0)
    n, hq, hkv, d, page, used = 32768, 32, 8, 8, 4096, 8
    D = gpu.DeviceArray.from_numpy
    k, v = (draw((used, hkv, page, d), rng, F32).astype(F16) for _ in range(2))
    table = np.full((1, 1024), 0xffffffff, np.uint32)
    table[0, :used] = rng.permutation(used)
    q = draw((n, hq, d), rng, F32).astype(F16)
    out = gpu.DeviceArray((n, hq, d), F32)
    pages = gpu.kv_pages(D(k), D(v), D(table), D(np.array([0, n], np.uint32)), D(np.zeros(1, np.uint32)))
    print("paged attention, a long prompt", flush=True)
    gpu.paged_attention(out, D(q), pages)
    got = out.numpy()
    K, V = (x[table[0, :used]].transpose(0, 2, 1, 3).reshape(n, hkv, d) for x in (k, v))
    for row in (0, 1, 31, 32, 127, 128, 4095, 4096, 20001, n - 2, n - 1):
        see = np.arange(n)[None] <= row
        want, tol = att.attend(q[row:row + 1], K, V, see, F16, F32)
        att.near(got[row:row + 1], want, tol, f"row {row}")
