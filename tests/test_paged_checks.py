"""Refusals and sizes of the operators over a KV cache in pages and of the check
of drafted tokens: argument checks that need no GPU."""
import ctypes

import pytest

from vai_amd import _capi

INVALID, SHAPE, DTYPE, WORKSPACE, UNSUPPORTED = 1001, 1002, 1003, 1004, 1005


def change(a, kw):
    for k, v in kw.items():
        setattr(a if hasattr(type(a), k) else a.pages, k, v)
    return a


def pages():
    p = _capi.KvPages()
    p.k_pages = p.v_pages = p.page_table = p.seq_start = p.counts = 256
    p.sequences, p.num_pages, p.page_size, p.max_pages, p.page_dtype = 2, 10, 16, 4, 1
    return p


def append_args(**kw):
    a = _capi.PagedAppendArgs()
    a.q_out = a.qkv = 256
    a.pages = pages()
    a.tokens, a.hq, a.hkv, a.head_dim, a.rope, a.theta, a.norm, a.w_dtype = 3, 4, 2, 64, 1, 1e4, 1, 2
    return change(a, kw)


def attention_args(**kw):
    a = _capi.PagedAttentionArgs()
    a.out = a.q = a.workspace = 256
    a.workspace_bytes = 1 << 40
    a.pages = pages()
    a.tokens, a.hq, a.hkv, a.head_dim, a.causal, a.q_dtype, a.o_dtype = 3, 4, 2, 64, 1, 1, 1
    return change(a, kw)


PAGES = [
    (INVALID, dict(k_pages=None)), (INVALID, dict(v_pages=None)), (INVALID, dict(page_table=None)),
    (INVALID, dict(seq_start=None)), (INVALID, dict(counts=None)), (DTYPE, dict(page_dtype=2)), (DTYPE, dict(page_dtype=3)),
    (SHAPE, dict(sequences=0)), (SHAPE, dict(num_pages=0)), (SHAPE, dict(page_size=0)), (SHAPE, dict(max_pages=0)),
    (UNSUPPORTED, dict(sequences=4097)), (UNSUPPORTED, dict(max_pages=(1 << 26) + 1)),
    (UNSUPPORTED, dict(max_pages=0xffffffff, page_size=0xffffffff)), (SHAPE, dict(page_stride=2 * 16 * 64 - 1)),
    (UNSUPPORTED, dict(page_stride=1 << 58)),
]


@pytest.mark.parametrize("want, kw", PAGES + [
    (INVALID, dict(qkv=None)), (DTYPE, dict(i_dtype=2)), (DTYPE, dict(o_dtype=3)), (DTYPE, dict(q_weight=256)),
    (INVALID, dict(rope=3)), (INVALID, dict(norm=2)), (INVALID, dict(theta=0.0)), (INVALID, dict(theta=float("nan"))),
    (INVALID, dict(eps=-1.0)), (SHAPE, dict(tokens=0)), (SHAPE, dict(hq=0)), (SHAPE, dict(hkv=0)), (SHAPE, dict(head_dim=0)),
    (SHAPE, dict(rot_dim=66)), (SHAPE, dict(rot_dim=7)), (SHAPE, dict(head_dim=65)), (SHAPE, dict(row_stride=8 * 64 - 1)),
    (UNSUPPORTED, dict(head_dim=2050)), (UNSUPPORTED, dict(hq=65536)), (UNSUPPORTED, dict(tokens=1 << 31)),
])
def test_append_refusals(want, kw):
    assert _capi.lib().vai_paged_append_launch(ctypes.byref(append_args(**kw)), None) == want


@pytest.mark.parametrize("want, kw", PAGES + [
    (INVALID, dict(out=None)), (INVALID, dict(q=None)), (DTYPE, dict(q_dtype=2)), (DTYPE, dict(o_dtype=3)),
    (SHAPE, dict(tokens=0)), (SHAPE, dict(hq=0)), (SHAPE, dict(hkv=0)), (SHAPE, dict(head_dim=0)), (SHAPE, dict(hq=3)),
    (SHAPE, dict(q_stride=4 * 64 - 1)), (UNSUPPORTED, dict(head_dim=257)), (INVALID, dict(causal=2)),
    (INVALID, dict(scale=float("nan"))), (UNSUPPORTED, dict(tokens=1 << 30)),
    (UNSUPPORTED, dict(tokens=1 << 20, max_pages=1 << 26)),
    (WORKSPACE, dict(workspace=None)), (WORKSPACE, dict(workspace_bytes=64)), (INVALID, dict(workspace=264)),
])
def test_attention_refusals(want, kw):
    assert _capi.lib().vai_paged_attention_launch(ctypes.byref(attention_args(**kw)), None) == want


def verify_args(**kw):
    a = _capi.VerifyDraftsArgs()
    a.out_tokens = a.accepted = a.target = a.tokens = a.uniform = a.seq_start = a.workspace = 256
    a.workspace_bytes = 1 << 40
    a.sequences, a.rows, a.vocab = 2, 6, 1000
    return change(a, kw)


@pytest.mark.parametrize("want, kw", [
    (INVALID, dict(out_tokens=None)), (INVALID, dict(accepted=None)), (INVALID, dict(target=None)),
    (INVALID, dict(tokens=None)), (INVALID, dict(uniform=None)), (INVALID, dict(seq_start=None)),
    (INVALID, dict(new_counts=256)), (DTYPE, dict(target_dtype=2)), (DTYPE, dict(draft=256, draft_dtype=3)),
    (SHAPE, dict(sequences=0)), (SHAPE, dict(rows=0)), (SHAPE, dict(vocab=0)), (SHAPE, dict(target_stride=999)),
    (SHAPE, dict(draft=256, draft_stride=999)), (UNSUPPORTED, dict(sequences=4097)), (UNSUPPORTED, dict(rows=1 << 24)),
    (UNSUPPORTED, dict(vocab=1 << 24)), (UNSUPPORTED, dict(rows=1 << 20, vocab=1 << 23)),
    (WORKSPACE, dict(workspace=None)), (WORKSPACE, dict(workspace_bytes=64)), (INVALID, dict(workspace=264)),
])
def test_verify_refusals(want, kw):
    assert _capi.lib().vai_verify_drafts_launch(ctypes.byref(verify_args(**kw)), None) == want


def test_null_arguments_and_sizes():
    L = _capi.lib()
    assert L.vai_paged_append_launch(None, None) == L.vai_paged_attention_launch(None, None) == INVALID
    assert L.vai_verify_drafts_launch(None, None) == INVALID
    assert L.vai_paged_attention_workspace_size(None) == L.vai_verify_drafts_workspace_size(None) == 0
    assert L.vai_paged_attention_workspace_size(ctypes.byref(attention_args(hq=3))) == 0
    assert L.vai_verify_drafts_workspace_size(ctypes.byref(verify_args(vocab=0))) == 0
    # a refused size is 0, an accepted one is not; both do not depend on the workspace given
    assert L.vai_paged_attention_workspace_size(ctypes.byref(attention_args(workspace=None))) > 0
    assert L.vai_verify_drafts_workspace_size(ctypes.byref(verify_args(workspace=None))) > 0


def test_struct_sizes_match_the_header():
    """ctypes' layout of the argument structs is the compiler's (sizes worked from the header's fields)."""
    assert ctypes.sizeof(_capi.KvPages) == 6 * 8 + 5 * 4 + 4
    assert ctypes.sizeof(_capi.PagedAppendArgs) == 5 * 8 + 72 + 14 * 4
    assert ctypes.sizeof(_capi.PagedAttentionArgs) == 4 * 8 + 72 + 11 * 4 + 4
    assert ctypes.sizeof(_capi.VerifyDraftsArgs) == 12 * 8 + 7 * 4 + 4


def test_python_checks():
    class Handle:
        def __init__(self, shape, code=1):
            self.shape, self.code, self.ptr = shape, code, 256

    k, table = Handle((10, 2, 16, 64)), Handle((3, 4))
    good = _capi.kv_pages(k, k, table, Handle((4,)), Handle((3,)))
    with pytest.raises(_capi.VaiError, match="dtype and a shape"):
        _capi.kv_pages(k, Handle((10, 2, 16, 64), 0), table, Handle((4,)), Handle((3,)))
    with pytest.raises(_capi.VaiError, match="counts"):
        _capi.kv_pages(k, k, table, Handle((3,)), Handle((3,)))
    with pytest.raises(_capi.VaiError, match="heads of 32"):
        _capi.paged_append_args(Handle((5, 4, 32)), Handle((5, 8 * 32)), good)
    with pytest.raises(_capi.VaiError, match="share a dtype"):
        _capi.paged_append_args(Handle((5, 4, 64)), Handle((5, 8 * 64)), good, Handle((64,), 0), Handle((64,), 1))
    with pytest.raises(_capi.VaiError, match="heads of 32"):
        _capi.paged_attention_args(Handle((5, 4, 32)), Handle((5, 4, 32)), good)
    rows = Handle((6, 100))
    with pytest.raises(_capi.VaiError, match="6 rows"):
        _capi.verify_drafts_args(Handle((5,)), Handle((2,)), rows, Handle((6,)), Handle((6,)), Handle((3,)))
    with pytest.raises(_capi.VaiError, match="2 sequences"):
        _capi.verify_drafts_args(Handle((6,)), Handle((3,)), rows, Handle((6,)), Handle((6,)), Handle((3,)))
