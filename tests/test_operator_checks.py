"""Refusals and sizes of the 8-bit Linear, the head norms and the 4-bit cache:
argument checks that need no GPU."""
import ctypes

import numpy as np
import pytest

from vai_amd import _capi

INVALID, SHAPE, DTYPE, WORKSPACE, UNSUPPORTED = 1001, 1002, 1003, 1004, 1005


def linear_i8_args(**kw):
    a = _capi.LinearI8Args()
    a.out = a.inp = a.weight = a.w_scale = a.workspace = 256
    a.M, a.N, a.K, a.b_dtype, a.scalar_scale = 40, 32, 100, 2, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("want, kw", [
    (INVALID, dict(out=None)), (INVALID, dict(inp=None)), (INVALID, dict(weight=None)), (INVALID, dict(w_scale=None)),
    (SHAPE, dict(M=0)), (SHAPE, dict(N=0)), (SHAPE, dict(K=0)), (UNSUPPORTED, dict(K=131073)),
    (UNSUPPORTED, dict(M=1 << 21)), (DTYPE, dict(o_dtype=2)), (DTYPE, dict(i_dtype=3)), (DTYPE, dict(bias=256)),
    (INVALID, dict(epilogue=6)), (INVALID, dict(residual_order=2)), (INVALID, dict(weight=264)),
    (SHAPE, dict(bias=256, b_dtype=0, bias_repeat=33)), (SHAPE, dict(residual=256, residual_repeat=32 * 7)),
    (WORKSPACE, dict()), (WORKSPACE, dict(workspace=None, workspace_bytes=1 << 30)),
    (INVALID, dict(workspace=257, workspace_bytes=1 << 30)),
])
def test_linear_i8_refusals(want, kw):
    assert _capi.lib().vai_linear_i8_launch(ctypes.byref(linear_i8_args(**kw)), None) == want


def test_linear_i8_null_and_python_checks():
    lib = _capi.lib()
    assert lib.vai_linear_i8_launch(None, None) == INVALID
    assert lib.vai_linear_i8_workspace_size(None) == 0
    assert lib.vai_linear_i8_workspace_size(ctypes.byref(linear_i8_args(K=0))) == 0
    # the rounded rows of X and their scales fit
    assert lib.vai_linear_i8_workspace_size(ctypes.byref(linear_i8_args())) >= 40 * (100 + 4)

    class Handle:
        def __init__(self, shape, code):
            self.shape, self.code, self.ptr = shape, code, 256

    with pytest.raises(_capi.VaiError, match="112 expected"):
        _capi.linear_i8_args(Handle((2, 8), 0), Handle((2, 100), 0), Handle((8, 100), None), Handle((8,), 0))


@pytest.mark.parametrize("want, args", [
    (INVALID, (None, 256, 256, 0, 1, 16)), (INVALID, (256, None, 256, 0, 1, 16)), (INVALID, (256, 256, None, 0, 1, 16)),
    (DTYPE, (256, 256, 256, 2, 1, 16)), (SHAPE, (256, 256, 256, 0, 0, 16)), (SHAPE, (256, 256, 256, 0, 1, 0)),
    (UNSUPPORTED, (256, 256, 256, 0, 1, 131073)), (INVALID, (260, 256, 256, 0, 1, 16))])
def test_quantize_refusals(want, args):
    assert _capi.lib().vai_quantize_i8_launch(*args, None) == want


def rope_args(**kw):
    a = _capi.QkNormRopeArgs()
    a.q_out = a.k_out = a.v_out = a.qkv = 256
    a.batch, a.tokens, a.hq, a.hkv, a.head_dim, a.rope, a.theta, a.norm, a.w_dtype = 1, 2, 4, 2, 64, 1, 1e4, 1, 2
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("want, kw", [
    (INVALID, dict(q_out=None)), (INVALID, dict(k_out=None)), (INVALID, dict(qkv=None)),
    (DTYPE, dict(i_dtype=2)), (DTYPE, dict(o_dtype=3)), (DTYPE, dict(q_weight=256)),
    (INVALID, dict(rope=3)), (INVALID, dict(norm=2)), (INVALID, dict(theta=0.0)), (INVALID, dict(theta=float("nan"))),
    (INVALID, dict(theta=float("inf"))), (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=float("nan"))),
    (SHAPE, dict(batch=0)), (SHAPE, dict(tokens=0)), (SHAPE, dict(hq=0)), (SHAPE, dict(hkv=0)), (SHAPE, dict(head_dim=0)),
    (SHAPE, dict(rot_dim=66)), (SHAPE, dict(rot_dim=7)), (SHAPE, dict(head_dim=65)), (SHAPE, dict(row_stride=8 * 64 - 1)),
    (UNSUPPORTED, dict(head_dim=2050)), (UNSUPPORTED, dict(hq=65536)),
])
def test_qk_norm_rope_refusals(want, kw):
    assert _capi.lib().vai_qk_norm_rope_launch(ctypes.byref(rope_args(**kw)), None) == want


def test_qk_norm_rope_null_and_python_checks():
    assert _capi.lib().vai_qk_norm_rope_launch(None, None) == INVALID

    class Handle:
        def __init__(self, shape, code):
            self.shape, self.code, self.ptr = shape, code, 256

    q, k, x = Handle((4, 2, 64), 0), Handle((2, 2, 64), 0), Handle((2, 512), 0)
    with pytest.raises(_capi.VaiError, match="share a dtype"):
        _capi.qk_norm_rope_args(q, k, None, x, Handle((64,), 0), Handle((64,), 1))
    with pytest.raises(_capi.VaiError, match="share a dtype"):
        _capi.qk_norm_rope_args(q, Handle((2, 2, 64), 1), None, x)


def q4_args(**kw):
    a = _capi.AttentionArgs()
    a.out = a.q = a.k = a.v = a.k_cache = a.v_cache = a.cache_count = 256
    a.batch, a.hq, a.hkv, a.tq, a.tkv, a.head_dim = 1, 4, 2, 1, 1, 64
    a.q_dtype = a.kv_dtype = a.o_dtype = 1
    a.cache_size, a.cache_dtype = 128, _capi.Q4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("want, kw", [
    (INVALID, dict(k_cache=None)), (INVALID, dict(cache_count=None)), (INVALID, dict(k_cache=264)),
    (INVALID, dict(v_cache=264)), (INVALID, dict(k=None)), (DTYPE, dict(kv_dtype=3)), (DTYPE, dict(q_dtype=3)),
    (DTYPE, dict(o_dtype=3)), (SHAPE, dict(batch=2)), (SHAPE, dict(tkv=129)), (SHAPE, dict(cache_ring=1, cache_size=100)),
    (SHAPE, dict(cache_ring=1, tkv=129)), (SHAPE, dict(hq=3)), (UNSUPPORTED, dict(head_dim=257)),
    (WORKSPACE, dict(tq=100, tkv=100)), (DTYPE, dict(cache_size=0, kv_dtype=3)),
])
def test_q4_attention_refusals(want, kw):
    assert _capi.lib().vai_attention_launch(ctypes.byref(q4_args(**kw)), None) == want


def test_cache_sizes():
    """5 bits a value in rows of 64, 128 or 256, positions in tiles of 32."""
    assert _capi.attention_cache_bytes(8, 4096, 128, _capi.Q4) == 8 * 4096 * 80
    assert _capi.attention_cache_bytes(2, 33, 64, _capi.Q4) == 2 * 64 * 40
    assert _capi.attention_cache_bytes(1, 1, 65, _capi.Q4) == 32 * 80
    assert _capi.attention_cache_bytes(1, 131072 * 64, 256, _capi.Q4) == 131072 * 64 * 160   # past 2^30
    assert _capi.attention_cache_bytes(1, 32, 257, _capi.Q4) == 0
    assert _capi.attention_cache_bytes(0, 32, 64, _capi.Q4) == 0
    assert _capi.attention_cache_bytes(2, 33, 64, _capi.F16) == 2 * 33 * 64 * 2
    assert _capi.attention_cache_bytes(2, 33, 1000, _capi.F32) == 2 * 33 * 1000 * 4
    assert _capi.attention_cache_bytes(2, 33, 64, _capi.NONE) == 0
    with pytest.raises(_capi.VaiError, match="no cache"):
        _capi.CachePlane(1, 32, 300, _capi.Q4)


@pytest.mark.parametrize("want, kw", [
    (INVALID, dict(k_out=None)), (INVALID, dict(v_cache=None)), (DTYPE, dict(o_dtype=3)), (DTYPE, dict(cache_dtype=2)),
    (SHAPE, dict(hkv=0)), (SHAPE, dict(rows=0)), (SHAPE, dict(rows=65)), (SHAPE, dict(first_row=64)),
    (SHAPE, dict(head_dim=0)), (UNSUPPORTED, dict(head_dim=300)), (INVALID, dict(k_cache=264))])
def test_cache_read_refusals(want, kw):
    a = _capi.AttentionCacheReadArgs()
    a.k_out = a.v_out = a.k_cache = a.v_cache = 256
    a.cache_dtype, a.hkv, a.cache_size, a.head_dim, a.rows = _capi.Q4, 2, 64, 64, 1
    for k, v in kw.items():
        setattr(a, k, v)
    assert _capi.lib().vai_attention_cache_read(ctypes.byref(a), None) == want


def test_struct_sizes_match_the_header():
    """ctypes' layout of the argument structs is the compiler's (sizes worked from the header's fields)."""
    assert ctypes.sizeof(_capi.LinearI8Args) == 8 * 8 + 11 * 4 + 4
    assert ctypes.sizeof(_capi.AttentionCacheReadArgs) == 4 * 8 + 7 * 4 + 4
    assert ctypes.sizeof(_capi.QkNormRopeArgs) == 9 * 8 + 15 * 4 + 4
    assert np.dtype(np.int8).itemsize == 1
