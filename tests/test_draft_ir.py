"""CPU checks of the MXFP4 type and the drafted-token ops: sizes, strides, views,
refused constructors, supports_op, the import by name."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref


@pytest.fixture
def ctx(wx):
    c = wx.load().wamx_init(512)
    yield c
    wx.load().wamx_free(c)


def test_mxfp4_sizes_and_views(wx, ctx):
    lib, MX = wx.load(), wx.TYPE_MXFP4
    assert lib.wamx_type_size(MX) == 17 and lib.wamx_blck_size(MX) == 32 and lib.wamx_blck_size(wx.TYPE_F32) == 1
    t = lib.wamx_new_tensor_3d(ctx, MX, 96, 5, 2)
    assert tuple(t.contents.nb) == (17, 51, 255, 510)
    assert lib.wamx_nbytes(t) == 510 and lib.wamx_is_contiguous(t)
    v = lib.wamx_view_2d(ctx, t, 64, 3, 51, 51 + 17)
    assert v and lib.wamx_nbytes(v) == 2 * 51 + 34 and not lib.wamx_is_contiguous(v)
    assert not lib.wamx_new_tensor_2d(ctx, MX, 40, 2)
    assert "whole blocks" in wx.last_error()
    assert not lib.wamx_reshape_2d(ctx, t, 48, 20)


def test_other_types_keep_their_strides(wx, ctx):
    lib = wx.load()
    for typ, es in ((wx.TYPE_F32, 4), (wx.TYPE_BF16, 2), (wx.TYPE_F16, 2), (wx.TYPE_I32, 4)):
        t = lib.wamx_new_tensor_4d(ctx, typ, 5, 7, 2, 3)
        assert tuple(t.contents.nb) == (es, 5 * es, 35 * es, 70 * es) and lib.wamx_nbytes(t) == 210 * es
        assert lib.wamx_is_contiguous(t)


def test_mxfp4_readers(wx, ctx):
    lib = wx.load()
    ok = lambda t: bool(lib.wamx_backend_supports_op(None, t))  # noqa: E731
    w, x = lib.wamx_new_tensor_2d(ctx, wx.TYPE_MXFP4, 64, 16), lib.wamx_new_tensor_2d(ctx, wx.TYPE_F32, 64, 3)
    assert ok(lib.wamx_mul_mat(ctx, w, x))
    assert ok(lib.wamx_linear(ctx, w, x, None, wx.EPI_NONE, None, None))
    assert ok(lib.wamx_cast(ctx, w, wx.TYPE_BF16)) and ok(lib.wamx_cast(ctx, x, wx.TYPE_MXFP4))
    assert ok(lib.wamx_get_rows(ctx, w, lib.wamx_new_tensor_1d(ctx, wx.TYPE_I32, 4)))
    # a half-float or 4-bit activation, an element-wise op, a repack are not offered
    h = lib.wamx_new_tensor_2d(ctx, wx.TYPE_F16, 64, 3)
    assert not ok(lib.wamx_mul_mat(ctx, w, h)) and not ok(lib.wamx_mul_mat(ctx, x, w))
    assert not ok(lib.wamx_add(ctx, w, w)) and not ok(lib.wamx_cont(ctx, w)) and not ok(lib.wamx_scale(ctx, w, 2.0))
    # columns in another order, rows that are cut inside a block's bytes
    t = lib.wamx_transpose(ctx, lib.wamx_new_tensor_2d(ctx, wx.TYPE_MXFP4, 64, 64))
    assert not t or not ok(lib.wamx_cast(ctx, t, wx.TYPE_F32))
    strided = lib.wamx_view_2d(ctx, lib.wamx_new_tensor_2d(ctx, wx.TYPE_F32, 128, 4), 64, 4, 128 * 4, 0)
    assert ok(lib.wamx_cast(ctx, strided, wx.TYPE_MXFP4))
    assert not ok(lib.wamx_cast(ctx, lib.wamx_transpose(ctx, lib.wamx_new_tensor_2d(ctx, wx.TYPE_F32, 64, 64)), wx.TYPE_MXFP4))


def test_head_norm_constructor(wx, ctx):
    lib, BF, I = wx.load(), wx.TYPE_BF16, wx.TYPE_I32
    n = lambda t, *ne: lib.wamx_new_tensor_4d(ctx, t, *ne, *([1] * (4 - len(ne))))  # noqa: E731
    x, w, k, past, pos = n(BF, 256, 6), n(BF, 128), n(BF, 128, 10, 2, 2), n(I, 2), n(I, 6)
    good = dict(x=x, w=w, dst=k, past=past, pos=pos, mode=2, dims=128, eps=1e-6, base=1e4)
    call = lambda **o: lib.wamx_qk_head_norm_rope(ctx, *{**good, **o}.values())  # noqa: E731
    t = call()
    assert t and lib.wamx_backend_supports_op(None, t)
    assert call(past=None) and call(dims=0, pos=None) and call(mode=0, dims=64)
    for bad in (dict(mode=1), dict(dims=24), dict(dims=144), dict(pos=None), dict(eps=-1.0), dict(base=0.0),
                dict(w=n(BF, 64)), dict(w=n(wx.TYPE_F32, 128)), dict(x=n(BF, 256, 5)), dict(x=n(wx.TYPE_F32, 256, 6)),
                dict(x=n(BF, 256, 22)), dict(past=n(I, 3)), dict(pos=n(I, 5)), dict(past=n(wx.TYPE_F32, 2)),
                dict(dst=n(BF, 96, 10, 2, 2)), dict(dst=n(wx.TYPE_F32, 128, 10, 2, 2))):
        assert not call(**bad), bad
        assert "wamx_qk_head_norm_rope" in wx.last_error()
    vt = n(BF, 16, 128, 2, 2)
    assert lib.wamx_vt_append(ctx, x, vt, past) and lib.wamx_vt_append(ctx, x, vt, None)
    assert not lib.wamx_vt_append(ctx, x, n(BF, 2, 128, 2, 2), past) and not lib.wamx_vt_append(ctx, x, k, past)


def test_tree_attn_constructor(wx, ctx):
    lib, BF, I = wx.load(), wx.TYPE_BF16, wx.TYPE_I32
    n = lambda t, *ne: lib.wamx_new_tensor_4d(ctx, t, *ne, *([1] * (4 - len(ne))))  # noqa: E731
    q, k, v, par, past = n(BF, 64, 5, 4, 2), n(BF, 64, 24, 2, 2), n(BF, 24, 64, 2, 2), n(I, 5, 2), n(I, 2)
    good = dict(q=q, k=k, v=v, par=par, past=past, scale=0.125)
    call = lambda **o: lib.wamx_tree_attn(ctx, *{**good, **o}.values())  # noqa: E731
    t = call()
    assert t and tuple(t.contents.ne) == (256, 5, 2, 1) and lib.wamx_backend_supports_op(None, t)
    assert call(past=None)
    for bad in (dict(q=n(BF, 80, 5, 4, 2)), dict(q=n(BF, 64, 5, 3, 2)), dict(q=n(BF, 64, 25, 4, 2), par=n(I, 25, 2)),
                dict(q=n(BF, 64, 257, 4, 2), par=n(I, 257, 2)), dict(k=n(BF, 64, 23, 2, 2)), dict(v=n(BF, 24, 64, 1, 2)),
                dict(v=n(BF, 23, 64, 2, 2), k=n(BF, 64, 23, 2, 2)), dict(par=n(I, 4, 2)), dict(par=n(wx.TYPE_F32, 5, 2)),
                dict(past=n(I, 1)), dict(q=n(wx.TYPE_F32, 64, 5, 4, 2))):
        assert not call(**bad), bad
        assert "wamx_tree_attn" in wx.last_error()


def test_null_backend_is_refused(wx):
    lib = wx.load()
    a = np.zeros(64, np.float32).ctypes.data
    assert lib.wamx_op_quantize_mxfp4(None, a, 0, 32, a, 1, 32) != 0
    assert lib.wamx_op_mul_mat_mxfp4(None, a, a, 30, 32, a, 0, 1, 1, 1, 32) != 0
    assert lib.wamx_op_tree_attn(None, a, a, a, a, None, a, 1, 1, 64, 1, 1, 8, 8, 1.0) != 0
    assert "null argument" in wx.last_error()


def test_reference_round_trip():
    """The tests' own quantiser: values on the grid come back, others to the nearest level."""
    r = np.random.default_rng(1)
    x = r.integers(-2, 3, (4, 64)).astype(np.float64)
    x[:, ::32] = 6
    np.testing.assert_array_equal(ref.dequantize(ref.quantize(x)), x)
    y = r.standard_normal((4, 64))
    q = ref.dequantize(ref.quantize(y))
    # within half the widest step, 2 of 6, of each block's scale
    assert (np.abs(q - y) <= np.exp2(np.floor(np.log2(np.abs(y).reshape(4, 2, 32).max(2))) - 2).repeat(32, 1) * 2 + 1e-12).all()
