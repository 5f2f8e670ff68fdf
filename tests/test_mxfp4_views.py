"""Views of MXFP4 tensors (no GPU needed): a block cannot be turned out of its
row, so a transposed weight is refused where it is made, where it is imported
and where it is read; rows inside one another are refused; what keeps rows
whole still passes."""
from __future__ import annotations

import ctypes as C

import pytest


@pytest.fixture
def ctx(wx):
    c = wx.load().wamx_init(512)
    yield c
    wx.load().wamx_free(c)


def readers(wx, ctx, w):
    """Every op that reads 4-bit rows, on w: name -> whether it is offered."""
    lib, K = wx.load(), w.contents.ne[0]
    x = lib.wamx_new_tensor_2d(ctx, wx.TYPE_F32, K, 2)
    ids = lib.wamx_new_tensor_1d(ctx, wx.TYPE_I32, 3)
    made = dict(cast=lib.wamx_cast(ctx, w, wx.TYPE_F32), rows=lib.wamx_get_rows(ctx, w, ids),
                product=lib.wamx_mul_mat(ctx, w, x), linear=lib.wamx_linear(ctx, w, x, None, wx.EPI_NONE, None, None))
    return {k: bool(t) and bool(lib.wamx_backend_supports_op(None, t)) for k, t in made.items()}


@pytest.mark.parametrize("ne", [(32, 64), (32, 32), (64, 64), (64, 32), (32, 96)])
def test_transposes_are_refused(wx, ctx, ne):
    lib = wx.load()
    t = lib.wamx_new_tensor_2d(ctx, wx.TYPE_MXFP4, *ne)
    assert not lib.wamx_transpose(ctx, t) and "mxfp4" in wx.last_error()
    assert not lib.wamx_permute(ctx, t, 1, 2, 0, 3) and "mxfp4" in wx.last_error()


def test_permutes_of_whole_rows_pass(wx, ctx):
    lib = wx.load()
    t = lib.wamx_new_tensor_3d(ctx, wx.TYPE_MXFP4, 64, 5, 3)
    p = lib.wamx_permute(ctx, t, 0, 2, 1, 3)
    assert p and tuple(p.contents.ne) == (64, 3, 5, 1) and tuple(p.contents.nb)[:3] == (17, 170, 34)
    assert lib.wamx_backend_supports_op(None, lib.wamx_cast(ctx, p, wx.TYPE_F32))
    assert lib.wamx_backend_supports_op(None, lib.wamx_mul_mat(ctx, p, lib.wamx_new_tensor_3d(ctx, wx.TYPE_F32, 64, 2, 5)))
    # other types turn as they did
    assert lib.wamx_transpose(ctx, lib.wamx_new_tensor_2d(ctx, wx.TYPE_BF16, 32, 64))


@pytest.mark.parametrize("nb1,ok", [(34, True), (40, True), (51, True), (33, False), (17, False), (0, False)])
def test_rows_within_one_another_are_refused(wx, ctx, nb1, ok):
    lib = wx.load()
    t = lib.wamx_new_tensor_2d(ctx, wx.TYPE_MXFP4, 64, 16)
    v = lib.wamx_view_2d(ctx, t, 64, 4, nb1, 0)
    assert readers(wx, ctx, v) == dict.fromkeys(("cast", "rows", "product", "linear"), ok)
    # one row has no other to meet (MUL_MAT wants nb[0] <= nb[1] of any weight)
    assert readers(wx, ctx, lib.wamx_view_2d(ctx, t, 64, 1, nb1, 0)) == dict(cast=True, rows=True, linear=True,
                                                                             product=nb1 >= 17)


def test_planes_within_rows_are_refused(wx, ctx):
    lib = wx.load()
    t = lib.wamx_new_tensor_3d(ctx, wx.TYPE_MXFP4, 64, 16, 2)
    for nb2, ok in ((34 * 16, True), (34, True), (17, False)):
        v = lib.wamx_view_3d(ctx, t, 64, 2, 2, 34, nb2, 0)
        assert bool(lib.wamx_backend_supports_op(None, lib.wamx_cast(ctx, v, wx.TYPE_F32))) is ok


class Desc(C.Structure):
    _fields_ = [("op", C.c_char_p), ("unary_op", C.c_char_p), ("type", C.c_char_p), ("ne", C.c_int64 * 4),
                ("nb", C.c_size_t * 4), ("op_params", C.c_int32 * 16), ("flags", C.c_int32), ("src", C.c_int32 * 10),
                ("view_src", C.c_int32), ("view_offs", C.c_size_t), ("data", C.c_void_p), ("name", C.c_char_p)]


def desc(op, t, ne, nb, src=(), view=-1, params=()):
    s = list(src) + [-1] * (10 - len(src))
    p = list(params) + [0] * (16 - len(params))
    return Desc(op, None, t, (C.c_int64 * 4)(*ne), (C.c_size_t * 4)(*nb), (C.c_int32 * 16)(*p), 0, (C.c_int32 * 10)(*s),
                view, 0, None, op)


@pytest.mark.parametrize("op,params", [(b"TRANSPOSE", ()), (b"PERMUTE", (1, 0, 2, 3))])
@pytest.mark.parametrize("between", [(), (b"VIEW",), (b"RESHAPE", b"VIEW")])
def test_imported_transposes_are_refused(wx, ctx, op, params, between):
    """32 x 32 values: the turned view's strides are those of whole rows."""
    lib = wx.load()
    sq, nb = (32, 32, 1, 1), (17, 17, 544, 544)
    d = [desc(b"NONE", b"mxfp4", sq, nb), desc(op, b"mxfp4", sq, nb, (0,), 0, params)]
    for b in between:
        d.append(desc(b, b"mxfp4", sq, nb, (len(d) - 1,), 0))
    w = len(d) - 1
    d.append(desc(b"NONE", b"f32", (32, 2, 1, 1), (4, 128, 256, 256)))
    x = len(d) - 1
    d += [desc(b"MUL_MAT", b"f32", (32, 2, 1, 1), (4, 128, 256, 256), (w, x)),
          desc(b"CPY", b"f32", sq, (4, 128, 4096, 4096), (w,))]
    made = [(1, False), (len(d) - 2, False), (len(d) - 1, False)]
    # the same readers on the tensor itself
    d += [desc(b"MUL_MAT", b"f32", (32, 2, 1, 1), (4, 128, 256, 256), (0, x)),
          desc(b"CPY", b"f32", sq, (4, 128, 4096, 4096), (0,))]
    made += [(len(d) - 2, True), (len(d) - 1, True)]
    for i, ok in made:
        g = lib.wamx_graph_from_ggml(ctx, (Desc * len(d))(*d), len(d), (C.c_int32 * 1)(i), 1)
        assert g, wx.last_error()
        node = lib.wamx_graph_node(g, lib.wamx_graph_n_nodes(g) - 1)
        assert bool(lib.wamx_backend_supports_op(None, node)) is ok, (i, d[i].op)


def test_imported_copy_into_a_transpose_is_refused(wx, ctx):
    lib = wx.load()
    sq, nb = (32, 32, 1, 1), (17, 17, 544, 544)
    for turned in (False, True):
        d = [desc(b"NONE", b"mxfp4", sq, nb), desc(b"TRANSPOSE" if turned else b"VIEW", b"mxfp4", sq, nb, (0,), 0),
             desc(b"NONE", b"f32", sq, (4, 128, 4096, 4096)), desc(b"CPY", b"mxfp4", sq, nb, (2, 1), 0)]
        g = lib.wamx_graph_from_ggml(ctx, (Desc * 4)(*d), 4, (C.c_int32 * 1)(3), 1)
        node = lib.wamx_graph_node(g, lib.wamx_graph_n_nodes(g) - 1)
        assert bool(lib.wamx_backend_supports_op(None, node)) is not turned
