"""The MXFP4 type inside graphs: element-wise nodes and row ops behind a 4-bit
product (which the framework folds into other products), weights and
activations in planes, copies of views whose planes do not follow each other.
Integers throughout, so results are exact; a row op's output is that of the
same op on the product's exact bits."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_fusion import Graph
from test_gpu_mxfp4 import int_weights

pytestmark = pytest.mark.gpu


def weights(rng, M, K):
    """Packed weights of -1, 0, 1 (scale 1): every sum below 2^8 is exact in bf16."""
    v = rng.integers(-1, 2, (M, K)).astype(np.float64)
    p = np.empty((M, K // 32, 17), np.uint8)
    code = np.where(v > 0, 2, np.where(v < 0, 10, 0)).astype(np.uint8).reshape(M, K // 32, 32)
    p[..., 0], p[..., 1:] = 127, code[..., :16] | code[..., 16:] << 4
    p = p.reshape(M, -1)
    assert (ref.dequantize(p) == v).all()
    return p, v.astype(np.float32)


def form(wx, typ, a):
    return np.asarray(a, np.float32) if typ == wx.TYPE_F32 else wx.f32_to_bf16(np.asarray(a, np.float32))


def fused(be, g, *outs):
    before = be.lib.wamx_backend_fused_nodes(be.ptr)
    g.compute(*outs)
    return be.lib.wamx_backend_fused_nodes(be.ptr) - before


@pytest.mark.parametrize("N", [1, 20, 48, 70])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("nodes", ["bias gelu", "add mul", "mul bias", "gelu"])
def test_elementwise_nodes_behind_a_product(wx, be, N, out, nodes):
    print(f"behind a product: {nodes} N {N} {out}", flush=True)
    lib, rng, M, K = be.lib, np.random.default_rng(N), 132, 96
    T, dt = (wx.TYPE_F32, np.float32) if out == "f32" else (wx.TYPE_BF16, np.uint16)
    g, alone = Graph(wx, be), Graph(wx, be)
    try:
        w, x, row, full = g.t(wx.TYPE_MXFP4, K, M), g.t(wx.TYPE_BF16, K, N), g.t(T, M), g.t(T, M, N)
        wv, wd = weights(rng, M, K)
        xv = rng.integers(-1, 2, (N, K)).astype(np.float32)
        rv, fv = rng.integers(-4, 5, M).astype(np.float32), rng.integers(-1, 2, (N, M)).astype(np.float32)
        y = lib.wamx_mul_mat_out_type(g.ctx, w, x, T)
        cur, want, outs, wants = y, xv @ wd.T, [y], [xv @ wd.T]
        for kind in nodes.split():
            if kind == "gelu":
                cur = lib.wamx_gelu(g.ctx, cur)
                before_gelu, want = want, None
            else:
                cur = (lib.wamx_mul if kind == "mul" else lib.wamx_add)(g.ctx, cur, row if kind == "bias" else full)
                want = want * fv if kind == "mul" else want + (rv if kind == "bias" else fv)
            outs.append(cur), wants.append(want)
        leaf = alone.t(T, M, N)
        gelu = lib.wamx_gelu(alone.ctx, leaf)
        g.alloc(), alone.alloc()
        g.set(w, wv), g.set(x, wx.f32_to_bf16(xv)), g.set(row, form(wx, T, rv)), g.set(full, form(wx, T, fv))
        assert fused(be, g, cur) == 0
        for t, a in zip(outs, wants):
            if a is None:
                alone.set(leaf, form(wx, T, before_gelu))
                alone.compute(gelu)
                np.testing.assert_array_equal(g.get(t, dt, (N, M)), alone.get(gelu, dt, (N, M)))
            else:
                assert np.abs(a).max() < 256
                np.testing.assert_array_equal(g.get(t, dt, (N, M)), form(wx, T, a))
    finally:
        g.close(), alone.close()


@pytest.mark.parametrize("N", [1, 33, 64, 130])
@pytest.mark.parametrize("op", ["norm", "modulation", "qk"])
def test_row_ops_behind_a_linear(wx, be, rng, N, op):
    """The rows of a 4-bit LINEAR, then the op on a leaf that holds the same bits."""
    print(f"behind a linear: {op} N {N}", flush=True)
    lib, H, DH, K = be.lib, 4, 64, 160
    M = H * DH
    g, alone = Graph(wx, be), Graph(wx, be)
    wv, wd = weights(rng, M, K)
    xv = rng.integers(-1, 2, (N, K)).astype(np.float32)
    bias = rng.integers(-3, 4, M).astype(np.float32)
    yv = xv @ wd.T + bias
    assert np.abs(yv).max() < 256
    sc, sh = 1 + 0.1 * rng.standard_normal(M), 0.1 * rng.standard_normal(M)

    def behind(gr, lin, sets):
        if op == "qk":
            nw, pos, dst = gr.t(wx.TYPE_BF16, M), gr.t(wx.TYPE_I32, N), gr.t(wx.TYPE_BF16, DH, N, H)
            sets += [(nw, wx.f32_to_bf16(sc.astype(np.float32))), (pos, np.arange(3, 3 + N, dtype=np.int32))]
            return lib.wamx_qk_norm_rope(gr.ctx, lin, nw, dst, 0, 0, pos, None, None, 1e-6, 1e4)
        T = wx.TYPE_F32 if op == "modulation" else wx.TYPE_BF16
        a, b = gr.t(T, M), gr.t(T, M)
        sets += [(a, form(wx, T, sc)), (b, form(wx, T, sh))]
        make = lib.wamx_norm_modulation_bf16 if op == "modulation" else lib.wamx_layer_norm_bf16
        return make(gr.ctx, lin, a, b, 1e-6)

    try:
        w, x, b = g.t(wx.TYPE_MXFP4, K, M), g.t(wx.TYPE_BF16, K, N), g.t(wx.TYPE_BF16, M)
        lin = lib.wamx_linear(g.ctx, w, x, b, wx.EPI_BIAS, None, None)
        sets = [(w, wv), (x, wx.f32_to_bf16(xv)), (b, wx.f32_to_bf16(bias))]
        t = behind(g, lin, sets)
        assert lin and t, wx.last_error()
        leaf, sets1 = alone.t(wx.TYPE_BF16, M, N), []
        t1 = behind(alone, leaf, sets1)
        sets1.append((leaf, wx.f32_to_bf16(yv.astype(np.float32))))
        for gr, ss in ((g, sets), (alone, sets1)):
            gr.alloc()
            for leaf_, a in ss:
                gr.set(leaf_, a)
        assert fused(be, g, t) == 0
        alone.compute(t1)
        np.testing.assert_array_equal(g.get(lin, np.uint16, (N, M)), wx.f32_to_bf16(yv.astype(np.float32)))
        np.testing.assert_array_equal(g.get(t, np.uint16, (N * M,)), alone.get(t1, np.uint16, (N * M,)))
    finally:
        g.close(), alone.close()


@pytest.mark.parametrize("N", [1, 5, 40, 100])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("wp,xp", [((1, 1), (2, 3)), ((2, 1), (4, 3)), ((2, 3), (2, 3)), ((1, 3), (3, 6))])
@pytest.mark.parametrize("layout", ["packed", "strided", "permuted"])
def test_products_in_planes(wx, be, N, xt, wp, xp, layout):
    """Weight planes broadcast over x's (x plane i reads weight plane i / ratio);
    x with gaps behind its rows and planes; both as permuted views."""
    print(f"planes w {wp} x {xp} {layout} N {N} {xt}", flush=True)
    lib, rng, M, K = be.lib, np.random.default_rng(N), 20, 64
    X, es = (wx.TYPE_F32, 4) if xt == "f32" else (wx.TYPE_BF16, 2)
    RB = K // 32 * 17
    packed = int_weights(rng, wp[0] * wp[1] * M, K).reshape(wp[1], wp[0], M, RB)
    xv = rng.integers(-3, 4, (xp[1], xp[0], N, K)).astype(np.float32)
    g = Graph(wx, be)
    try:
        if layout == "permuted":  # memory [.][row][plane][values]
            wl, xl = g.t(wx.TYPE_MXFP4, K, wp[0], M, wp[1]), g.t(X, K, xp[0], N, xp[1])
            w, x = lib.wamx_permute(g.ctx, wl, 0, 2, 1, 3), lib.wamx_permute(g.ctx, xl, 0, 2, 1, 3)
            wm, xm = packed.transpose(0, 2, 1, 3), xv.transpose(0, 2, 1, 3)
        elif layout == "strided":  # a block behind every row, a row behind every plane
            wl, xl = g.t(wx.TYPE_MXFP4, K + 32, M + 1, wp[0], wp[1]), g.t(X, K + 3, N + 1, xp[0], xp[1])
            w = lib.wamx_view_4d(g.ctx, wl, K, M, *wp, *list(wl.contents.nb)[1:], 0)
            x = lib.wamx_view_4d(g.ctx, xl, K, N, *xp, *list(xl.contents.nb)[1:], 0)
            wm = np.full((wp[1], wp[0], M + 1, RB + 17), 0xFF, np.uint8)
            wm[:, :, :M, :RB] = packed
            xm = np.full((xp[1], xp[0], N + 1, K + 3), np.nan, np.float32)
            xm[:, :, :N, :K] = xv
        else:
            wl = w = g.t(wx.TYPE_MXFP4, K, M, *wp)
            xl = x = g.t(X, K, N, *xp)
            wm, xm = packed, xv
        y = lib.wamx_mul_mat(g.ctx, w, x)
        assert y and lib.wamx_backend_supports_op(None, y), wx.last_error()
        g.alloc()
        g.set(wl, wm), g.set(xl, form(wx, X, xm))
        g.compute(y)
        wd = ref.dequantize(packed.reshape(-1, RB)).reshape(wp[1], wp[0], M, K).astype(np.float32)
        wd = wd.repeat(xp[1] // wp[1], 0).repeat(xp[0] // wp[0], 1)
        np.testing.assert_array_equal(g.get(y, np.float32, (xp[1], xp[0], N, M)), xv @ wd.transpose(0, 1, 3, 2))
    finally:
        g.close()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(64, 5, 3, 2), (32, 1, 4, 2), (96, 7, 1, 3)])
def test_copies_of_views(wx, be, typ, shape):
    """To the type from rows with gaps behind rows and planes, and from it to such
    rows; from a permuted 4-bit tensor and a slice of its rows."""
    print(f"copies {typ} {shape}", flush=True)
    lib, rng = be.lib, np.random.default_rng(sum(shape))
    T, dt = {"f32": (wx.TYPE_F32, np.float32), "f16": (wx.TYPE_F16, np.float16), "bf16": (wx.TYPE_BF16, np.uint16)}[typ]
    cast = lambda a: wx.f32_to_bf16(a) if typ == "bf16" else a.astype(dt)  # noqa: E731
    C, R, P, Q = shape
    v = rng.integers(-4, 5, (Q, P, R, C)).astype(np.float32)
    v[..., ::32] = 6  # every value is a code of the block
    v[np.abs(v) == 5] = 4
    g = Graph(wx, be)
    try:
        big, dst = g.t(T, C + 5, R + 1, P, Q), g.t(T, C + 5, R + 1, P, Q)
        src = lib.wamx_view_4d(g.ctx, big, C, R, P, Q, *list(big.contents.nb)[1:], 0)
        out = lib.wamx_view_4d(g.ctx, dst, C, R, P, Q, *list(dst.contents.nb)[1:], 0)
        q = lib.wamx_cast(g.ctx, src, wx.TYPE_MXFP4)
        back = lib.wamx_cpy(g.ctx, q, out)
        turned = lib.wamx_cast(g.ctx, lib.wamx_permute(g.ctx, q, 0, 3, 1, 2), T)
        nb = list(q.contents.nb)
        lo = R // 2
        part = lib.wamx_cast(g.ctx, lib.wamx_view_4d(g.ctx, q, 32, R - lo, P, Q, *nb[1:], lo * nb[1] + (C // 32 - 1) * 17), T)
        for t in (q, back, turned, part):
            assert t and lib.wamx_backend_supports_op(None, t), wx.last_error()
        g.alloc()
        full = np.full((Q, P, R + 1, C + 5), np.nan, np.float32)
        full[:, :, :R, :C] = v
        fill = np.full((Q, P, R + 1, C + 5), 7, np.float32)
        g.set(big, cast(full)), g.set(dst, cast(fill))
        g.compute(back, turned, part)
        fill[:, :, :R, :C] = v
        np.testing.assert_array_equal(g.get(dst, dt, fill.shape), cast(fill))
        np.testing.assert_array_equal(g.get(q, np.uint8, (Q * P * R, C // 32 * 17)), ref.quantize(v.reshape(-1, C)))
        # dims (C, R, P, Q) -> (C, P, Q, R)
        np.testing.assert_array_equal(g.get(turned, dt, (R, Q, P, C)), cast(v.transpose(2, 0, 1, 3)))
        np.testing.assert_array_equal(g.get(part, dt, (Q, P, R - lo, 32)), cast(v[:, :, lo:, C - 32:]))
    finally:
        g.close()
