"""MXFP4 products at sizes that reach every tile, every split of K and every
few-token form, with row strides past 32-bit offsets, activations rounded in
parts, and split products replayed between other users of the workspace.  All
values are halves whose sums stay below 2^24, so every order of summation gives
the same f32 and the results are compared for equality."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_mxfp4 import Graph, int_weights, product

pytestmark = pytest.mark.gpu

# 224 x 256, 128 x 256, 128 x 128 and 64 x 64 tiles, whole and with K in 2, 4, 8.
TILES = [(6963, 1175, 256), (4350, 1172, 5024), (1753, 1183, 4960), (4289, 1162, 256), (1056, 1159, 3904),
         (2745, 1140, 256), (1601, 938, 3040), (837, 845, 3008), (515, 661, 4032), (75, 68, 256), (70, 66, 1280),
         (65, 71, 2112), (69, 66, 4096), (7000, 2049, 64), (6500, 50, 96)]
TILES += [(1829, 1106, 5024), (974, 1039, 3360), (2707, 130, 4800), (590, 769, 2848), (65, 72, 1760)]
# One to four tiles of tokens by one, two and four groups of rows, and four K splits.
FEW = [(40, 9, 96), (40, 30, 96), (40, 47, 96), (40, 64, 96), (6405, 9, 64), (6405, 30, 64), (6390, 41, 64), (6390, 64, 64),
       (12805, 16, 64), (12805, 17, 64), (12805, 33, 64), (1000, 35, 12288), (1030, 64, 12320), (2060, 40, 12288),
       (4090, 48, 12416)]


def case(wx, be, M, N, K, xt, yt="f32"):
    rng = np.random.default_rng(M * 5 + N * 3 + K)
    w = int_weights(rng, M, K)
    xi = rng.integers(-3, 4, (N, K)).astype(np.float32)
    want = xi @ ref.dequantize(w).astype(np.float32).T
    got = product(wx, be, w, wx.f32_to_bf16(xi) if xt == "bf16" else xi, xt, yt)
    np.testing.assert_array_equal(got, want if yt == "f32" else wx.f32_to_bf16(want))


@pytest.mark.parametrize("M,N,K", TILES + FEW)
@pytest.mark.parametrize("xt,yt", [("bf16", "f32"), ("f32", "bf16")])
def test_every_plan_is_exact(wx, be, M, N, K, xt, yt):
    print(f"product {M}x{N}x{K} {xt} {yt}", flush=True)
    case(wx, be, M, N, K, xt, yt)


def test_f32_activations_rounded_in_parts(wx, be):
    """More tokens than the workspace holds rounded: two parts, of one result."""
    case(wx, be, 32, 5003, 4096, "f32")


@pytest.mark.parametrize("N", [3, 70])
def test_rows_further_apart_than_32_bit_offsets(wx, be, N):
    M, K, ldx = 40, 64, 1 << 22
    rng = np.random.default_rng(N)
    w = int_weights(rng, M, K)
    xi = rng.integers(-3, 4, (N, K)).astype(np.float32)
    xb = np.zeros((N, ldx), np.uint16)
    xb[:, :K] = wx.f32_to_bf16(xi)
    dw, dx, dy = be.array(w), be.array(xb), be.empty(N * M * 4)
    wx.check(be.lib.wamx_op_mul_mat_mxfp4(be.ptr, dw.ptr, dx.ptr, wx.TYPE_BF16, ldx, dy.ptr, wx.TYPE_F32, M, M, N, K))
    np.testing.assert_array_equal(dy.download(np.float32, (N, M)), xi @ ref.dequantize(w).astype(np.float32).T)


@pytest.mark.parametrize("xt", ["bf16", "f32"])
def test_rows_so_far_apart_that_they_go_one_by_one(wx, be, xt):
    M, N, K, ldx = 40, 5, 96, (1 << 23) + 5
    rng = np.random.default_rng(7)
    w = int_weights(rng, M, K)
    xi = rng.integers(-3, 4, (N, K)).astype(np.float32)
    xb = np.zeros((N, ldx), np.uint16 if xt == "bf16" else np.float32)
    xb[:, :K] = wx.f32_to_bf16(xi) if xt == "bf16" else xi
    dw, dx, dy = be.array(w), be.array(xb), be.empty(N * M * 4)
    wx.check(be.lib.wamx_op_mul_mat_mxfp4(be.ptr, dw.ptr, dx.ptr, wx.TYPE_BF16 if xt == "bf16" else wx.TYPE_F32, ldx,
                                          dy.ptr, wx.TYPE_F32, M, M, N, K))
    np.testing.assert_array_equal(dy.download(np.float32, (N, M)), xi @ ref.dequantize(w).astype(np.float32).T)


def test_split_products_replayed_between_other_calls(wx, be):
    """Two computed graphs with split products, replayed in turn with single calls
    that use a workspace too between them."""
    sizes = [(256, 40, 12288), (96, 130, 8192)]
    graphs = []
    for M, N, K in sizes:
        g = Graph(wx, be)
        w, x = g.leaf(wx.TYPE_MXFP4, K, M), g.leaf(wx.TYPE_F32, K, N)
        g.place()
        y = be.lib.wamx_mul_mat(g.ctx, w, x)
        g.build(y)
        graphs.append((g, w, x, y))
    for step in range(4):
        rng = np.random.default_rng(step)
        wants = []
        for (M, N, K), (g, w, x, y) in zip(sizes, graphs):
            wv, xv = int_weights(rng, M, K), rng.integers(-3, 4, (N, K)).astype(np.float32)
            g.set(w, wv), g.set(x, xv)
            wants.append(xv @ ref.dequantize(wv).astype(np.float32).T)
        for again in range(2):
            for (M, N, K), (g, w, x, y), want in zip(sizes, graphs, wants):
                g.compute()
                case(wx, be, 70, 66, 1280, "f32")
                np.testing.assert_array_equal(g.get(y, np.float32, (N, M)), want)
    for g, *_ in graphs:
        g.close()
