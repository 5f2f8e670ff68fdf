"""4-bit products over rows longer than the workspace holds one of: K has no
limit below 2^30 for any number of tokens and either type of activations."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_mxfp4 import Graph, int_weights, typ

pytestmark = pytest.mark.gpu

LONG = (1 << 24) + 32  # a row of 32 MB in bf16, and one block


def sparse(rng, rows, K, dtype):
    """Rows of zeros with 24 small integers, the first and last value and both sides of 2^24 among them."""
    x = np.zeros((rows, K), dtype)
    at = np.sort(rng.choice(K, (rows, 24)), 1)
    at[:, :4] = [0, K - 1, min(1 << 24, K - 2), min((1 << 24) - 1, K - 3)]
    v = rng.integers(1, 4, at.shape) * rng.choice([-1, 1], at.shape)
    return x, at, v


def expected(w, at, v):
    """Exact: sums of some halves.  w packed [M, K / 32 * 17]."""
    M = w.shape[0]
    b = w.reshape(M, -1, 17)
    out = np.zeros((len(at), M))
    for n in range(len(at)):
        last = {int(k): int(a) for k, a in zip(at[n], v[n])}  # a column picked twice holds its last value
        for k, a in last.items():
            row = np.ascontiguousarray(b[:, k // 32]).reshape(M, 17)
            out[n] += a * ref.dequantize(row)[:, k % 32]
    return out.astype(np.float32)


@pytest.mark.parametrize("N", [32, 33])
@pytest.mark.parametrize("xt", ["f32", "bf16"])
def test_rows_longer_than_the_workspace(wx, be, N, xt):
    print(f"long rows N {N} {xt}", flush=True)
    rng, M = np.random.default_rng(N), 5
    w = int_weights(rng, M, LONG)
    x, at, v = sparse(rng, N, LONG, np.float32 if xt == "f32" else np.uint16)
    for n in range(N):
        x[n, at[n]] = v[n] if xt == "f32" else wx.f32_to_bf16(v[n].astype(np.float32))
    dw, dx, dy = be.array(w), be.array(x), be.array(np.full((N + 1, M), -5, np.float32))
    del x
    wx.check(be.lib.wamx_op_mul_mat_mxfp4(be.ptr, dw.ptr, dx.ptr, typ(wx, xt), LONG, dy.ptr, wx.TYPE_F32, M, M, N, LONG))
    got = dy.download(np.float32, (N + 1, M))
    np.testing.assert_array_equal(got[:N], expected(w, at, v))
    assert (got[N] == -5).all()


def test_long_rows_in_a_graph(wx, be):
    """Activations whose rows lie within one another: 33 windows of one long row."""
    rng, M, N = np.random.default_rng(3), 4, 33
    w = int_weights(rng, M, LONG)
    g = Graph(wx, be)
    leaf, x = g.leaf(wx.TYPE_MXFP4, LONG, M), g.leaf(wx.TYPE_F32, LONG + 8 * N)
    g.place()
    rows = be.lib.wamx_view_2d(g.ctx, x, LONG, N, 32, 0)
    y = be.lib.wamx_mul_mat(g.ctx, leaf, rows)
    assert be.lib.wamx_backend_supports_op(None, y)
    g.build(y)
    xv, at, v = sparse(rng, 1, LONG + 8 * N, np.float32)
    xv[0, at[0]] = v[0]
    g.set(leaf, w), g.set(x, xv)
    g.compute()
    k = np.flatnonzero(xv[0])
    ats, vs = [], []
    for n in range(N):
        here = k[(k >= 8 * n) & (k < 8 * n + LONG)]
        ats.append(here - 8 * n), vs.append(xv[0, here])
    np.testing.assert_array_equal(g.get(y, np.float32, (N, M)), expected(w, ats, vs))
    g.close()
