"""MXFP4 on the device: quantisation and dequantisation bit for bit, products
with 4-bit weights against exact integers and against 64 bits, the LINEAR
epilogues, and the type in computed graphs (CPY, MUL_MAT, LINEAR, GET_ROWS)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import draft_ref as ref

pytestmark = pytest.mark.gpu

NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def typ(wx, name):
    return {"f32": wx.TYPE_F32, "f16": wx.TYPE_F16, "bf16": wx.TYPE_BF16}[name]


def held(wx, a, name):
    """(device form, the f64 values it holds) of floats a."""
    if name == "bf16":
        h = wx.f32_to_bf16(np.asarray(a, np.float32))
        return h, wx.bf16_to_f32(h).astype(np.float64)
    h = np.asarray(a).astype(NP[name])
    return h, h.astype(np.float64)


def quantize(wx, be, x, name, ld=None):
    rows, cols = x.shape
    ld = ld or cols
    buf = np.zeros((rows, ld), x.dtype)
    buf[:, :cols] = x
    buf[:, cols:] = x.reshape(-1)[0]
    dx, dq = be.array(buf), be.array(np.full(rows * cols // 32 * 17 + 32, 0xAB, np.uint8))
    wx.check(be.lib.wamx_op_quantize_mxfp4(be.ptr, dx.ptr, typ(wx, name), ld, dq.ptr, rows, cols))
    got = dq.download(np.uint8, (rows * cols // 32 * 17 + 32,))
    assert (got[-32:] == 0xAB).all(), "bytes behind the last block"
    return got[:-32].reshape(rows, -1)


@pytest.mark.parametrize("rows,cols,ld", [(1, 32, 32), (3, 64, 64), (5, 96, 100), (77, 1024, 1024), (257, 32, 33),
                                          (33, 4096 + 32, 4200)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_quantize_bits(wx, be, rng, rows, cols, ld, name):
    print(f"quantize {rows}x{cols} ld {ld} {name}", flush=True)
    a = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 6, (rows, 1)))
    # ties, exact levels, zeros and signed zeros among them
    a[0, :8] = [0.25, -0.75, 1.25, 2.5, 3.5, 5.0, -0.0, 6.0]
    a[-1, -32:] = 0.0
    x, v = held(wx, a, name)
    got, want = quantize(wx, be, x, name, ld), ref.quantize(v)
    np.testing.assert_array_equal(got, want)


def test_quantize_ends_of_the_range(wx, be):
    """Subnormal, huge, infinite and NaN values, in f32."""
    a = np.zeros((8, 32), np.float32)
    a[0, :4] = [1e-45, -1e-45, 2e-39, 1e-38]
    a[1, :3] = [np.finfo(np.float32).max, -1e38, 3e37]
    a[2, 5] = np.inf
    a[3, 7] = np.nan
    a[4, :3] = [2.0 ** -126, 2.0 ** -127, 2.0 ** -128]
    a[5, :2] = [2.0 ** -124, 2.0 ** -127]
    a[6, :] = -np.inf
    got = quantize(wx, be, a, "f32")
    np.testing.assert_array_equal(got, ref.quantize(a))
    dq, dy = be.array(got), be.empty(a.nbytes)
    wx.check(be.lib.wamx_op_dequantize_mxfp4(be.ptr, dq.ptr, dy.ptr, wx.TYPE_F32, 32, 8, 32))
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(dy.download(np.float32, (8, 32)), ref.dequantize(got).astype(np.float32))


@pytest.mark.parametrize("rows,cols,ld", [(1, 32, 32), (9, 160, 171), (130, 2048, 2048)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_dequantize_bits(wx, be, rng, rows, cols, ld, name):
    """Every code and scales over f32's range; rows behind and beside stay."""
    p = rng.integers(0, 256, (rows, cols // 32, 17)).astype(np.uint8)
    p[..., 0] = rng.integers(100, 140, p.shape[:2])
    p[0, 0, 0] = 255
    if name == "f32":
        p[-1, -1, 0] = 0
    p = p.reshape(rows, -1)
    if name == "bf16":
        fill, want = np.uint16(0x1234), wx.f32_to_bf16(ref.dequantize(p).astype(np.float32))
    else:
        fill, want = NP[name](7.0), ref.dequantize(p).astype(NP[name])
    dq, dy = be.array(p), be.array(np.full((rows + 1, ld), fill))
    wx.check(be.lib.wamx_op_dequantize_mxfp4(be.ptr, dq.ptr, dy.ptr, typ(wx, name), ld, rows, cols))
    got = dy.download(NP[name], (rows + 1, ld))
    if name == "bf16":
        nan = np.isnan(wx.bf16_to_f32(want))
        assert np.isnan(wx.bf16_to_f32(got[:rows, :cols])[nan]).all()
        np.testing.assert_array_equal(got[:rows, :cols][~nan], want[~nan])
    else:
        np.testing.assert_array_equal(got[:rows, :cols], want)
    assert (got[:rows, cols:] == fill).all() and (got[rows] == fill).all()


def int_weights(rng, M, K):
    """Packed weights whose values are multiples of 1/2 up to 24."""
    p = rng.integers(0, 256, (M, K // 32, 17)).astype(np.uint8)
    p[..., 0] = 127 + rng.integers(0, 3, p.shape[:2])
    return p.reshape(M, -1)


def product(wx, be, w, x, xt, yt, ldx=None, ldy=None):
    M, N, K = w.shape[0], x.shape[0], x.shape[1]
    ldx, ldy = ldx or K, ldy or M
    xb = np.zeros((N, ldx), x.dtype)
    xb[:, :K] = x
    if ldx > K:
        xb[:, K:] = x.dtype.type(0x7FC0) if xt == "bf16" else np.nan
    dw, dx = be.array(w), be.array(xb)
    dy = be.array(np.full((N + 1, ldy), -5, np.float32) if yt == "f32" else np.full((N + 1, ldy), 0x1234, np.uint16))
    wx.check(be.lib.wamx_op_mul_mat_mxfp4(be.ptr, dw.ptr, dx.ptr, typ(wx, xt), ldx, dy.ptr, typ(wx, yt), ldy, M, N, K))
    got = dy.download(np.float32 if yt == "f32" else np.uint16, (N + 1, ldy))
    fill = -5 if yt == "f32" else 0x1234
    assert (got[N] == fill).all() and (got[:N, M:] == fill).all(), "written outside the result"
    return got[:N, :M]


# One to many tokens around the tiles' edges, output widths with remainders, K
# of one block up to long rows that end inside a step; one size per kernel
# variant at least.
SIZES = [(1, 1, 32), (16, 1, 64), (17, 2, 96), (33, 15, 160), (100, 16, 4096), (64, 17, 1024), (250, 31, 352),
         (130, 33, 2080), (256, 48, 1024), (77, 64, 128), (300, 65, 96), (128, 100, 544), (515, 129, 1056),
         (1000, 200, 2048), (256, 256, 512), (700, 333, 416), (2050, 300, 64), (384, 1025, 288), (4100, 40, 320),
         (20000, 3, 96), (264, 520, 4128)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("xt", ["bf16", "f32"])
def test_product_integers_exact(wx, be, M, N, K, xt):
    """Sums of halves below 2^24 are exact in f32 in any order."""
    print(f"product {M}x{N}x{K} {xt}", flush=True)
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    w = int_weights(rng, M, K)
    xi = rng.integers(-3, 4, (N, K)).astype(np.float32)
    x = wx.f32_to_bf16(xi) if xt == "bf16" else xi
    want = xi @ ref.dequantize(w).astype(np.float32).T
    odd = 1 if N % 2 else 0
    np.testing.assert_array_equal(product(wx, be, w, x, xt, "f32", K + 3 * odd, M + 5 * odd), want)


@pytest.mark.parametrize("M,N,K", [(100, 1, 4096), (333, 48, 2048), (514, 300, 1056), (256, 520, 4096)])
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")])
def test_product_random(wx, be, rng, M, N, K, xt, yt):
    """|error| <= (K + 8) 2^-24 sum |w x| for the f32 sums (each step of a sum
    is off by half a unit of at most that much), plus half a bf16 step."""
    w = ref.quantize(rng.standard_normal((M, K)) * 0.02)
    x, v = held(wx, rng.standard_normal((N, K)), xt)
    v = wx.bf16_to_f32(wx.f32_to_bf16(v.astype(np.float32))).astype(np.float64)
    wd = ref.dequantize(w)
    want, mass = v @ wd.T, np.abs(v) @ np.abs(wd).T
    got = product(wx, be, w, x, xt, yt)
    got = got.astype(np.float64) if yt == "f32" else wx.bf16_to_f32(got).astype(np.float64)
    tol = (K + 8) * 2.0 ** -24 * mass + (2.0 ** -8 * np.abs(want) if yt == "bf16" else 0)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)


def test_product_scales_and_specials(wx, be):
    """Scale bytes 0 and 255, and Inf / NaN activations: they reach exactly the
    outputs whose sums hold them (K ends inside a step, so nothing of the padding does)."""
    for N in (1, 70):
        M, K = 40, 96
        rng = np.random.default_rng(5)
        w = int_weights(rng, M, K).reshape(M, 3, 17)
        w[:, :, 1:] |= 0x11  # no zero codes
        w[:, :, 1:] &= 0x77
        w[3, 1, 0] = 255
        w[4, :, 0] = 0
        w = w.reshape(M, -1)
        x = rng.integers(1, 4, (N, K)).astype(np.float32)
        if N > 1:
            x[1, 40] = np.inf
            x[2, 95] = np.nan
        got = product(wx, be, w, wx.f32_to_bf16(x), "bf16", "f32")
        wd = ref.dequantize(w)
        with np.errstate(invalid="ignore"):
            want = x.astype(np.float64) @ wd.T
        assert np.isnan(got[:, 3]).all()
        keep = [m for m in range(M) if m not in (3, 4)]
        np.testing.assert_array_equal(got[:, keep], want[:, keep].astype(np.float32))
        fine = [n for n in range(N) if n not in (1, 2)] if N > 1 else [0]
        # subnormal products: an absolute bound of one f32 step each
        assert (np.abs(got[fine, 4] - want[fine, 4]) <= K * 2.0 ** -149).all()


@pytest.mark.parametrize("N", [1, 20, 48, 130, 300])
@pytest.mark.parametrize("epi", ["none", "bias", "gelu", "gated", "residual"])
def test_linear_epilogues(wx, be, orc, rng, N, epi):
    """The same rounding points as LINEAR on bf16 weights: integer products are
    exact, so the bits equal those of the same weight held in bf16."""
    M, K = 160, 352
    w = int_weights(rng, M, K)
    wb = wx.f32_to_bf16(ref.dequantize(w).astype(np.float32))
    assert (wx.bf16_to_f32(wb) == ref.dequantize(w)).all()
    x = wx.f32_to_bf16(rng.integers(-2, 3, (N, K)).astype(np.float32))
    bias = wx.f32_to_bf16(rng.standard_normal(M).astype(np.float32))
    res = wx.f32_to_bf16(rng.standard_normal((N, M)).astype(np.float32))
    gate = rng.standard_normal(M).astype(np.float32)
    code = dict(none=wx.EPI_NONE, bias=wx.EPI_BIAS, gelu=wx.EPI_BIAS_GELU, gated=wx.EPI_BIAS_GATED,
                residual=wx.EPI_BIAS_RESIDUAL)[epi]
    d = [be.array(a) for a in (w, wb, x, bias, res, gate)]
    a, b = be.empty(N * M * 2), be.empty(N * M * 2)
    tail = (d[2].ptr, wx.TYPE_BF16, d[3].ptr, code, d[4].ptr, d[5].ptr)
    wx.check(be.lib.wamx_op_linear_mxfp4(be.ptr, d[0].ptr, *tail, a.ptr, M, N, K))
    wx.check(be.lib.wamx_op_linear(be.ptr, d[1].ptr, *tail, b.ptr, M, N, K))
    np.testing.assert_array_equal(a.download(np.uint16, (N, M)), b.download(np.uint16, (N, M)))


def test_refusals(wx, be):
    lib, d = be.lib, be.empty(1 << 16)
    p = d.ptr
    assert lib.wamx_op_quantize_mxfp4(be.ptr, p, wx.TYPE_F32, 40, p, 1, 40) != 0 and "32-value blocks" in wx.last_error()
    assert lib.wamx_op_quantize_mxfp4(be.ptr, p, wx.TYPE_I32, 32, p, 1, 32) != 0
    assert lib.wamx_op_quantize_mxfp4(be.ptr, p, wx.TYPE_F32, 31, p, 1, 32) != 0
    assert lib.wamx_op_quantize_mxfp4(be.ptr, None, wx.TYPE_F32, 32, p, 1, 32) != 0
    assert lib.wamx_op_quantize_mxfp4(be.ptr, p, wx.TYPE_F32, 32, p, 0, 32) == 0
    assert lib.wamx_op_dequantize_mxfp4(be.ptr, p, p, wx.TYPE_F32, 31, 1, 32) != 0
    assert lib.wamx_op_mul_mat_mxfp4(be.ptr, p, p, wx.TYPE_BF16, 48, p, wx.TYPE_F32, 8, 8, 1, 48) != 0
    assert "multiple of 32" in wx.last_error()
    assert lib.wamx_op_mul_mat_mxfp4(be.ptr, p, p, wx.TYPE_F16, 32, p, wx.TYPE_F32, 8, 8, 1, 32) != 0
    assert lib.wamx_op_mul_mat_mxfp4(be.ptr, p, p, wx.TYPE_BF16, 32, p, wx.TYPE_F32, 7, 8, 1, 32) != 0
    assert lib.wamx_op_mul_mat_mxfp4(be.ptr, p, p, wx.TYPE_BF16, 32, p, wx.TYPE_F32, 8, 8, 0, 32) == 0
    assert lib.wamx_op_linear_mxfp4(be.ptr, p, p, wx.TYPE_BF16, None, wx.EPI_BIAS, None, None, p, 8, 1, 32) != 0
    assert "bias required" in wx.last_error()


class Graph:
    def __init__(self, wx, be):
        self.wx, self.be, self.lib = wx, be, be.lib
        self.ctx, self.leaves, self.gal = be.lib.wamx_init(256), be.lib.wamx_init(64), None

    def leaf(self, t, *ne):
        return self.lib.wamx_new_tensor_4d(self.leaves, t, *ne, *([1] * (4 - len(ne))))

    def place(self):
        self.buf = self.lib.wamx_backend_alloc_ctx_tensors(self.leaves, self.be.ptr)
        assert self.buf, self.wx.last_error()

    def set(self, t, a):
        a = np.ascontiguousarray(a)
        self.wx.check(self.lib.wamx_backend_tensor_set(t, a.ctypes.data, 0, a.nbytes))

    def get(self, t, dtype, shape):
        a = np.empty(shape, dtype)
        self.wx.check(self.lib.wamx_backend_tensor_get(t, a.ctypes.data, 0, a.nbytes))
        return a

    def build(self, *outs):
        self.g = self.lib.wamx_new_graph(self.ctx, 256)
        for t in outs:
            assert t, self.wx.last_error()
            self.lib.wamx_set_output(t)
            self.lib.wamx_build_forward_expand(self.g, t)
        self.lib.wamx_graph_assign_uid(self.g)
        self.gal = self.lib.wamx_gallocr_new(self.be.ptr)
        assert self.lib.wamx_gallocr_alloc_graph(self.gal, self.g), self.wx.last_error()

    def compute(self):
        self.wx.check(self.lib.wamx_backend_graph_compute(self.be.ptr, self.g))

    def close(self):
        if self.gal:
            self.lib.wamx_gallocr_free(self.gal)
        self.lib.wamx_buffer_free(self.buf)
        self.lib.wamx_free(self.ctx)
        self.lib.wamx_free(self.leaves)


def test_graph_quantize_multiply_and_gather(wx, be, rng):
    """CPY to MXFP4, MUL_MAT (rows in planes, and a row slice of the weight),
    LINEAR, CPY back and GET_ROWS in one computed graph, replayed."""
    lib, M, K = be.lib, 96, 128
    g = Graph(wx, be)
    w, x = g.leaf(wx.TYPE_F32, K, M), g.leaf(wx.TYPE_F32, K, 3, 2)
    ids, xb = g.leaf(wx.TYPE_I32, 4), g.leaf(wx.TYPE_BF16, K, 5)
    g.place()
    q = lib.wamx_cast(g.ctx, w, wx.TYPE_MXFP4)
    assert q.contents.nb[1] == K // 32 * 17 and lib.wamx_nbytes(q) == M * K // 32 * 17
    back = lib.wamx_cast(g.ctx, q, wx.TYPE_F32)
    y = lib.wamx_mul_mat(g.ctx, q, x)
    part = lib.wamx_view_2d(g.ctx, q, K, 40, K // 32 * 17, 8 * (K // 32 * 17))
    yp = lib.wamx_mul_mat(g.ctx, part, x)
    rows = lib.wamx_get_rows(g.ctx, q, ids)
    lin = lib.wamx_linear(g.ctx, q, xb, None, wx.EPI_NONE, None, None)
    g.build(back, y, yp, rows, lin)
    for seed in range(3):
        r = np.random.default_rng(seed)
        # halves up to 6 with a 6 in every block: exact
        wv = r.integers(-2, 3, (M, K)).astype(np.float32)
        wv[:, ::32] = 6
        xv = r.integers(-3, 4, (2, 3, K)).astype(np.float32)
        xbv = r.integers(-1, 2, (5, K)).astype(np.float32)
        idv = np.array([0, 95, 17, 17], np.int32)
        g.set(w, wv), g.set(x, xv), g.set(ids, idv), g.set(xb, wx.f32_to_bf16(xbv))
        g.compute()
        np.testing.assert_array_equal(g.get(back, np.float32, (M, K)), wv)
        np.testing.assert_array_equal(g.get(y, np.float32, (2, 3, M)), xv @ wv.T)
        np.testing.assert_array_equal(g.get(yp, np.float32, (2, 3, 40)), xv @ wv[8:48].T)
        np.testing.assert_array_equal(g.get(rows, np.float32, (4, K)), wv[idv])
        np.testing.assert_array_equal(g.get(lin, np.uint16, (5, M)), wx.f32_to_bf16((xbv @ wv.T).astype(np.float32)))
    g.close()


def test_graph_get_rows_outside_the_table_is_nan(wx, be):
    g = Graph(wx, be)
    w, ids = g.leaf(wx.TYPE_MXFP4, 64, 3), g.leaf(wx.TYPE_I32, 3)
    g.place()
    r = be.lib.wamx_get_rows(g.ctx, w, ids)
    g.build(r)
    wv = np.tile(np.arange(32, dtype=np.float64) % 7 - 3, (3, 2))
    g.set(w, ref.quantize(wv)), g.set(ids, np.array([2, -1, 3], np.int32))
    g.compute()
    got = g.get(r, np.float32, (3, 64))
    np.testing.assert_array_equal(got[0], ref.dequantize(ref.quantize(wv))[2].astype(np.float32))
    assert np.isnan(got[1:]).all()
    g.close()


def test_ggml_graph_with_a_quantised_weight(wx, be, rng):
    """A MUL_MAT on an "mxfp4" weight crosses the import boundary by name."""
    M, N, K = 48, 7, 96
    w = int_weights(rng, M, K)
    x = rng.integers(-3, 4, (N, K)).astype(np.float32)
    dw, dx, dy = be.array(w), be.array(x), be.empty(N * M * 4)

    class Desc(C.Structure):
        _fields_ = [("op", C.c_char_p), ("unary_op", C.c_char_p), ("type", C.c_char_p), ("ne", C.c_int64 * 4),
                    ("nb", C.c_size_t * 4), ("op_params", C.c_int32 * 16), ("flags", C.c_int32), ("src", C.c_int32 * 10),
                    ("view_src", C.c_int32), ("view_offs", C.c_size_t), ("data", C.c_void_p), ("name", C.c_char_p)]

    def desc(op, t, ne, nb, src, ptr):
        s = list(src) + [-1] * (10 - len(src))
        return Desc(op, None, t, (C.c_int64 * 4)(*ne), (C.c_size_t * 4)(*nb), (C.c_int32 * 16)(), 0, (C.c_int32 * 10)(*s),
                    -1, 0, ptr, op)

    rb = K // 32 * 17
    d = (Desc * 3)(desc(b"NONE", b"mxfp4", (K, M, 1, 1), (17, rb, rb * M, rb * M), (), dw.ptr),
                   desc(b"NONE", b"f32", (K, N, 1, 1), (4, 4 * K, 4 * K * N, 4 * K * N), (), dx.ptr),
                   desc(b"MUL_MAT", b"f32", (M, N, 1, 1), (4, 4 * M, 4 * M * N, 4 * M * N), (0, 1), dy.ptr))
    ctx = be.lib.wamx_init(16)
    graph = be.lib.wamx_graph_from_ggml(ctx, d, 3, (C.c_int32 * 1)(2), 1)
    assert graph, wx.last_error()
    wx.check(be.lib.wamx_backend_graph_compute(be.ptr, graph))
    np.testing.assert_array_equal(dy.download(np.float32, (N, M)), x @ ref.dequantize(w).astype(np.float32).T)
    be.lib.wamx_free(ctx)
