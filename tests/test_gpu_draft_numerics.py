"""Tree attention where the softmax can go wrong: NaN rows and keys through the
joins of split caches, scores of -Inf, maxima that rise slowly or in jumps; and
its graph replayed between other users of the workspace."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_draft import HALF, TREES, bf, head_norm_case, val
from test_gpu_mxfp4 import Graph, int_weights

pytestmark = pytest.mark.gpu

# One workgroup a sequence; units joined a row at a time (few rows, many rows);
# units joined many rows at a time (few rows, many rows).
FORMS = [(3, 4, 2, 64, [20, 7]), (1, 4, 1, 128, [9000, 100]), (65, 2, 1, 64, [5000, 3000]), (3, 4, 2, 256, [900, 1000]),
         (40, 8, 2, 128, [1500, 0])]


def inputs(wx, rng, t, heads, kv, dh, past, positive=False):
    B, cap = len(past), max(past) + t + 3
    ld = (cap + 7) // 8 * 8
    q = rng.standard_normal((B, heads, t, dh))
    q = bf(wx, np.abs(q) + 0.1 if positive else q)[0]
    k, v = bf(wx, rng.standard_normal((B, kv, cap, dh)))[0], bf(wx, rng.standard_normal((B, kv, dh, ld)))[0]
    par = np.array([TREES["random"](rng, t) for _ in past], np.int32)
    return q, k, v, par, np.array(past, np.int32)


def run(wx, be, q, k, v, par, past, scale=None):
    B, heads, t, dh = q.shape
    kv, cap, ld = k.shape[1], k.shape[2], v.shape[3]
    d = [be.array(a) for a in (q, k, v, par, past)]
    out = be.empty(B * t * heads * dh * 2)
    wx.check(be.lib.wamx_op_tree_attn(be.ptr, *[a.ptr for a in d], out.ptr, heads, kv, dh, t, B, cap, ld,
                                      dh ** -0.5 if scale is None else scale))
    return val(wx, out.download(np.uint16, (B, t, heads, dh)))


def close(wx, got, q, k, v, par, past, scale):
    """The bounds of the other tests of this operator: probabilities enter the
    product in bf16, scores are f32 sums, the result is rounded once."""
    for b in range(len(past)):
        want, mass = ref.tree_attn(val(wx, q[b]), val(wx, k[b]), val(wx, v[b]), par[b], int(past[b]), scale)
        err = np.abs(got[b] - want)
        tol = (HALF + 2.0 ** -12) * mass + HALF * np.abs(want)
        assert (err <= tol).all(), (b, np.max(err - tol), np.argwhere(~(err <= tol))[:3])


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
def test_nan_query_rows_stay_nan_and_alone(wx, be, rng, t, heads, kv, dh, past):
    print(f"nan rows t {t} heads {heads}/{kv} dh {dh} past {past}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past)
    clean = run(wx, be, q, k, v, par, past)
    bad = q.copy()
    hit = np.zeros((2, t, heads), bool)
    for b, h, i in ((0, 0, 0), (0, heads - 1, t - 1), (1, 1, t // 2)):
        bad[b, h, i, 5] = 0x7FC0
        hit[b, i, h] = True
    got = run(wx, be, bad, k, v, par, past)
    assert np.isnan(got[hit]).all()
    np.testing.assert_array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
def test_a_nan_key_of_the_cache_reaches_its_heads(wx, be, rng, t, heads, kv, dh, past):
    print(f"nan key t {t} heads {heads}/{kv} dh {dh} past {past}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past)
    clean = run(wx, be, q, k, v, par, past)
    bad = k.copy()
    bad[0, kv - 1, past[0] // 2, 1] = 0x7FC0
    got = run(wx, be, q, bad, v, par, past)
    first = heads - heads // kv
    assert np.isnan(got[0, :, first:]).all()
    np.testing.assert_array_equal(got[0, :, :first], clean[0, :, :first])
    np.testing.assert_array_equal(got[1], clean[1])


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
def test_scores_of_minus_infinity_have_no_weight(wx, be, rng, t, heads, kv, dh, past):
    """Keys of -Inf against positive queries, whole tiles of them first: the rest decides."""
    print(f"-inf keys t {t} heads {heads}/{kv} dh {dh} past {past}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past, positive=True)
    n = min(int(past[past > 0].min()) - 2, 200)
    k[:, :, :n] = 0xFF80
    got = run(wx, be, q, k, v, par, past)
    short = np.where(past > 0, past - n, past)
    for b in range(len(past)):
        keep = slice(n if past[b] else 0, None)
        if past[b] == 0:  # its drafted slots lie among the -Inf keys: nothing is left of them
            continue
        close(wx, got[b:b + 1], q[b:b + 1], k[b:b + 1, :, keep], v[b:b + 1, :, :, keep], par[b:b + 1], short[b:b + 1], dh ** -0.5)


@pytest.mark.parametrize("t,heads,kv,dh,past", FORMS)
@pytest.mark.parametrize("step", [0.02, 0.13, -0.05, 2.0])
def test_rising_and_falling_scores(wx, be, rng, t, heads, kv, dh, past, step):
    """Scores step * slot: within a tile of 64 slots they pass a running maximum
    by less and by more than the 8 (in powers of two) that moves it."""
    print(f"rising t {t} heads {heads}/{kv} dh {dh} past {past} step {step}", flush=True)
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, past)
    q[:], k[:] = 0, 0
    q[..., 0] = 0x3F80  # 1
    slots = np.arange(k.shape[2]) % 2000
    k[..., 0] = wx.f32_to_bf16((slots * step).astype(np.float32))
    close(wx, run(wx, be, q, k, v, par, past, 1.0), q, k, v, par, past, 1.0)


@pytest.mark.parametrize("t", [1, 8, 64, 130])
def test_appends_at_every_place_in_a_tile(wx, be, rng, t):
    """V^T is written eight slots at a time where all eight are new; the slots
    beside them keep what they hold."""
    print(f"append t {t}", flush=True)
    past = [0, 1, 7, 8, 57, 63, 64, 65, 200 - t]
    head_norm_case(wx, be, rng, len(past), t, 2, 1, 64, 64, 2, past, 200)
    head_norm_case(wx, be, rng, len(past), t, 2, 2, 128, 32, 0, past, 203, ld_pad=5)


def test_two_split_graphs_replayed_between_single_calls(wx, be):
    lib, rng = be.lib, np.random.default_rng(5)
    sets = [(2, 4, 1, 128, [4000, 37]), (40, 8, 2, 64, [3000, 500])]
    graphs = []
    for t, heads, kv, dh, past in sets:
        q, k, v, par, pst = inputs(wx, rng, t, heads, kv, dh, past)
        cap = ld = v.shape[3]  # a cache's K and V^T have as many slots
        data = (q, np.concatenate([k, k[:, :, :cap - k.shape[2]]], 2), v, par, pst)
        g, B = Graph(wx, be), len(past)
        q, k = g.leaf(wx.TYPE_BF16, dh, t, heads, B), g.leaf(wx.TYPE_BF16, dh, cap, kv, B)
        v, par, pst = g.leaf(wx.TYPE_BF16, ld, dh, kv, B), g.leaf(wx.TYPE_I32, t, B), g.leaf(wx.TYPE_I32, B)
        g.place()
        y = lib.wamx_tree_attn(g.ctx, q, k, v, par, pst, dh ** -0.5)
        g.build(y)
        for leaf, a in zip((q, k, v, par, pst), data):
            g.set(leaf, a)
        graphs.append((g, pst, y, data))
    for step in range(4):
        for g, pst, y, (q, k, v, par, past) in graphs:
            now = np.maximum(past - 600 * step, 0).astype(np.int32)
            g.set(pst, now)
            g.compute()
            B, heads, t, dh = q.shape
            got = val(wx, g.get(y, np.uint16, (B, t, heads, dh)))
            np.testing.assert_array_equal(got, run(wx, be, q, k, v, par, now))
    for g, *_ in graphs:
        g.close()


def test_split_kernels_on_two_lanes(wx, be):
    """A split 4-bit product on one lane beside a split attention on the other,
    each with a workspace of its lane; the attention's result meets the product's
    next weight.  Replayed, and equal to the single calls."""
    lib, rng = be.lib, np.random.default_rng(6)
    M, N, K, t, heads, kv, dh = 256, 40, 12288, 5, 4, 2, 64
    q, k, v, par, past = inputs(wx, rng, t, heads, kv, dh, [2900, 700])
    cap = v.shape[3]
    k = np.concatenate([k, k[:, :, :cap - k.shape[2]]], 2)
    g, B, BF, I = Graph(wx, be), 2, wx.TYPE_BF16, wx.TYPE_I32
    w, x, w2 = g.leaf(wx.TYPE_MXFP4, K, M), g.leaf(BF, K, N), g.leaf(wx.TYPE_MXFP4, heads * dh, 96)
    tq, tk, tv = g.leaf(BF, dh, t, heads, B), g.leaf(BF, dh, cap, kv, B), g.leaf(BF, cap, dh, kv, B)
    tpar, tpast = g.leaf(I, t, B), g.leaf(I, B)
    g.place()
    lib.wamx_set_lane(g.ctx, 1)
    at = lib.wamx_tree_attn(g.ctx, tq, tk, tv, tpar, tpast, dh ** -0.5)
    y2 = lib.wamx_mul_mat(g.ctx, w2, lib.wamx_reshape_2d(g.ctx, at, heads * dh, B * t))
    lib.wamx_set_lane(g.ctx, 0)
    y = lib.wamx_mul_mat(g.ctx, w, x)
    g.build(y, y2)
    w2v = ref.quantize(rng.standard_normal((96, heads * dh)) * 0.05)
    for leaf, a in ((tq, q), (tk, k), (tv, v), (tpar, par), (w2, w2v)):
        g.set(leaf, a)
    for step in range(4):
        wv, xv = int_weights(rng, M, K), rng.integers(-3, 4, (N, K)).astype(np.float32)
        now = (past - 500 * (step % 2)).astype(np.int32)
        g.set(w, wv), g.set(x, wx.f32_to_bf16(xv)), g.set(tpast, now)
        g.compute()
        np.testing.assert_array_equal(g.get(y, np.float32, (N, M)), xv @ ref.dequantize(wv).astype(np.float32).T)
        a = wx.f32_to_bf16(run(wx, be, q, k, v, par, now).reshape(B * t, heads * dh).astype(np.float32))
        d, dw, out = be.array(a), be.array(w2v), be.empty(B * t * 96 * 4)
        wx.check(lib.wamx_op_mul_mat_mxfp4(be.ptr, dw.ptr, d.ptr, BF, heads * dh, out.ptr, wx.TYPE_F32, 96, 96, B * t, heads * dh))
        np.testing.assert_array_equal(g.get(y2, np.float32, (B * t, 96)), out.download(np.float32, (B * t, 96)))
    g.close()
