"""Tree attention where the softmax can go wrong: NaN rows and keys through the
joins of split caches, scores of -Inf, maxima that rise slowly or in jumps; and
its graph replayed between other users of the workspace."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_draft import HALF, TREES, bf, head_norm_case, val
from test_gpu_mxfp4 import Graph

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
