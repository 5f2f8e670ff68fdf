"""Drafted tokens over a resident cache: per-head norm + rotation + append, tree
attention, and the whole 4-bit block as one computed graph, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import draft_ref as ref
from test_gpu_mxfp4 import Graph, int_weights

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8  # half a bf16 step, relative


def bf(wx, a):
    """(bits, f64 values)."""
    h = wx.f32_to_bf16(np.asarray(a, np.float32))
    return h, wx.bf16_to_f32(h).astype(np.float64)


def val(wx, h):
    return wx.bf16_to_f32(h).astype(np.float64)


# ---------------------------------------------------------------------------
# Head norm
# ---------------------------------------------------------------------------
def head_norm_case(wx, be, rng, batch, t, heads, kv, dh, dims, mode, past, cap, parts="qkv", ld_pad=0, base=1e6, pos=None):
    cols = (heads + 2 * kv) * dh
    xb, xv = bf(wx, rng.standard_normal((batch * t, cols + ld_pad)))
    xb[:, cols:] = 0x7FC0
    wq, wqv = bf(wx, 1 + 0.1 * rng.standard_normal(dh))
    wk, wkv = bf(wx, 1 + 0.1 * rng.standard_normal(dh))
    pos = np.asarray(pos if pos is not None else rng.integers(0, 200000, batch * t), np.int32)
    past = np.asarray(past, np.int32)
    ld = cap + 5
    k0, _ = bf(wx, rng.standard_normal((batch, kv, cap, dh)))
    v0, _ = bf(wx, rng.standard_normal((batch, kv, dh, ld)))
    q0 = np.full((batch, heads, t, dh), 0x4242, np.uint16)
    d = {n: be.array(a) for n, a in dict(x=xb, wq=wq, wk=wk, pos=pos, past=past, q=q0, k=k0, v=v0).items()}
    wx.check(be.lib.wamx_op_qkv_head_norm_rope(
        be.ptr, d["x"].ptr, cols + ld_pad, d["wq"].ptr, d["wk"].ptr, d["pos"].ptr, d["past"].ptr,
        d["q"].ptr if "q" in parts else None, d["k"].ptr if "k" in parts else None, d["v"].ptr if "v" in parts else None,
        heads, kv, dh, t, batch, cap, ld, mode, dims, 1e-6, base))
    q, k, v = (d[n].download(np.uint16, a.shape) for n, a in (("q", q0), ("k", k0), ("v", v0)))
    x = xv[:, :cols].reshape(batch, t, heads + 2 * kv, dh)

    def close(got, want, what):
        # one rounding to bf16; f32 norm and rotation: some 2^-20 of the pair's size (sin, cos in turns)
        tol = HALF * np.abs(want) + 2.0 ** -16 * max(1.0, np.abs(want).max())
        err = np.abs(val(wx, got) - want)
        assert (err <= tol).all(), (what, np.max(err - tol))

    for b in range(batch):
        pb = pos.reshape(batch, t)[b]
        qr = ref.rotate(ref.head_norm(x[b, :, :heads], wqv, 1e-6), pb, dims, mode, base).transpose(1, 0, 2)
        kr = ref.rotate(ref.head_norm(x[b, :, heads:heads + kv], wkv, 1e-6), pb, dims, mode, base).transpose(1, 0, 2)
        if "q" in parts:
            close(q[b], qr, "q")
        else:
            assert (q[b] == 0x4242).all()
        slots = past[b] + np.arange(t)
        ok = (slots >= 0) & (slots < cap)
        wantk, wantv = k0[b].copy(), v0[b].copy()
        if "k" in parts and ok.any():
            close(k[b][:, slots[ok]], kr[:, ok], "k")
            wantk[:, slots[ok]] = k[b][:, slots[ok]]
        np.testing.assert_array_equal(k[b], wantk)  # every other slot as it was
        if "v" in parts:
            wantv[:, :, slots[ok]] = xb[:, :cols].reshape(batch, t, -1, dh)[b, ok, heads + kv:].transpose(1, 2, 0)
        np.testing.assert_array_equal(v[b], wantv)


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("mode", [0, 2])
@pytest.mark.parametrize("dims", ["all", "half", 16, 0])
def test_head_norm_rotations(wx, be, rng, dh, mode, dims):
    n = dict(all=dh, half=dh // 2).get(dims, dims)
    print(f"head norm dh {dh} mode {mode} dims {n}", flush=True)
    head_norm_case(wx, be, rng, 2, 3, 5, 2, dh, n, mode, [4, 0], 9)


@pytest.mark.parametrize("batch,t,heads,kv,past,cap", [
    (1, 1, 1, 1, [0], 1), (1, 1, 24, 24, [77], 80), (3, 1, 8, 1, [0, 5, 9], 10), (2, 63, 4, 2, [1, 30], 128),
    (1, 64, 3, 3, [64], 128), (2, 65, 7, 1, [0, 3], 70), (1, 400, 28, 4, [11], 420), (4, 130, 32, 8, [0, 1, 2, 3], 140)])
def test_head_norm_sizes(wx, be, rng, batch, t, heads, kv, past, cap):
    print(f"head norm {batch}x{t} heads {heads}/{kv}", flush=True)
    head_norm_case(wx, be, rng, batch, t, heads, kv, 128, 128, 2, past, cap, ld_pad=3)


@pytest.mark.parametrize("parts", ["q", "k", "v", "qk", "kv"])
def test_head_norm_parts(wx, be, rng, parts):
    head_norm_case(wx, be, rng, 2, 5, 4, 2, 64, 64, 0, [3, 1], 12, parts=parts)


def test_head_norm_slots_outside_the_cache_are_dropped(wx, be, rng):
    """A length that leaves no room writes the slots that exist, and nothing else."""
    head_norm_case(wx, be, rng, 4, 6, 4, 2, 64, 64, 0, [-3, 7, 100, 2147483647], 10)


def test_head_norm_far_and_negative_positions(wx, be, rng):
    head_norm_case(wx, be, rng, 1, 6, 2, 1, 128, 128, 0, [0], 8, base=10000.0,
                   pos=[0, 1, -1, 2147483647, -2147483648, 1000003])


def test_head_norm_specials(wx, be):
    """A head of zeros gives zeros; an Inf or NaN stays in its head."""
    lib, dh = be.lib, 64
    x = np.ones((1, 3 * dh), np.float32)
    x[0, :dh] = 0
    x[0, dh + 3] = np.nan
    w = wx.f32_to_bf16(np.ones(dh, np.float32))
    d = [be.array(a) for a in (wx.f32_to_bf16(x), w, np.zeros(1, np.int32))]
    q = be.array(np.zeros((3, dh), np.uint16))
    wx.check(lib.wamx_op_qkv_head_norm_rope(be.ptr, d[0].ptr, 3 * dh, d[1].ptr, None, d[2].ptr, None, q.ptr, None, None,
                                            3, 0, dh, 1, 1, 0, 0, 2, dh, 1e-6, 1e4))
    got = val(wx, q.download(np.uint16, (3, dh)))
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and (got[2] == 1).all()


# ---------------------------------------------------------------------------
# Tree attention
# ---------------------------------------------------------------------------
TREES = {
    "chain": lambda r, t: [i - 1 for i in range(t)],
    "star": lambda r, t: [-1] * t,
    "binary": lambda r, t: [(i - 1) // 2 if i else -1 for i in range(t)],
    "random": lambda r, t: [int(r.integers(-1, i)) if i else -1 for i in range(t)],
    "backwards": lambda r, t: [i + 1 if i + 1 < t else -1 for i in range(t)],
}


def tree_case(wx, be, rng, batch, t, heads, kv, dh, past, cap, tree="random", parents=None, scale=None, qstd=1.0,
              fill=None, ld=None):
    scale = scale if scale is not None else dh ** -0.5
    past = np.asarray(past, np.int32)
    ld = ld or (cap + 7) // 8 * 8
    par = np.asarray(parents if parents is not None else [TREES[tree](rng, t) for _ in range(batch)], np.int32)
    q, qv = bf(wx, rng.standard_normal((batch, heads, t, dh)) * qstd)
    k, _ = bf(wx, rng.standard_normal((batch, kv, cap, dh)))
    v, _ = bf(wx, rng.standard_normal((batch, kv, dh, ld)))
    if fill is not None:  # behind the last drafted slot: anything
        for b in range(batch):
            n = max(0, past[b] + t)
            k[b, :, n:], v[b, :, :, n:] = fill, fill
    d = [be.array(a) for a in (q, k, v, par, past)]
    out = be.array(np.full((batch * t + 1, heads * dh), 0x4242, np.uint16))
    wx.check(be.lib.wamx_op_tree_attn(be.ptr, *[a.ptr for a in d], out.ptr, heads, kv, dh, t, batch, cap, ld, scale))
    got = out.download(np.uint16, (batch * t + 1, heads * dh))
    assert (got[-1] == 0x4242).all(), "written behind the result"
    for b in range(batch):
        want, mass = ref.tree_attn(qv[b], val(wx, k[b]), val(wx, v[b]), par[b], int(past[b]), scale)
        err = np.abs(val(wx, got[b * t:(b + 1) * t]).reshape(t, heads, dh) - want)
        # Probabilities enter the product in bf16 (half a step each), scores are
        # f32 sums of dh products (about 2^-17 of p for scores up to some tens),
        # and the result is rounded once.
        tol = (HALF + 2.0 ** -12) * mass + HALF * np.abs(want)
        assert (err <= tol).all(), (b, np.max(err - tol), np.argwhere(err > tol)[:3])
    return got


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("tree", list(TREES))
def test_tree_shapes(wx, be, rng, dh, tree):
    print(f"tree {tree} dh {dh}", flush=True)
    tree_case(wx, be, rng, 2, 13, 4, 2, dh, [50, 3], 80, tree, fill=0x7FC0)


@pytest.mark.parametrize("batch,t,heads,kv,past,cap", [
    (1, 1, 1, 1, [0], 1), (1, 1, 1, 1, [1], 2), (1, 1, 8, 8, [31], 32), (2, 2, 4, 4, [0, 30], 33), (1, 8, 24, 24, [120], 128),
    (3, 16, 2, 1, [47, 48, 49], 70), (1, 17, 2, 2, [15], 40), (2, 31, 4, 2, [64, 33], 100), (1, 33, 6, 2, [100], 160),
    (1, 64, 8, 2, [300], 364), (2, 65, 2, 1, [63, 0], 130), (1, 129, 2, 2, [7], 140), (1, 256, 4, 4, [5], 261),
    (1, 200, 16, 2, [333], 540)])
@pytest.mark.parametrize("dh", [64, 128])
def test_tree_sizes(wx, be, rng, batch, t, heads, kv, past, cap, dh):
    print(f"tree {batch}x{t} heads {heads}/{kv} past {past} dh {dh}", flush=True)
    tree_case(wx, be, rng, batch, t, heads, kv, dh, past, cap, fill=0xFF80)


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("t,heads,kv", [(1, 4, 1), (5, 4, 2), (20, 2, 2), (40, 4, 2)])
def test_tree_long_cache_is_split(wx, be, rng, dh, t, heads, kv):
    print(f"tree long dh {dh} t {t}", flush=True)
    tree_case(wx, be, rng, 2, t, heads, kv, dh, [9000, 4097], 9100, fill=0x7FC0)


def test_tree_capacity_far_above_the_lengths(wx, be, rng):
    """Splits planned from the capacity; short, empty and full sequences in one call."""
    tree_case(wx, be, rng, 4, 4, 4, 2, 64, [0, 1, 12000, 20], 12004, fill=0x7F80)


@pytest.mark.parametrize("batch", [64, 65, 70])
def test_tree_many_sequences(wx, be, rng, batch):
    """Slots shared out by length up to 64 sequences, evenly above; some empty, some long."""
    past = [0 if b % 7 == 0 else 3000 - 40 * b for b in range(batch)]
    tree_case(wx, be, rng, batch, 2, 2, 1, 64, past, 3008, fill=0x7F80)


@pytest.mark.parametrize("scale", [0.0, -0.125])
def test_tree_zero_and_negative_scale(wx, be, rng, scale):
    tree_case(wx, be, rng, 2, 5, 4, 2, 64, [100, 40], 120, scale=scale)
    tree_case(wx, be, rng, 1, 40, 4, 2, 128, [100], 160, scale=scale)


def test_tree_slots_without_a_token(wx, be, rng):
    """Padding sees nothing, gives zero rows, and nothing sees it."""
    par = [[-1, 0, -2, 1, 99, -5, 3], [-2] * 7]
    got = tree_case(wx, be, rng, 2, 7, 4, 2, 128, [20, 20], 40, parents=par)
    assert not got[[2, 4, 5] + list(range(7, 14))].any()


def test_tree_lengths_that_do_not_fit_give_zeros(wx, be, rng):
    got = tree_case(wx, be, rng, 4, 3, 2, 2, 64, [-1, 38, 37, 2147483647], 40)
    assert not got[0:6].any() and got[6:9].any() and not got[9:12].any()


def test_tree_cycles_end(wx, be, rng):
    """Parents that form a cycle: each token sees the members it reaches."""
    tree_case(wx, be, rng, 1, 5, 2, 1, 64, [10], 20, parents=[[2, 0, 1, 3, 3]])


@pytest.mark.parametrize("qstd", [0.01, 30.0])
def test_tree_flat_and_peaked_scores(wx, be, rng, qstd):
    """Scores up to hundreds: the running maximum carries them.  At 30 a score
    is a f32 sum of 128 products near 30 each, off by up to 2^-10 or so, so the
    probabilities keep 2^-10; that fits within HALF + 2^-12 times twice."""
    tree_case(wx, be, rng, 1, 9, 4, 2, 128, [2000], 2050, qstd=qstd, scale=128 ** -0.5 / (4 if qstd > 1 else 1))


def test_tree_infinite_and_nan_drafts_reach_their_descendants_only(wx, be, rng):
    """V of a drafted slot holds Inf or NaN: rows whose path misses the slot are
    as if it were not there."""
    for dh in (64, 128, 256):
        t, past, cap = 6, 40, 64
        par = [-1, 0, 0, 1, 2, -1]
        q, qv = bf(wx, rng.standard_normal((1, 2, t, dh)))
        k, kv = bf(wx, rng.standard_normal((1, 1, cap, dh)))
        v, _ = bf(wx, rng.standard_normal((1, 1, dh, cap)))
        bad = v.copy()
        bad[0, 0, 3, past + 1] = 0x7F80  # +Inf in token 1, seen by 1 and 3
        bad[0, 0, 5, past + 4] = 0x7FC0  # NaN in token 4, seen by 4
        kbad = k.copy()
        kbad[0, 0, past + 5] = 0x7FC0    # NaN keys of token 5, seen by 5

        def run(kk, vv):
            d = [be.array(a) for a in (q, kk, vv, np.array(par, np.int32), np.array([past], np.int32))]
            o = be.empty(t * 2 * dh * 2)
            wx.check(be.lib.wamx_op_tree_attn(be.ptr, *[a.ptr for a in d], o.ptr, 2, 1, dh, t, 1, cap, cap, dh ** -0.5))
            return val(wx, o.download(np.uint16, (t, 2, dh)))

        clean, got = run(k, v), run(kbad, bad)
        assert (got[[1, 3], :, 3] == np.inf).all() and np.isnan(got[4, :, 5]).all() and np.isnan(got[5]).all()
        want = clean.copy()
        want[[1, 3], :, 3], want[4, :, 5], want[5] = got[[1, 3], :, 3], got[4, :, 5], got[5]
        np.testing.assert_array_equal(got, want)


def test_tree_same_bits_every_run(wx, be, rng):
    a = tree_case(wx, be, np.random.default_rng(3), 2, 24, 8, 2, 128, [5000, 4000], 5100)
    b = tree_case(wx, be, np.random.default_rng(3), 2, 24, 8, 2, 128, [5000, 4000], 5100)
    np.testing.assert_array_equal(a, b)


def test_refusals(wx, be):
    lib, d = be.lib, be.empty(1 << 16)
    p = d.ptr

    def tree(**o):
        a = dict(q=p, k=p, vt=p, par=p, past=None, out=p, heads=2, kv=1, dh=64, t=2, b=1, cap=8, ld=8, scale=1.0)
        a.update(o)
        return lib.wamx_op_tree_attn(be.ptr, *a.values())

    for bad in (dict(dh=80), dict(t=257, cap=300, ld=304), dict(cap=1), dict(heads=3, kv=2), dict(ld=12, cap=9), dict(ld=0),
                dict(q=p + 2), dict(vt=p + 8), dict(par=None), dict(kv=0), dict(b=70000)):
        assert tree(**bad) != 0, bad
        assert "wamx_op_tree_attn" in wx.last_error()
    assert tree(t=0) == 0 and tree(b=0) == 0

    def norm(**o):
        a = dict(x=p, ldx=512, wq=p, wk=p, pos=p, past=None, q=p, k=p, vt=p, heads=2, kv=1, dh=64, t=1, b=1, cap=4, ld=4,
                 mode=0, dims=64, eps=1e-6, base=1e4)
        a.update(o)
        return lib.wamx_op_qkv_head_norm_rope(be.ptr, *a.values())

    for bad in (dict(dh=96), dict(mode=1), dict(dims=24), dict(dims=80), dict(pos=None), dict(ldx=255), dict(t=5), dict(ld=3),
                dict(wq=None), dict(eps=-1.0), dict(base=0.0), dict(heads=-1)):
        assert norm(**bad) != 0, bad
        assert "wamx_op_qkv_head_norm_rope" in wx.last_error()
    assert norm(t=0) == 0


# ---------------------------------------------------------------------------
# The operators together
# ---------------------------------------------------------------------------
def test_block_as_one_graph(wx, be):
    """4-bit QKV product, head norm and rotation into the cache, tree attention,
    4-bit output product: one computed graph, replayed with other lengths, trees
    and inputs, equal to the single calls bit for bit."""
    rng = np.random.default_rng(11)
    lib, B, T, H, KV, dh, K, cap = be.lib, 2, 9, 4, 2, 64, 160, 96
    inner, cols = H * dh, (H + 2 * KV) * dh
    g = Graph(wx, be)
    leaf = lambda t, *ne: g.leaf(t, *ne)  # noqa: E731
    I, BF, MX = wx.TYPE_I32, wx.TYPE_BF16, wx.TYPE_MXFP4
    x, wqkv, wo = leaf(BF, K, B * T), leaf(MX, K, cols), leaf(MX, inner, K)
    nq, nk = leaf(BF, dh), leaf(BF, dh)
    pos, past, par = leaf(I, B * T), leaf(I, B), leaf(I, T, B)
    qb, kc, vc = leaf(BF, dh, T, H, B), leaf(BF, dh, cap, KV, B), leaf(BF, cap, dh, KV, B)
    g.place()
    qkv = lib.wamx_linear(g.ctx, wqkv, x, None, wx.EPI_NONE, None, None)
    part = lambda c, n: lib.wamx_view_2d(g.ctx, qkv, n * dh, B * T, cols * 2, c * dh * 2)  # noqa: E731
    q = lib.wamx_qk_head_norm_rope(g.ctx, part(0, H), nq, qb, None, pos, 2, dh, 1e-6, 1e4)
    k = lib.wamx_qk_head_norm_rope(g.ctx, part(H, KV), nk, kc, past, pos, 2, dh, 1e-6, 1e4)
    v = lib.wamx_vt_append(g.ctx, part(H + KV, KV), vc, past)
    assert q and k and v, wx.last_error()
    at = lib.wamx_tree_attn(g.ctx, q, k, v, par, past, dh ** -0.5)
    y = lib.wamx_linear(g.ctx, wo, lib.wamx_reshape_2d(g.ctx, at, inner, B * T), None, wx.EPI_NONE, None, None)
    g.build(y)
    data = dict(wqkv=ref.quantize(rng.standard_normal((cols, K)) * 0.05), wo=ref.quantize(rng.standard_normal((K, inner)) * 0.05),
                nq=bf(wx, 1 + 0.1 * rng.standard_normal(dh))[0], nk=bf(wx, 1 + 0.1 * rng.standard_normal(dh))[0],
                kc=bf(wx, rng.standard_normal((B, KV, cap, dh)))[0], vc=bf(wx, rng.standard_normal((B, KV, dh, cap)))[0])
    for t, n in ((wqkv, "wqkv"), (wo, "wo"), (nq, "nq"), (nk, "nk"), (kc, "kc"), (vc, "vc")):
        g.set(t, data[n])
    ka, va = data["kc"], data["vc"]
    for step in range(4):
        xs = bf(wx, rng.standard_normal((B * T, K)))[0]
        pasts = np.array([3 + 20 * step, 87 - 9 * step], np.int32)
        posv = (pasts[:, None] + np.arange(T)).astype(np.int32)
        parv = np.array([TREES["random"](rng, T), TREES["binary"](rng, T)], np.int32)
        g.set(x, xs), g.set(past, pasts), g.set(pos, posv), g.set(par, parv)
        g.compute()
        got = g.get(y, np.uint16, (B * T, K))
        # the same through the single calls
        d = {n: be.array(a) for n, a in dict(x=xs, wqkv=data["wqkv"], wo=data["wo"], nq=data["nq"], nk=data["nk"], past=pasts,
                                             pos=posv, par=parv, k=ka, v=va).items()}
        pq, q1, a1, y1 = be.empty(B * T * cols * 2), be.empty(B * T * inner * 2), be.empty(B * T * inner * 2), be.empty(B * T * K * 2)
        wx.check(lib.wamx_op_linear_mxfp4(be.ptr, d["wqkv"].ptr, d["x"].ptr, BF, None, 0, None, None, pq.ptr, cols, B * T, K))
        wx.check(lib.wamx_op_qkv_head_norm_rope(be.ptr, pq.ptr, cols, d["nq"].ptr, d["nk"].ptr, d["pos"].ptr, d["past"].ptr,
                                                q1.ptr, d["k"].ptr, d["v"].ptr, H, KV, dh, T, B, cap, cap, 2, dh, 1e-6, 1e4))
        wx.check(lib.wamx_op_tree_attn(be.ptr, q1.ptr, d["k"].ptr, d["v"].ptr, d["par"].ptr, d["past"].ptr, a1.ptr, H, KV, dh, T,
                                       B, cap, cap, dh ** -0.5))
        wx.check(lib.wamx_op_linear_mxfp4(be.ptr, d["wo"].ptr, a1.ptr, BF, None, 0, None, None, y1.ptr, K, B * T, inner))
        np.testing.assert_array_equal(got, y1.download(np.uint16, (B * T, K)))
        ka, va = d["k"].download(np.uint16, ka.shape), d["v"].download(np.uint16, va.shape)
        np.testing.assert_array_equal(g.get(kc, np.uint16, ka.shape), ka)
        np.testing.assert_array_equal(g.get(vc, np.uint16, va.shape), va)
        # and the block's middle against 64 bits
        for b in range(B):
            want, mass = ref.tree_attn(val(wx, q1.download(np.uint16, (B, H, T, dh))[b]), val(wx, ka[b]), val(wx, va[b]),
                                       parv[b], int(pasts[b]), dh ** -0.5)
            err = np.abs(val(wx, a1.download(np.uint16, (B, T, H, dh))[b]) - want)
            assert (err <= (HALF + 2.0 ** -12) * mass + HALF * np.abs(want)).all()
    g.close()
