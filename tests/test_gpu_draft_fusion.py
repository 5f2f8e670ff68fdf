"""The head norms of a step's queries and keys and its V^T append, one launch of
a computed graph where nothing forbids it: same bits as the nodes by themselves,
and apart where they differ or meet in memory."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_draft import bf
from test_gpu_mxfp4 import Graph

pytestmark = pytest.mark.gpu

B, T, H, KV, DH, CAP = 2, 7, 6, 2, 64, 40
COLS = (H + 2 * KV) * DH


class Step:
    """Rows of packed columns, norms, lengths and caches, and the graph's nodes by name."""

    def __init__(self, wx, be, rng, order, **o):
        lib = be.lib
        self.wx, self.be, self.g = wx, be, Graph(wx, be)
        g, BF, I = self.g, wx.TYPE_BF16, wx.TYPE_I32
        leaf = {"x": (BF, COLS, B * T), "nq": (BF, DH), "nk": (BF, DH), "pos": (I, B * T), "pos2": (I, B * T), "past": (I, B),
                "past2": (I, B), "q": (BF, DH, T, H, B), "k": (BF, DH, CAP, KV, B), "v": (BF, CAP, DH, KV, B)}
        self.t = {n: g.leaf(*a) for n, a in leaf.items()}
        g.place()
        t = self.t
        part = lambda c, n: lib.wamx_view_2d(g.ctx, t["x"], n * DH, B * T, COLS * 2, c * DH * 2)  # noqa: E731
        make = {
            "q": lambda: lib.wamx_qk_head_norm_rope(g.ctx, part(0, H), t["nq"], t["q"], None, t["pos"], 2, o.get("dims_q", DH), 1e-6, 1e4),
            "k": lambda: lib.wamx_qk_head_norm_rope(g.ctx, part(H, KV), t["nk"], t["k"], t["past"], t[o.get("pos_k", "pos")], 2, DH,
                                                    1e-6, 1e4),
            "v": lambda: lib.wamx_vt_append(g.ctx, part(H + KV, KV), t["v"], t[o.get("past_v", "past")])}
        self.order = order
        g.build(*[make[n]() for n in order])
        data = {"x": bf(wx, rng.standard_normal((B * T, COLS)))[0], "nq": bf(wx, 1 + 0.1 * rng.standard_normal(DH))[0],
                "nk": bf(wx, 1 + 0.1 * rng.standard_normal(DH))[0], "pos": rng.integers(0, 5000, B * T).astype(np.int32),
                "pos2": rng.integers(0, 5000, B * T).astype(np.int32), "past": np.array([3, 30], np.int32),
                "past2": np.array([9, 0], np.int32), "q": np.full((B, H, T, DH), 0x4242, np.uint16),
                "k": bf(wx, rng.standard_normal((B, KV, CAP, DH)))[0], "v": bf(wx, rng.standard_normal((B, KV, DH, CAP)))[0]}
        self.data, self.o = data, o
        for n, a in data.items():
            g.set(t[n], a)

    def fused(self):
        before = self.be.lib.wamx_backend_fused_nodes(self.be.ptr)
        self.g.compute()
        return self.be.lib.wamx_backend_fused_nodes(self.be.ptr) - before

    def results(self):
        return {n: self.g.get(self.t[n], np.uint16, self.data[n].shape) for n in "qkv"}

    def alone(self):
        """The parts as calls of their own."""
        be, d = self.be, {n: self.be.array(a) for n, a in self.data.items()}
        for n in self.order:
            pos = d[self.o.get("pos_k", "pos")] if n == "k" else d["pos"]
            past = None if n == "q" else d[self.o.get("past_v", "past")].ptr if n == "v" else d["past"].ptr
            dims = self.o.get("dims_q", DH) if n == "q" else DH
            self.wx.check(be.lib.wamx_op_qkv_head_norm_rope(
                be.ptr, d["x"].ptr, COLS, d["nq"].ptr, d["nk"].ptr, pos.ptr, past, *[d[m].ptr if m == n else None for m in "qkv"],
                H, KV, DH, T, B, CAP, CAP, 2, dims, 1e-6, 1e4))
        return {n: d[n].download(np.uint16, self.data[n].shape) for n in "qkv"}


@pytest.mark.parametrize("order,along", [("qkv", 2), ("vkq", 2), ("kqv", 2), ("qk", 1), ("kv", 1), ("vq", 1), ("k", 0)])
def test_one_launch_same_bits(wx, be, rng, order, along):
    s = Step(wx, be, rng, order)
    assert s.fused() == along
    got, want = s.results(), s.alone()
    for n in "qkv":
        np.testing.assert_array_equal(got[n], want[n])
    s.g.close()


@pytest.mark.parametrize("order,o,along", [("qkv", {"dims_q": 32}, 1), ("qkv", {"pos_k": "pos2"}, 1), ("qkv", {"past_v": "past2"}, 1),
                                           ("kvq", {"past_v": "past2"}, 1)])
def test_differing_nodes_stay_apart(wx, be, rng, order, o, along):
    s = Step(wx, be, rng, order, **o)
    assert s.fused() == along
    got, want = s.results(), s.alone()
    for n in "qkv":
        np.testing.assert_array_equal(got[n], want[n])
    s.g.close()


def test_a_node_that_reads_an_earlier_ones_result_waits(wx, be, rng):
    """The second norm's rows are the first's result; the values that follow read the rows it wrote over."""
    lib = be.lib
    g, BF, I = Graph(wx, be), wx.TYPE_BF16, wx.TYPE_I32
    x, w, pos = g.leaf(BF, DH, T), g.leaf(BF, DH), g.leaf(I, T)
    a, b = g.leaf(BF, DH, T, 1, 1), g.leaf(BF, DH, T, 1, 1)
    g.place()
    first = lib.wamx_qk_head_norm_rope(g.ctx, x, w, a, None, pos, 0, 16, 1e-6, 1e4)
    second = lib.wamx_qk_head_norm_rope(g.ctx, lib.wamx_reshape_2d(g.ctx, first, DH, T), w, b, None, pos, 0, 16, 1e-6, 1e4)
    g.build(second)
    xs, ws, ps = bf(wx, rng.standard_normal((T, DH)))[0], bf(wx, 1 + 0.1 * rng.standard_normal(DH))[0], np.arange(T, dtype=np.int32)
    g.set(x, xs), g.set(w, ws), g.set(pos, ps)
    before = lib.wamx_backend_fused_nodes(be.ptr)
    g.compute()
    assert lib.wamx_backend_fused_nodes(be.ptr) == before
    d = [be.array(v) for v in (xs, ws, ps)]
    one, two = be.empty(T * DH * 2), be.empty(T * DH * 2)
    for src, dst in ((d[0], one), (one, two)):
        wx.check(lib.wamx_op_qkv_head_norm_rope(be.ptr, src.ptr, DH, d[1].ptr, None, d[2].ptr, None, dst.ptr, None, None, 1, 0, DH, T,
                                                1, T, T, 0, 16, 1e-6, 1e4))
    np.testing.assert_array_equal(g.get(b, np.uint16, (T, DH)), two.download(np.uint16, (T, DH)))
    g.close()


def test_replays_with_other_lengths(wx, be, rng):
    s = Step(wx, be, rng, "qkv")
    for step in range(4):
        s.data["past"] = np.array([step * 11, 33 - step * 10], np.int32)
        s.data["x"] = bf(wx, rng.standard_normal((B * T, COLS)))[0]
        for n in ("x", "past"):
            s.g.set(s.t[n], s.data[n])
        s.g.compute()
        want = s.alone()
        got = s.results()
        for n in "qkv":
            np.testing.assert_array_equal(got[n], want[n])
        s.data["k"], s.data["v"] = got["k"], got["v"]
    s.g.close()


def test_a_cache_view_off_its_alignment_is_refused(wx, be, rng):
    """What the single call refuses, the graph's constructor does too."""
    lib = be.lib
    g, BF, I = Graph(wx, be), wx.TYPE_BF16, wx.TYPE_I32
    q, v, par, past = g.leaf(BF, DH, 1, 1, 1), g.leaf(BF, 8, DH, 1, 1), g.leaf(I, 1, 1), g.leaf(I, 1)
    store = g.leaf(BF, DH * 8 + 8)
    g.place()
    for offset, ok in ((0, True), (2, False), (8, False), (16, True)):
        k = lib.wamx_view_4d(g.ctx, store, DH, 8, 1, 1, DH * 2, DH * 16, DH * 16, offset)
        o = lib.wamx_tree_attn(g.ctx, q, k, v, par, past, 1.0)
        assert bool(o) == ok and (ok or "16-byte aligned" in wx.last_error())
    g.close()
