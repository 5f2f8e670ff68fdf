"""The 4-bit decode block's operators, as cases that can be timed.

  quantize   rows of f32, f16 or bf16 to MXFP4 (32 values share one power of
             two, each value in 4 bits) and back to the values they stand for
  product    y = W x with W in MXFP4 and 16-bit or f32 activations: one token,
             the tokens of an action chunk, prompts
  headnorm   a packed QKV projection to the attention's operands in one call:
             RMSNorm of every query and key head, rotation by position, keys
             and transposed values written behind the resident cache
  tree       attention of a tree of drafted tokens over the resident cache:
             every token sees the cache, its ancestors and itself

`own` selects the framework's operators; otherwise the plain torch forms run.
Tensors are torch's; the backend takes their device pointers and runs on a
blocking stream, which the null stream that torch uses is ordered with.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 30}
EPS = 1e-6


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One activation row set of an odd prompt, kept in 4 bits.
        dict(name="quantize_rows", kind="quantize", rows=77, cols=4096, x="bf16"),
        # A whole FFN weight quantised when a model is loaded.
        dict(name="quantize_weight", kind="quantize", rows=14336, cols=4096, x="f32"),
        # One token through an output projection: all latency and weight bytes.
        dict(name="product_1", kind="product", m=4096, n=1, k=4096, x="bf16", y="bf16"),
        # The 48 tokens of an action chunk through the FFN's first product.
        dict(name="product_48", kind="product", m=14336, n=48, k=4096, x="bf16", y="bf16"),
        # An odd prompt, f32 activations and result as a ggml graph has them, an odd output width.
        dict(name="product_333", kind="product", m=10250, n=333, k=2048, x="f32", y="f32"),
        # A long prompt through the FFN's first product.
        dict(name="product_2048", kind="product", m=14336, n=2048, k=4096, x="bf16", y="bf16"),
        # One decoded token of one sequence: latency.
        dict(name="headnorm_1", kind="headnorm", batch=1, t=1, heads=24, kv=24, dh=128, dims=128, mode=0, past=1025),
        # Two ragged prompts with grouped heads, rotated by halves.
        dict(name="headnorm_4000", kind="headnorm", batch=2, t=2001, heads=32, kv=8, dh=128, dims=128, mode=2, past=600),
        # A short draft behind a short prompt: latency.
        dict(name="tree_8", kind="tree", batch=1, t=8, heads=24, kv=24, dh=128, past=120),
        # Drafts of 64 tokens for four sequences with long caches, four query heads to a key head.
        dict(name="tree_64", kind="tree", batch=4, t=64, heads=32, kv=8, dh=128, past=16000),
        # One token at a time over a very long cache, narrow heads.
        dict(name="tree_1_long", kind="tree", batch=2, t=1, heads=16, kv=4, dh=64, past=100000),
        # An odd draft, one key head per query head, wide heads.
        dict(name="tree_33_wide", kind="tree", batch=3, t=33, heads=8, kv=8, dh=256, past=5001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "headnorm", "tree", "tree"])
    if kind == "quantize":
        cols = 32 * _log(rng, 1, 448)
        rows = min(_log(rng, 1, 14336), 58720256 // cols)
        return dict(kind=kind, rows=rows, cols=cols, x=rng.choice(["f32", "f16", "bf16"]))
    if kind == "product":
        # Widths with every remainder, and the round ones.
        m = rng.choice([_log(rng, 33, 14336), 128 * rng.randint(4, 112)])
        k = 32 * rng.choice([_log(rng, 2, 448), 4 * rng.randint(4, 112)])
        n = _log(rng, 1, 2048)
        while m * n * k > 14336 * 2048 * 4096:
            n //= 2
        return dict(kind=kind, m=m, n=n, k=k, x=rng.choice(["bf16", "bf16", "f32"]), y=rng.choice(["bf16", "bf16", "f32"]))
    heads, kv = rng.choice([(24, 24), (32, 8), (16, 16), (16, 2), (12, 4), (8, 1), (5, 5), (28, 4)])
    dh = rng.choice([64, 128, 128, 256])
    if kind == "headnorm":
        t = _log(rng, 1, 2000)
        batch = rng.randint(1, max(1, min(8, 4000 // t)))
        return dict(kind=kind, batch=batch, t=t, heads=heads, kv=kv, dh=dh, dims=rng.choice([dh, dh, dh // 2, dh // 4]),
                    mode=rng.choice([0, 2]), past=_log(rng, 1, 2000 // batch))
    t = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 200)])
    batch = rng.randint(1, 8)
    past = _log(rng, 8, 100000)
    while 2 * batch * kv * dh * past > 2 * 4 * 8 * 128 * 16000 or batch * heads * t * dh * past > 4 * 32 * 64 * 128 * 16000:
        past = past * 3 // 4
    return dict(kind=kind, batch=batch, t=t, heads=heads, kv=kv, dh=dh, past=past)


# ---------------------------------------------------------------------------
# MXFP4 in plain torch.  A block is 32 values of a row in 17 bytes: the biased
# exponent e of its scale 2^(e - 127), then 16 bytes, byte j holding value j in
# its low and value j + 16 in its high half.  A value is sign, 2 exponent bits
# and 1 mantissa bit.
# ---------------------------------------------------------------------------
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# Halfway points between levels; a value on one goes to the level with an even code.
MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def _quantize(x):
    """[rows, cols] f32 -> packed bytes [rows, cols / 32, 17]."""
    b = x.float().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(dim=2)
    # floor(log2 top) - 2 puts the largest value in [4, 8) before rounding.
    exponent = torch.frexp(top)[1] - 1 - 2
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127)).clamp(-127, 127)
    scaled = torch.ldexp(b.abs(), -exponent[:, :, None])
    code = torch.zeros(b.shape, device=b.device, dtype=torch.uint8)
    for i, mid in enumerate(MIDDLES):
        code += (scaled >= mid) if i % 2 else (scaled > mid)
    code += torch.signbit(b) * 8
    packed = torch.empty((*b.shape[:2], 17), device=b.device, dtype=torch.uint8)
    packed[:, :, 0] = (exponent + 127).to(torch.uint8)
    packed[:, :, 1:] = code[:, :, :16] + code[:, :, 16:] * 16
    return packed


def _dequantize(packed, dtype=torch.float32):
    """Packed bytes [rows, blocks, 17] -> [rows, 32 * blocks]."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=packed.device, dtype=dtype)
    code = torch.cat([packed[:, :, 1:] % 16, packed[:, :, 1:] // 16], dim=2)
    scale = torch.ldexp(torch.ones((), device=packed.device, dtype=dtype), packed[:, :, :1].to(torch.int32) - 127)
    return (levels[code.int()] * scale).reshape(packed.shape[0], -1)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
_BE = None


def _wamx():
    root = str(Path(__file__).resolve().parent.parent / "wam.cpp_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import wamx

    return wamx


def _backend():
    """The process's backend (a program opens one per GPU)."""
    global _BE
    if _BE is None:
        _BE = _wamx().Backend(0)
    return _BE


def _normal(g, shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)


def _pad(n, to):
    return (n + to - 1) // to * to


def _tree(rng, t):
    """Parents of t drafted tokens: several guesses per step, some steps deep."""
    wide = rng.choice([1, 2, 3, 4])
    return [-1 if i == 0 else rng.randint(max(-1, i - 1 - 2 * wide), i - 1) for i in range(t)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    c = dict(case)
    s = {"case": c}
    kind = c["kind"]
    if kind == "quantize":
        # Rows of different magnitude, as the rows of weights and activations are.
        size = torch.exp(_normal(g, (c["rows"], 1), 1.0, torch.float32))
        s["x"] = (_normal(g, (c["rows"], c["cols"]), 0.5, torch.float32) * size).to(DTYPE[c["x"]])
        s["packed"] = torch.empty((c["rows"], c["cols"] // 32, 17), device="cuda", dtype=torch.uint8)
        s["y"] = torch.empty((c["rows"], c["cols"]), device="cuda", dtype=DTYPE[c["x"]])
    elif kind == "product":
        s["w"] = _quantize(_normal(g, (c["m"], c["k"]), 0.02, torch.float32))
        s["x"] = _normal(g, (c["n"], c["k"]), 1.0, DTYPE[c["x"]])
        s["y"] = torch.empty((c["n"], c["m"]), device="cuda", dtype=DTYPE[c["y"]])
    else:
        b, t, heads, kv, dh = c["batch"], c["t"], c["heads"], c["kv"], c["dh"]
        # Ragged sequences: the longest has `past` cached tokens.
        past = [c["past"]] + [rng.randint(c["past"] // 2, c["past"]) for _ in range(b - 1)]
        s["past"] = torch.tensor(past, device="cuda", dtype=torch.int32)
        s["capacity"] = _pad(c["past"] + t, 64)
        s["k"] = _normal(g, (b, kv, s["capacity"], dh))
        s["vt"] = _normal(g, (b, kv, dh, s["capacity"]))
        if kind == "headnorm":
            s["x"] = _normal(g, (b * t, (heads + 2 * kv) * dh), 0.8)
            s["wq"] = (1 + _normal(g, (dh,), 0.1, torch.float32)).bfloat16()
            s["wk"] = (1 + _normal(g, (dh,), 0.1, torch.float32)).bfloat16()
            s["pos"] = (s["past"][:, None] + torch.arange(t, device="cuda", dtype=torch.int32)).reshape(-1).contiguous()
            s["q"] = torch.empty((b, heads, t, dh), device="cuda", dtype=torch.bfloat16)
        else:
            s["q"] = _normal(g, (b, heads, t, dh))
            s["parents"] = torch.tensor([_tree(rng, t) for _ in range(b)], device="cuda", dtype=torch.int32)
            s["out"] = torch.empty((b, t, heads * dh), device="cuda", dtype=torch.bfloat16)
    if own:
        _backend()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
BASE = 1000000.0


def _turn(x, pos, dims, mode, real):
    """The first `dims` of the last axis of x [b, h, t, dh] rotated by pos [b, t]; mode 0 pairs neighbours, 2 halves."""
    i = torch.arange(dims // 2, device=x.device, dtype=torch.float64)
    # Far positions times a frequency lose the angle in 32 bits.
    angle = pos.double()[:, None, :, None] * torch.exp(i * (-2.0 / dims * math.log(BASE)))
    cos, sin = torch.cos(angle).to(real), torch.sin(angle).to(real)
    y = x.clone()
    a, b = (slice(0, dims, 2), slice(1, dims, 2)) if mode == 0 else (slice(0, dims // 2), slice(dims // 2, dims))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _plain_headnorm(s):
    c = s["case"]
    b, t, heads, kv, dh = c["batch"], c["t"], c["heads"], c["kv"], c["dh"]
    x = s["x"].float().reshape(b, t, heads + 2 * kv, dh).transpose(1, 2)
    pos = s["pos"].reshape(b, t)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["wq"].float()
    k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["wk"].float()
    q, k = (_turn(y, pos, c["dims"], c["mode"], torch.float32) for y in (q, k))
    slot = (s["past"].long()[:, None] + torch.arange(t, device=x.device))[:, None, :, None].expand(b, kv, t, dh)
    s["k"].scatter_(2, slot, k.bfloat16())
    s["vt"].scatter_(3, slot.transpose(2, 3), v.transpose(2, 3).bfloat16())
    return q.bfloat16(), s["k"], s["vt"]


def _plain_tree(s):
    c = s["case"]
    b, t, heads, kv, dh = c["batch"], c["t"], c["heads"], c["kv"], c["dh"]
    dev = s["q"].device
    # seen[i][j]: token j is token i or one of its ancestors.
    token = torch.arange(t, device=dev)
    seen = (s["parents"][:, :, None] == token).float() + torch.eye(t, device=dev)
    for _ in range(max(1, (t - 1).bit_length())):
        seen = (seen @ seen > 0).float()
    key = torch.arange(s["capacity"], device=dev) - s["past"].long()[:, None]
    drafted = seen.gather(2, key.clamp(0, t - 1)[:, None, :].expand(b, t, -1)) > 0
    mask = (key < 0)[:, None, :] | (drafted & (key >= 0)[:, None, :] & (key < t)[:, None, :])
    out = []
    for i in range(b):
        q = s["q"][i].float().reshape(kv, heads // kv * t, dh)
        scores = (q @ s["k"][i].float().transpose(1, 2).contiguous()).reshape(kv, heads // kv, t, -1) / math.sqrt(dh)
        scores = scores.masked_fill(~mask[i], -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        v = s["vt"][i].float().transpose(1, 2).contiguous()
        o = (p.reshape(kv, heads // kv * t, -1) @ v).reshape(heads, t, dh) / p.sum(-1).reshape(heads, t, 1)
        out.append(o.transpose(0, 1).reshape(t, heads * dh))
    return torch.stack(out).bfloat16()


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        if kind == "quantize":
            return _dequantize(_quantize(s["x"])).to(s["x"].dtype)
        if kind == "product":
            # MUL_MAT's rule: the activations enter as bf16.
            return (s["x"].bfloat16().float() @ _dequantize(s["w"]).t()).to(s["y"].dtype)
        return _plain_headnorm(s) if kind == "headnorm" else _plain_tree(s)
    wamx, be = _wamx(), _backend()
    lib = be.lib
    if kind == "quantize":
        rows, cols, x = c["rows"], c["cols"], TYPE_ID[c["x"]]
        wamx.check(lib.wamx_op_quantize_mxfp4(be.ptr, s["x"].data_ptr(), x, cols, s["packed"].data_ptr(), rows, cols))
        wamx.check(lib.wamx_op_dequantize_mxfp4(be.ptr, s["packed"].data_ptr(), s["y"].data_ptr(), x, cols, rows, cols))
        return s["y"]
    if kind == "product":
        wamx.check(lib.wamx_op_mul_mat_mxfp4(be.ptr, s["w"].data_ptr(), s["x"].data_ptr(), TYPE_ID[c["x"]], c["k"],
                                             s["y"].data_ptr(), TYPE_ID[c["y"]], c["m"], c["m"], c["n"], c["k"]))
        return s["y"]
    b, t, heads, kv, dh = c["batch"], c["t"], c["heads"], c["kv"], c["dh"]
    if kind == "headnorm":
        wamx.check(lib.wamx_op_qkv_head_norm_rope(
            be.ptr, s["x"].data_ptr(), (heads + 2 * kv) * dh, s["wq"].data_ptr(), s["wk"].data_ptr(), s["pos"].data_ptr(),
            s["past"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["vt"].data_ptr(), heads, kv, dh, t, b,
            s["capacity"], s["capacity"], c["mode"], c["dims"], EPS, BASE))
        return s["q"], s["k"], s["vt"]
    wamx.check(lib.wamx_op_tree_attn(
        be.ptr, s["q"].data_ptr(), s["k"].data_ptr(), s["vt"].data_ptr(), s["parents"].data_ptr(), s["past"].data_ptr(),
        s["out"].data_ptr(), heads, kv, dh, t, b, s["capacity"], s["capacity"], 1.0 / math.sqrt(dh)))
    return s["out"]


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------
def _size(t):
    return {"f32": 4, "f16": 2, "bf16": 2}[t]


def work(case):
    c = case
    if c["kind"] == "quantize":
        n = c["rows"] * c["cols"]
        # Read, the packed form written, the values written.
        return {"bytes": n * (2 * _size(c["x"])) + n * 17 // 32, "flops": 4 * n}
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k * 17 // 32 + n * k * _size(c["x"]) + n * m * _size(c["y"]), "flops": 2 * m * n * k}
    b, t, heads, kv, dh = c["batch"], c["t"], c["heads"], c["kv"], c["dh"]
    if c["kind"] == "headnorm":
        values = b * t * (heads + 2 * kv) * dh
        return {"bytes": 4 * values + 4 * (dh + b * t + b), "flops": 10 * values}
    # The other sequences have three quarters of `past` on average.
    keys = c["past"] + (b - 1) * 3 * c["past"] // 4 + b * t
    return {"bytes": 4 * kv * dh * keys + 4 * b * t * heads * dh + 4 * b * (t + 1), "flops": 4 * heads * t * dh * keys}


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "quantize":
        x = s["x"].double().reshape(c["rows"], -1, 32)
        # The levels of a block are LEVELS times 2^(e - 2), 2^e the power of two at or below its largest value.
        top = x.abs().amax(2, keepdim=True)
        step = torch.exp2(torch.floor(torch.log2(top)).clamp(min=-125) - 2)
        step = torch.where(top > 0, step, torch.ones_like(step))
        a = x.abs() / step
        # Spacing 1/2 up to 2, 1 up to 4, 2 above; torch.round takes halves to even.
        grid = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
        v = torch.clamp(torch.round(a / grid) * grid, max=6.0)
        return (torch.sign(x) * v * step).reshape(c["rows"], -1)
    if c["kind"] == "product":
        bits = s["w"].to(torch.int64)
        half = torch.cat([bits[:, :, 1:] & 15, bits[:, :, 1:] >> 4], 2)
        e, f = (half >> 1) & 3, half & 1
        # Exponent 0 is the subnormal 1/2; else (1 + f/2) 2^(e - 1).
        mag = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2((e - 1).double()))
        w = torch.where(half >= 8, -mag, mag) * torch.exp2((bits[:, :, :1] - 127).double())
        return s["x"].bfloat16().double() @ w.reshape(c["m"], c["k"]).t()
    b, t, heads, kv, dh = c["batch"], c["t"], c["heads"], c["kv"], c["dh"]
    past = s["past"].tolist()
    if c["kind"] == "headnorm":
        x = s["x"].double().reshape(b, t, heads + 2 * kv, dh)
        k, vt, qs = s["k"].double(), s["vt"].double(), []
        freq = torch.tensor([BASE ** (-2.0 * i / c["dims"]) for i in range(c["dims"] // 2)], device="cuda", dtype=torch.float64)
        for i in range(b):
            h = x[i, :, :heads + kv]
            h = h / torch.sqrt((h ** 2).sum(2, keepdim=True) / dh + EPS)
            h = torch.cat([h[:, :heads] * s["wq"].double(), h[:, heads:] * s["wk"].double()], 1)
            z = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), s["pos"].reshape(b, t)[i].double()[:, None] * freq)
            turned, rest = h[:, :, :c["dims"]], h[:, :, c["dims"]:]
            if c["mode"] == 0:
                w = torch.view_as_complex(turned.reshape(t, heads + kv, -1, 2).contiguous()) * z[:, None]
                turned = torch.view_as_real(w).reshape(t, heads + kv, -1)
            else:
                w = torch.complex(*[p.contiguous() for p in turned.chunk(2, 2)]) * z[:, None]
                turned = torch.cat([w.real, w.imag], 2)
            h = torch.cat([turned, rest], 2)
            qs.append(h[:, :heads].transpose(0, 1))
            k[i, :, past[i]:past[i] + t] = h[:, heads:].transpose(0, 1)
            vt[i, :, :, past[i]:past[i] + t] = x[i, :, heads + kv:].permute(1, 2, 0)
        return torch.stack(qs), k, vt
    parents = s["parents"].tolist()
    rows = []
    for i in range(b):
        n = past[i]
        path = torch.zeros((t, t), dtype=torch.bool)
        for j in range(t):
            at = j
            while at >= 0:
                path[j, at] = True
                at = parents[i][at]
        hidden = torch.cat([torch.zeros((t, n), dtype=torch.bool), ~path], 1).cuda()
        heads_out = []
        for h in range(heads):
            kh = s["k"][i, h // (heads // kv), :n + t].double()
            vh = s["vt"][i, h // (heads // kv), :, :n + t].double()
            p = torch.softmax((s["q"][i, h].double() @ kh.t() / dh ** 0.5).masked_fill(hidden, -math.inf), 1)
            heads_out.append(p @ vh.t())
        rows.append(torch.cat(heads_out, 1))
    return torch.stack(rows)
