"""Timing cases of the residual-block operators that stand around a DeformConv2d: the block
norms (norm after the block, gate, residual scale, dropout, residual sum and the norm before
the next block, one operator), counter-based dropout and 8-bit pointwise products.

`own` false computes each operator in its plain form (elementary torch operations in 32
bits); `own` true makes the calls a user makes of torch_block. `exact` gives the outputs from
the definitions in 64 bits.

Definitions
  block norms   t = drop(alpha * scale[c] * act(gate) * N1(x)),  out = residual + t,
                y = N2(out), with N(v) = (v - m) * rsqrt(var + eps) * w[c] + b[c] over the
                channels of one position (RMS: m = 0, var = mean(v^2)).
  dropout       element i (or run of `group` elements) draws 16 bits u of
                Philox4x32-10(key = seed, counter = (i >> 3, offset)), half (i & 7); it is
                dropped (0) where u < T, T = floor(65536 p + 1/2), else v * 65536 / (65536 - T).
  8-bit product q = e4m3(v * 2^-e) in blocks of 128 along the contracted axis (weights:
                128 x 128), e the smallest integer with max|v| <= 448 * 2^e, at least -126;
                the product of the values that stand in q * 2^e.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _ops():
    pkg = os.path.abspath("jittor-dcn_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import torch_block
    return torch_block


# ---------------------------------------------------------------------------- cases
def listed():
    norm = dict(op="norm", layout="nchw", dtype="bf16", post="rms", pre="rms", gate="none",
                act="linear", p=0.0, train=True)
    drop = dict(op="dropout", dtype="bf16", p=0.1, group="element", residual=True, train=True)
    fp8 = dict(op="fp8", layout="rows", dtype="bf16", train=False)
    return [
        # one image's tokens between two blocks while serving: latency is what counts
        dict(norm, name="norm_serve_8_rows", layout="rows", b=1, c=1024, n=8, train=False),
        # training step at the bf16 map workload of the benchmark (64 images, 256 channels, 28x28)
        dict(norm, name="norm_train_map28_bf16", b=64, c=256, n=784, post="layer", pre="layer",
             gate="image", act="sigmoid", p=0.1),
        # fp32 maps of the headline workload (64 images, 256 channels, 56x56), forward only
        dict(norm, name="norm_infer_map56_f32", b=64, c=256, n=3136, dtype="f32", post="layer",
             pre="layer", train=False),
        # ragged token rows, full gate, odd channel count
        dict(norm, name="norm_train_rows_ragged", layout="rows", b=3, c=1001, n=2741,
             gate="full", act="silu"),
        # residual dropout of the same maps
        dict(drop, name="dropout_train_map28_bf16", b=64, c=256, n=784),
        # stochastic depth per image on the 512-channel 14x14 maps
        dict(drop, name="droppath_train_map14_f32", b=64, c=512, n=196, dtype="f32",
             group="image"),
        # channel dropout of one small odd map
        dict(drop, name="dropout2d_small_odd", b=2, c=33, n=49, dtype="f32", p=0.5,
             group="channel", residual=False),
        # one token through a served projection: the weight's bytes count
        dict(fp8, name="fp8_serve_one_token", b=1, n=1, c=4096, o=4096),
        # a batch of served maps through a 4x expansion
        dict(fp8, name="fp8_infer_map28", layout="nchw", b=64, n=784, c=256, o=1024),
        # odd sizes, training
        dict(fp8, name="fp8_train_ragged_f32", b=1, n=1777, c=1000, o=1500, dtype="f32",
             train=True),
        # a training step of a wide projection
        dict(fp8, name="fp8_train_wide", b=8, n=1024, c=2048, o=8192, train=True),
        # the largest product
        dict(fp8, name="fp8_infer_large", b=16, n=1024, c=8192, o=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "fp8", "fp8"])
    dtype, layout = rng.choice(["bf16", "bf16", "f32"]), rng.choice(["nchw", "rows"])
    train = rng.random() < 0.6
    if op == "fp8":
        c, o = _log(rng, 16, 8192), _log(rng, 16, 8192)
        if layout == "nchw":
            c, o = min(c, 2048), min(o, 4096)
            b, n = _log(rng, 1, 64), _log(rng, 16, 3136)
        else:
            b, n = 1, _log(rng, 1, 16384)
        while b * n * max(c, o) > 1 << 27 and n > 1:  # inputs and outputs of the largest listed
            n //= 2
        return dict(op=op, layout=layout, dtype=dtype, train=train, b=b, n=n, c=c, o=o)
    c = _log(rng, 16, 8192 if layout == "rows" else 1024)
    b, n = _log(rng, 1, 64), _log(rng, 1, 3136)
    while b * c * n > 64 * 256 * 784 and n > 1:
        n //= 2
    while b * c * n > 64 * 256 * 784:
        b = max(1, b // 2)
    if op == "dropout":
        return dict(op=op, dtype=dtype, train=train, b=b, c=c, n=n, p=rng.choice([0.1, 0.25, 0.5]),
                    group=rng.choice(["element", "element", "channel", "image"]),
                    residual=rng.random() < 0.5)
    return dict(op=op, layout=layout, dtype=dtype, train=train, b=b, c=c, n=n,
                post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["rms", "layer"]),
                gate=rng.choice(["none", "full", "image"]),
                act=rng.choice(["linear", "sigmoid", "silu"]), p=rng.choice([0.0, 0.0, 0.1]))


# ---------------------------------------------------------------------------- inputs
def _shape(case):
    b, c, n = case["b"], case["c"], case["n"]
    return (b, c, n, 1) if case.get("layout") == "nchw" or case["op"] == "dropout" else (b, n, c)


def prepare(case, seed):
    dev, dt = _dev(), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=dev).normal_(mean, std, generator=g)

    st = {"case": case, "rng": (0x5DEECE66D * 977 + seed, 16 * (seed % 1000003))}
    b, c, n, train = case["b"], case["c"], case["n"], case["train"]
    shape = _shape(case)
    if case["op"] == "norm":
        st["x"] = normal(*shape, std=0.7).to(dt)
        st["residual"] = normal(*shape, std=2.0, mean=0.1).to(dt)
        if case["gate"] == "full":
            st["gate"] = normal(*shape).to(dt)
        elif case["gate"] == "image":
            st["gate"] = normal(b, c).to(dt)
        st["scale"] = normal(c, std=0.1, mean=0.5).to(dt)
        for k in ("post", "pre"):
            if case[k] != "none":
                st["w_" + k] = normal(c, std=0.1, mean=1.0).to(dt)
            if case[k] == "layer":
                st["b_" + k] = normal(c, std=0.1).to(dt)
        if train:
            st["grad_out"], st["grad_y"] = normal(*shape).to(dt), normal(*shape).to(dt)
        leaves = ("x", "residual", "gate", "scale", "w_post", "b_post", "w_pre", "b_pre")
    elif case["op"] == "dropout":
        st["x"] = normal(*shape).to(dt)
        if case["residual"]:
            st["residual"] = normal(*shape).to(dt)
        if train:
            st["grad_y"] = normal(*shape).to(dt)
        leaves = ("x",)
    else:
        # activations with a few loud channels, as after a nonlinearity
        loud = torch.exp(normal(c, std=0.7))
        st["x"] = (normal(*shape) * (loud[:, None, None] if len(shape) == 4 else loud)).to(dt)
        w = normal(case["o"], c, std=c ** -0.5)
        if train:
            st["w"] = w.to(dt)
            gs = (b, case["o"], n, 1) if len(shape) == 4 else (b, n, case["o"])
            st["grad_y"] = normal(*gs, std=0.01).to(dt)
        else:
            # a served weight is kept in 8 bits: bytes [o][c up to 128s], exponents
            # [c / 128][o / 128] with a bias of 127
            q, e = _quant(torch.nn.functional.pad(w, (0, -c % 128, 0, -case["o"] % 128)), 128)
            st["w8"] = q[:case["o"]].to(torch.float8_e4m3fn).view(torch.uint8)
            st["w8_exp"] = (e.t() + 127).to(torch.uint8).contiguous()
        leaves = ("x", "w")
    st["leaves"] = [k for k in leaves if k in st]
    if own and train:
        for k in st["leaves"]:
            st[k].requires_grad_()
    if own and "w8" in st:
        st["weight"] = _ops().Fp8Weight(st["w8"], st["w8_exp"], c)
    return st


# ---------------------------------------------------------------------------- plain forms
def _philox(n, key, offset, dev):
    """16-bit draws of elements 0 .. n-1 (n up to a multiple of 8), int64 arithmetic mod 2^64."""
    m32 = 0xFFFFFFFF
    i = torch.arange((n + 7) // 8, device=dev, dtype=torch.int64)
    x0, x1 = i & m32, i >> 32
    x2, x3 = torch.full_like(i, offset & m32), torch.full_like(i, (offset >> 32) & m32)
    k0, k1 = key & m32, (key >> 32) & m32
    for _ in range(10):
        p0, p1 = x0 * 0xD2511F53, x2 * 0xCD9E8D57
        x0, x1, x2, x3 = (((p1 >> 32) & m32) ^ x1 ^ k0, p1 & m32,
                          ((p0 >> 32) & m32) ^ x3 ^ k1, p0 & m32)
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    w = torch.stack([x0, x1, x2, x3], 1)
    return torch.stack([w & 0xFFFF, w >> 16], 2).reshape(-1)[:n]


def _drop_factor(numel, group, p, rng, dev):
    """0 or 1 / (1 - T / 65536) for every element, in memory order."""
    t = int(math.floor(p * 65536 + 0.5))
    u = _philox(-(-numel // group), rng[0], rng[1], dev)
    f = torch.where(u < t, 0.0, 65536.0 / (65536 - t) if t < 65536 else 0.0)
    return f if group == 1 else f.repeat_interleave(group)[:numel]


def _act(g, act):
    """act(g) and its derivative."""
    if act == "linear":
        return g, torch.ones_like(g)
    s = 1 / (1 + torch.exp(-g))
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def _norm(v, kind, w, b, eps=EPS):
    """N(v) over the last axis, its normalised values and its scale."""
    m = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    d = v - m
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    h = d * r
    y = h * w
    return (y + b if b is not None else y), h, r


def _norm_grad(g, kind, w, h, r):
    """Gradients of N at v, w and b."""
    a = g * w
    d = a - h * (a * h).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - a.mean(-1, keepdim=True)
    return r * d, (g * h).reshape(-1, h.shape[-1]).sum(0), g.reshape(-1, h.shape[-1]).sum(0)


def _plain_norm(st):
    case, dt = st["case"], st["x"].dtype
    b, c, n = case["b"], case["c"], case["n"]
    maps = case["layout"] == "nchw"
    last = lambda t: t.float().reshape(b, c, n).transpose(1, 2) if maps else t.float()
    back = lambda t: (t.transpose(1, 2).reshape(b, c, n, 1) if maps else t).to(dt).contiguous()
    x, res = last(st["x"]), last(st["residual"])
    vec = {k: st[k].float() for k in ("scale", "w_post", "b_post", "w_pre", "b_pre") if k in st}
    if case["post"] != "none":
        v, h1, r1 = _norm(x, case["post"], vec["w_post"], vec.get("b_post"))
    else:
        v = x
    ga, gd = 1.0, None
    if case["gate"] != "none":
        gate = st["gate"].float()[:, None, :] if case["gate"] == "image" else last(st["gate"])
        ga, gd = _act(gate, case["act"])
    f = 1.0
    if case["p"] > 0:
        f = last(_drop_factor(b * c * n, 1, case["p"], st["rng"], x.device).reshape(_shape(case)))
    out = res + v * ga * vec["scale"] * f
    y, h2, r2 = _norm(out, case["pre"], vec["w_pre"], vec.get("b_pre"))
    got = {"out": back(out), "y": back(y)}
    if not case["train"]:
        return got
    gr, gw, gb = _norm_grad(last(st["grad_y"]), case["pre"], vec["w_pre"], h2, r2)
    gr = gr + last(st["grad_out"])
    got["grad_residual"] = back(gr)
    got["grad_w_pre"] = gw.to(dt)
    if "b_pre" in vec:
        got["grad_b_pre"] = gb.to(dt)
    gt = gr * f
    got["grad_scale"] = (gt * v * ga).reshape(-1, c).sum(0).to(dt)
    if gd is not None:
        gg = gt * v * vec["scale"]
        got["grad_gate"] = ((gg * gd).sum(1).to(dt) if case["gate"] == "image"
                            else back(gg * gd))
    gv = gt * ga * vec["scale"]
    if case["post"] != "none":
        gv, gw, gb = _norm_grad(gv, case["post"], vec["w_post"], h1, r1)
        got["grad_w_post"] = gw.to(dt)
        if "b_post" in vec:
            got["grad_b_post"] = gb.to(dt)
    got["grad_x"] = back(gv)
    return got


def _group(case):
    return {"element": 1, "channel": case["n"], "image": case["c"] * case["n"]}[case["group"]]


def _plain_dropout(st):
    case, x = st["case"], st["x"]
    f = _drop_factor(x.numel(), _group(case), case["p"], st["rng"], x.device).reshape(x.shape)
    y = x.float() * f
    if case["residual"]:
        y = y + st["residual"].float()
    got = {"y": y.to(x.dtype)}
    if case["train"]:
        got["grad_x"] = (st["grad_y"].float() * f).to(x.dtype)
    return got


def _quant(v, rows):
    """e4m3 values and exponents of v [R][K] (K a multiple of 128) in blocks of rows x 128."""
    r, k = v.shape
    blk = v.float().reshape(r // rows, rows, k // 128, 128)
    m, e = torch.frexp(blk.abs().amax((1, 3), keepdim=True))  # amax = m * 2^e, m in [1/2, 1)
    e = torch.where(m > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -126))
    e = e.clamp(min=-126)
    q = torch.ldexp(blk, -e).to(torch.float8_e4m3fn).float()
    return q.reshape(r, k), e.reshape(r // rows, k // 128)


def _quant_value(v, rows=1):
    """The values that v [R][K] stands for after the rounding, K of any length."""
    r, k = v.shape
    q, e = _quant(torch.nn.functional.pad(v.float(), (0, -k % 128, 0, -r % rows)), rows)
    s = e.repeat_interleave(rows, 0).repeat_interleave(128, 1)
    return torch.ldexp(q, s)[:r, :k]


def _plain_fp8(st):
    case, x = st["case"], st["x"]
    b, c, n, o, dt = case["b"], case["c"], case["n"], case["o"], x.dtype
    maps = case["layout"] == "nchw"
    rows = lambda t, k: (t.reshape(b, k, n).transpose(1, 2) if maps else t).reshape(b * n, k)
    back = lambda t, k: (t.reshape(b, n, k).transpose(1, 2).reshape(b, k, n, 1) if maps
                         else t.reshape(b, n, k)).to(dt).contiguous()
    xr = rows(x, c)
    if not case["train"]:
        e = (st["w8_exp"].to(torch.int32) - 127).t().repeat_interleave(128, 0)[:o]
        w = torch.ldexp(st["w8"].view(torch.float8_e4m3fn).float(), e.repeat_interleave(128, 1))
        return {"y": back(torch.matmul(_quant_value(xr), w[:, :c].t()), o)}
    wq = _quant_value(st["w"], 128)
    got = {"y": back(torch.matmul(_quant_value(xr), wq.t()), o)}
    gr = rows(st["grad_y"], o)
    got["grad_x"] = back(torch.matmul(_quant_value(gr), wq), c)

    def by_channel(t, k):
        # blocks of 128 positions; a map's blocks end with its image
        if not maps:
            return _quant_value(t.t().contiguous())
        t = t.reshape(b, n, k).transpose(1, 2).reshape(b * k, n)
        return _quant_value(t).reshape(b, k, n).transpose(0, 1).reshape(k, b * n)

    got["grad_w"] = torch.matmul(by_channel(gr, o), by_channel(xr, c).t()).to(dt)
    return got


# ---------------------------------------------------------------------------- one pass
def _own(st):
    tb, case = _ops(), st["case"]
    if case["op"] == "norm":
        def call():
            return tb.block_norm(
                st["x"], st["residual"], gate=st.get("gate"), gate_act=case["act"],
                scale=st["scale"], post=None if case["post"] == "none" else case["post"],
                post_weight=st.get("w_post"), post_bias=st.get("b_post"), pre=case["pre"],
                pre_weight=st["w_pre"], pre_bias=st.get("b_pre"), eps=EPS, drop_p=case["p"],
                rng=st["rng"])
        names = ("out", "y")
    elif case["op"] == "dropout":
        def call():
            return (tb.dropout(st["x"], case["p"], st["rng"], group=case["group"],
                               residual=st.get("residual")),)
        names = ("y",)
    else:
        def call():
            return (tb.fp8_pointwise(st["x"], st["w"] if case["train"] else st["weight"]),)
        names = ("y",)
    if not case["train"]:
        with torch.no_grad():
            return dict(zip(names, call()))
    outs = call()
    leaves = st["leaves"]
    grads = torch.autograd.grad(outs, [st[k] for k in leaves], [st["grad_" + k] for k in names])
    got = dict(zip(names, (t.detach() for t in outs)))
    got.update(("grad_" + k, t) for k, t in zip(leaves, grads))
    return got


def run(state):
    if own:
        got = _own(state)
    else:
        with torch.no_grad():
            got = {"norm": _plain_norm, "dropout": _plain_dropout,
                   "fp8": _plain_fp8}[state["case"]["op"]](state)
    return {k: got[k] for k in sorted(got)}


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    b, c, n, train = case["b"], case["c"], case["n"], case["train"]
    full = b * c * n
    if case["op"] == "norm":
        gate = {"none": 0, "full": full, "image": b * c}[case["gate"]]
        vecs = sum({"none": 0, "rms": c, "layer": 2 * c}[case[k]] for k in ("post", "pre")) + c
        elems = 4 * full + gate + vecs
        if train:  # reads x, residual, gate, two gradients; writes the gradients
            elems += 4 * full + gate + 2 * full + gate + 2 * vecs
        return {"bytes": elems * size, "flops": full * (60 if train else 20)}
    if case["op"] == "dropout":
        elems = full * (2 + case["residual"] + (2 if train else 0))
        return {"bytes": elems * size, "flops": full * (4 if train else 2)}
    o, t = case["o"], b * n
    if not train:
        return {"bytes": (t * c + t * o) * size + o * c, "flops": 2 * t * c * o}
    # x, w and the gradient read, the output and two gradients written
    return {"bytes": (2 * t * c + 2 * t * o + 2 * o * c) * size, "flops": 6 * t * c * o}


# ---------------------------------------------------------------------------- 64 bits
def _exact_u16(n, key, offset):
    """The 16-bit draws of elements 0 .. n-1 in numpy's unsigned 64-bit arithmetic."""
    u = np.uint64
    mask, sh = u(0xFFFFFFFF), u(32)
    i = np.arange(-(-n // 8), dtype=np.uint64)
    ctr = [i & mask, i >> sh, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    k = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, d = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(d >> sh) ^ ctr[1] ^ u(k[0]), d & mask, (a >> sh) ^ ctr[3] ^ u(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(ctr, 1).astype("<u4")
    return np.ascontiguousarray(words).view("<u2").reshape(-1)[:n].astype(np.int64)


def _exact_factor(case, st, group):
    numel = case["b"] * case["c"] * case["n"]
    t = int(math.floor(case["p"] * 65536 + 0.5))
    keep = _exact_u16(-(-numel // group), *st["rng"]) >= t
    f = np.where(keep, 65536.0 / (65536 - t) if t < 65536 else 0.0, 0.0)
    f = np.repeat(f, group)[:numel] if group > 1 else f
    return torch.from_numpy(f).to(_dev()).reshape(_shape(case))


def _exact_norm(case, st):
    ax = 1 if case["layout"] == "nchw" else 2
    names = st["leaves"]
    leaf = {k: st[k].detach().double().requires_grad_(case["train"]) for k in names}
    per_c = lambda v: v.reshape([-1 if i == ax else 1 for i in range(len(_shape(case)))])

    def normed(v, kind, w, b):
        if kind == "layer":
            v = v - v.mean(ax, keepdim=True)
        v = v * torch.rsqrt(v.square().mean(ax, keepdim=True) + EPS) * per_c(w)
        return v if b is None else v + per_c(b)

    t = leaf["x"]
    if case["post"] != "none":
        t = normed(t, case["post"], leaf["w_post"], leaf.get("b_post"))
    if case["gate"] != "none":
        g = leaf["gate"]
        if case["gate"] == "image":
            g = g[:, :, None, None] if ax == 1 else g[:, None, :]
        t = t * {"linear": lambda v: v, "sigmoid": torch.sigmoid,
                 "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](g)
    t = t * per_c(leaf["scale"])
    if case["p"] > 0:
        t = t * _exact_factor(case, st, 1)
    out = leaf["residual"] + t
    y = normed(out, case["pre"], leaf["w_pre"], leaf.get("b_pre"))
    got = {"out": out.detach(), "y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad((out, y), [leaf[k] for k in names],
                                    (st["grad_out"].double(), st["grad_y"].double()))
        got.update(("grad_" + k, g) for k, g in zip(names, grads))
    return got


def _exact_rounded(v, axis, both=False):
    """v (64 bits, 2-D) rounded to e4m3 in blocks of 128 along `axis` (both: 128 x 128)."""
    v = v.clone()
    step_r = 128 if both or axis == 0 else 1
    step_c = 128 if both or axis == 1 else 1
    r, c = v.shape
    pad = torch.zeros(-(-r // step_r) * step_r, -(-c // step_c) * step_c, dtype=v.dtype,
                      device=v.device)
    pad[:r, :c] = v
    blk = pad.reshape(pad.shape[0] // step_r, step_r, pad.shape[1] // step_c, step_c)
    top = blk.abs().amax((1, 3), keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -300) / 448.0))
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)      # log2's own rounding
    e = torch.where(top <= 224.0 * torch.exp2(e), e - 1, e).clamp(min=-126)
    s = blk * torch.exp2(-e)
    mag = torch.floor(torch.log2(s.abs().clamp(min=2.0 ** -60)))
    mag = torch.where(torch.exp2(mag) > s.abs(), mag - 1, mag).clamp(min=-6)
    ulp = torch.exp2(mag - 3)
    s = torch.round(s / ulp) * ulp * torch.exp2(e)
    return s.reshape(pad.shape)[:r, :c]


def _exact_fp8(case, st):
    b, c, n, o = case["b"], case["c"], case["n"], case["o"]
    maps = case["layout"] == "nchw"
    if (6 if case["train"] else 2) * b * n * c * o > 4e12:  # seconds in 64 bits
        return None

    def images(t, k):  # [b][n][k]
        t = t.detach().double()
        return t.reshape(b, k, n).transpose(1, 2) if maps else t.reshape(b, n, k)

    def whole(t):
        return t.transpose(1, 2).reshape(b, -1, n, 1) if maps else t

    x = images(st["x"], c)
    xt = _exact_rounded(x.reshape(b * n, c), 1)
    if not case["train"]:
        e = torch.exp2(st["w8_exp"].double() - 127).t()
        w = st["w8"].view(torch.float8_e4m3fn).double()
        w = (w * e.repeat_interleave(128, 0)[:o].repeat_interleave(128, 1))[:, :c]
        return {"y": whole((xt @ w.t()).reshape(b, n, o))}
    w = _exact_rounded(st["w"].detach().double(), 1, both=True)
    got = {"y": whole((xt @ w.t()).reshape(b, n, o))}
    g = images(st["grad_y"], o)
    got["grad_x"] = whole((_exact_rounded(g.reshape(b * n, o), 1) @ w).reshape(b, n, c))
    gw = torch.zeros(o, c, dtype=torch.float64, device=x.device)
    for i in range(b if maps else 1):  # a map's blocks end with its image
        gi = g[i] if maps else g.reshape(b * n, o)
        xi = x[i] if maps else x.reshape(b * n, c)
        gw += _exact_rounded(gi, 0).t().contiguous() @ _exact_rounded(xi, 0)
    got["grad_w"] = gw
    return got


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        got = _exact_norm(case, st)
    elif case["op"] == "dropout":
        f = _exact_factor(case, st, _group(case))
        y = st["x"].detach().double() * f
        got = {"y": y + st["residual"].double() if case["residual"] else y}
        if case["train"]:
            got["grad_x"] = st["grad_y"].double() * f
    else:
        got = _exact_fp8(case, st)
        if got is None:
            return None
    return {k: got[k].contiguous() for k in sorted(got)}
