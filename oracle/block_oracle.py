"""64-bit restatements of the residual-block operators (include/dcn.h), for the tests only:
Philox4x32-10 draws, dropout, block norms with their gradients by torch's float64 autograd,
and 8-bit block rounding. Written from the definitions, on the CPU."""
from __future__ import annotations

import numpy as np
import torch

M32 = 0xFFFFFFFF


def philox4x32_10(ctr, key):
    """Four words of Philox4x32-10 for one counter (4 words) and key (2 words), Python ints."""
    x, k = list(ctr), list(key)
    for _ in range(10):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(p1 >> 32) ^ x[1] ^ k[0], p1 & M32, (p0 >> 32) ^ x[3] ^ k[1], p0 & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return x


def draws(first, n, seed, offset):
    """The 16-bit draws of elements first .. first + n - 1."""
    b0 = first >> 3
    i = np.arange(b0, (first + n + 7) // 8, dtype=np.uint64)
    m, s = np.uint64(M32), np.uint64(32)
    x = [i & m, i >> s, np.full_like(i, offset & M32), np.full_like(i, (offset >> 32) & M32)]
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(p1 >> s) ^ x[1] ^ np.uint64(k0), p1 & m, (p0 >> s) ^ x[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    u = np.stack([h for w in x for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    return u.reshape(-1)[first - 8 * b0:][:n].astype(np.int64)


def drop_factor(n, group, p, seed, offset):
    """0 or 65536 / (65536 - T) per element, float64."""
    t = int(np.floor(p * 65536 + 0.5))
    nd = -(-n // group)
    f = np.where(draws(0, nd, seed, offset) < t, 0.0, 65536.0 / max(65536 - t, 1))
    return np.repeat(f, group)[:n]


# ---- block norms ---------------------------------------------------------------------------
ACTS = {"linear": lambda g: g, "sigmoid": torch.sigmoid, "silu": lambda g: g * torch.sigmoid(g)}


def norm(v, kind, w, b, eps):
    """N over the last axis, any float dtype."""
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    h = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    h = h if w is None else h * w
    return h if b is None else h + b


def block_forward(t, *, post=None, pre=None, act="linear", alpha=1.0, eps=1e-6, factor=None):
    """(out, y) of tensors t["x"], t["residual"], ... all [B][P][C] (gate [B][C] per image);
    factor: the dropout factor [B][P][C] or None. x absent: out is the residual."""
    if t.get("x") is None:
        return t["residual"], norm(t["residual"], pre, t.get("w_pre"), t.get("b_pre"), eps)
    v = norm(t["x"], post, t.get("w_post"), t.get("b_post"), eps)
    if t.get("gate") is not None:
        g = t["gate"]
        v = v * ACTS[act](g[:, None] if g.dim() == 2 else g)
    if t.get("scale") is not None:
        v = v * t["scale"]
    v = v * alpha
    if factor is not None:
        v = torch.where(factor == 0, torch.zeros_like(v), v * factor)
    out = v if t.get("residual") is None else t["residual"] + v
    return out, norm(out, pre, t.get("w_pre"), t.get("b_pre"), eps) if pre else None


def block_bounds(t, go, gy, *, post=None, pre=None, act="linear", alpha=1.0, eps=1e-6,
                 factor=None):
    """For every output, the value of its formula with every term replaced by its magnitude
    (no cancellation): a result computed with sums of n fp32 terms is within a small multiple
    of n · 2^-24 of it. A norm's r amplifies by mean(d²) r² >= 1 where its mean cancels."""
    one = torch.ones((), dtype=torch.float64)
    a = {k: v.abs() for k, v in t.items() if v is not None}
    g = t.get("gate")

    def mag(m, v, kind, w, b):  # magnitudes of N's output and of its normalised value; r
        if kind is None:
            return m, None, one
        mean = m.mean(-1, keepdim=True) if kind == "layer" else 0.0
        c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
        r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        d = m + mean
        q = ((d * d).mean(-1, keepdim=True) * r * r).clamp(min=1.0)
        h = d * r * q
        return h * a.get(w, one) + a.get(b, torch.zeros(())), h, r * q

    def back(m, kind, w, h, r):
        m = m * a.get(w, one)
        mean = m.mean(-1, keepdim=True) if kind == "layer" else 0.0
        return r * (m + mean + h * (m * h).mean(-1, keepdim=True))

    out, _ = block_forward(t, post=post, pre=pre, act=act, alpha=alpha, eps=eps, factor=factor)
    f = one if factor is None else factor
    lead = tuple(range(out.dim() - 1))
    res = {}
    if t.get("x") is not None:
        mv, h1, r1 = mag(a["x"], t["x"], post, "w_post", "b_post")
        av = ad = one
        if g is not None:
            gg = g[:, None] if g.dim() == 2 else g
            s = torch.sigmoid(gg)
            av, ad = {"linear": (gg.abs(), one), "sigmoid": (s, s * (1 + s)),
                      "silu": (gg.abs() * s, s * (1 + gg.abs() * (1 + s)))}[act]
        ms = a.get("scale", one) * abs(alpha)
        mo = a.get("residual", torch.zeros(())) + mv * ms * av * f
    else:
        mo = a["residual"]
    res["out"] = mo
    mg = torch.zeros_like(out) if go is None else go.abs()
    if pre:
        res["y"], h2, r2 = mag(mo, out, pre, "w_pre", "b_pre")
        m = torch.zeros_like(out) if gy is None else gy.abs()
        mg = mg + back(m, pre, "w_pre", h2, r2)
        res["w_pre"], res["b_pre"] = (m * h2).sum(lead), m.sum(lead)
    res["residual"] = mg
    if t.get("x") is not None:
        md = mg * f
        res["scale"] = (md * mv * av).sum(lead) * abs(alpha)
        if g is not None:
            m = md * mv * ms * ad
            res["gate"] = m.sum(1) if g.dim() == 2 else m
        m = md * ms * av
        if post:
            res["w_post"], res["b_post"] = (m * h1).sum(lead), m.sum(lead)
            m = back(m, post, "w_post", h1, r1)
        res["x"] = m
    return res


# ---- 8-bit blocks --------------------------------------------------------------------------
def fp8_round(v, rows, cols):
    """(bytes' values, exponents) of v [R][C] (float64, dims multiples of rows / cols) in blocks of
    rows x cols: exponent e = the smallest integer >= -126 with max|v| <= 448 * 2^e over the
    finite values, value = e4m3(v * 2^-e) by round-half-even on a grid of 2^(x - 3), x the
    value's exponent, at least -6; non-finite values become NaN."""
    v = np.asarray(v, np.float64)
    R, C = v.shape
    blk = v.reshape(R // rows, rows, C // cols, cols)
    mag = np.where(np.isfinite(blk), np.abs(blk), 0.0).max((1, 3), keepdims=True)
    m, x = np.frexp(mag)  # mag = m * 2^x
    e = np.where(mag > 0, x - 9 + (m > 0.875), -126)
    e = np.maximum(e, -126)
    with np.errstate(invalid="ignore"):
        s = np.ldexp(blk, -e)
        _, x = np.frexp(s)
        step = np.ldexp(1.0, np.maximum(x - 1, -6) - 3)
        q = np.rint(s / step) * step
    q = np.where(np.isfinite(blk), q, np.nan)
    return q.reshape(R, C), e[:, 0, :, 0]


def fp8_value(v, rows, cols):
    """The values that v [R][C] (any size) stands for after the rounding."""
    v = np.asarray(v, np.float64)
    R, C = v.shape
    p = np.zeros((-(-R // rows) * rows, -(-C // cols) * cols))
    p[:R, :C] = v
    q, e = fp8_round(p, rows, cols)
    return np.ldexp(q, np.repeat(np.repeat(e, rows, 0), cols, 1))[:R, :C]


def e4m3_decode(b):
    """Values of OCP e4m3 bytes."""
    b = np.asarray(b, np.uint8).astype(np.int64)
    s, x, m = b >> 7, (b >> 3) & 15, b & 7
    v = np.where(x == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (x - 10.0))
    v = np.where((x == 15) & (m == 7), np.nan, v)
    return np.where(s == 1, -v, v)
