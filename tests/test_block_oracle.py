"""CPU: the residual-block oracle (oracle/block_oracle.py) against published vectors and simple
restatements, and the refusals of the block entry points (their checks come before any device
call, so they run without a GPU)."""
import ctypes

import numpy as np
import pytest

import block_oracle as BO
import dcn_runtime as rt

OK_PTR = 1 << 20  # an aligned non-null address; refused calls never read it


@pytest.mark.parametrize("ctr,key,want", [
    # the published known answers of philox4x32 with 10 rounds
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((BO.M32,) * 4, (BO.M32,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_philox_known_answers(ctr, key, want):
    assert tuple(BO.philox4x32_10(ctr, key)) == want


@pytest.mark.parametrize("first", [0, 5, 8 * 2**32 - 3])
def test_draws_follow_the_scalar_generator(first):
    seed, off = 0x123456789ABCDEF0, 0xFEDCBA9876543210
    got = BO.draws(first, 21, seed, off)
    for j, u in enumerate(got):
        i = first + j
        w = BO.philox4x32_10(((i >> 3) & BO.M32, i >> 35, off & BO.M32, off >> 32),
                             (seed & BO.M32, seed >> 32))
        assert u == (w[(i & 7) >> 1] >> (16 * (i & 1))) & 0xFFFF


def _dropout(L, res=None, y=OK_PTR * 2, x=OK_PTR, rng=None, **kw):
    d = rt.DropoutDesc(**{**dict(n=64, group=1, dtype=rt.DCN_F32, p=0.5), **kw})
    return L.dcn_dropout_fwd(None, ctypes.byref(d), x, res, y, rng)


@pytest.mark.parametrize("kw,msg", [
    (dict(p=-0.1), "0 <= p <= 1"), (dict(p=1.5), "0 <= p <= 1"), (dict(p=float("nan")), "p <= 1"),
    (dict(n=-1), "element count"), (dict(group=0), "group"), (dict(dtype=2), "dtype"),
    (dict(x=None), "null tensor"), (dict(y=None), "null tensor"),
    (dict(x=OK_PTR + 2), "aligned"), (dict(rng=OK_PTR * 8 + 4), "8-byte"),
    (dict(y=OK_PTR + 16), "overlaps"), (dict(res=OK_PTR * 2 + 4), "overlaps"),
    (dict(rng=OK_PTR * 2 + 8), "overlaps"),
    (dict(), "null handle"),  # everything right but the handle
    (dict(y=OK_PTR), "null handle"), (dict(res=OK_PTR * 2), "null handle"),  # in place
])
def test_dropout_refusals(kw, msg):
    L = rt.load()
    assert _dropout(L, **kw) == -1
    assert msg in rt.last_error()


def test_null_descriptor():
    L = rt.load()
    assert L.dcn_dropout_fwd(None, None, OK_PTR, None, OK_PTR * 2, None) == -1


def test_drop_factor_mean():
    """The kept share of 2^20 draws is within 5 standard deviations of 1 - p, and the factor's
    mean within the same of 1."""
    n, p = 1 << 20, 0.1
    f = BO.drop_factor(n, 1, p, 7, 3)
    sd = (p * (1 - p) / n) ** 0.5
    assert abs(np.mean(f > 0) - (1 - p)) < 5 * sd + 1 / 65536
    assert abs(f.mean() - 1) < 5 * sd / (1 - p)


# ---- block norms
def _block(L, io=None, fwd=True, ws=OK_PTR * 64, ws_bytes=1 << 30, **kw):
    d = rt.BlockDesc(**{**dict(B=2, C=8, P=6, layout=0, dtype=0, post=1, pre=1, gate=0,
                               gate_act=0, eps_post=1e-6, eps_pre=1e-6, alpha=1.0, drop_p=0.0),
                        **kw})
    t = {n: OK_PTR * (i + 1) for i, n in enumerate(
        ("x", "residual", "out", "y") if fwd else ("x", "residual", "grad_out", "grad_y",
                                                   "grad_x", "grad_residual"))}
    t.update(io or {})
    t = rt.BlockIO(**t)
    if fwd:
        return L.dcn_block_norm_fwd(None, ctypes.byref(d), ctypes.byref(t))
    return L.dcn_block_norm_bwd(None, ctypes.byref(d), ctypes.byref(t), ws, ws_bytes)


FAR = OK_PTR * 100


@pytest.mark.parametrize("kw,io,msg", [
    (dict(B=0), {}, "positive"), (dict(C=-1), {}, "positive"), (dict(P=0), {}, "positive"),
    (dict(dtype=3), {}, "dtype"), (dict(layout=2), {}, "layout"), (dict(post=3), {}, "norm"),
    (dict(pre=-1), {}, "norm"), (dict(gate=4), {}, "gate kind"), (dict(gate_act=3), {}, "activ"),
    (dict(eps_pre=-1.0), {}, "eps"), (dict(eps_post=float("nan")), {}, "eps"),
    (dict(eps_post=float("inf")), {}, "eps"), (dict(drop_p=2.0), {}, "p <= 1"),
    (dict(drop_image=2), {}, "drop_image"), (dict(gate=1), {}, "come together"),
    (dict(), dict(gate=FAR), "come together"), (dict(), dict(x=None, residual=None), "neither"),
    (dict(), dict(x=None, out=None), "need x"), (dict(post=0, pre=0), dict(x=None), "nothing"),
    (dict(post=0), dict(w_post=FAR), "without a post"), (dict(pre=0), dict(b_pre=FAR), "a pre"),
    (dict(pre=0), {}, "come together"), (dict(), dict(y=None), "come together"),
    (dict(post=0), dict(x=None), "no out"), (dict(pre=0), dict(y=None, out=None), "no output"),
    (dict(), dict(rng=FAR + 4), "8-byte"), (dict(), dict(x=OK_PTR + 2), "aligned"),
    (dict(), dict(out=OK_PTR + 64), "overlaps"), (dict(), dict(out=OK_PTR), "overlaps"),
    (dict(), dict(y=OK_PTR * 2), "overlaps"), (dict(), dict(y=OK_PTR * 3 + 380), "two outputs"),
    (dict(), dict(w_pre=OK_PTR * 4), "overlaps"),
    (dict(B=1 << 20, C=1 << 20, P=2), {}, "2\\^40"), (dict(P=(1 << 30) + 1, C=1, B=1), {}, "2\\^30"),
    (dict(P=1, C=(1 << 23) + 1, B=1), {}, "2\\^23"),
    (dict(gate=2, P=6), dict(gate=OK_PTR * 2, out=OK_PTR * 2), "overlaps"),
    (dict(gate=1), dict(gate=OK_PTR * 2, out=OK_PTR * 2), "null handle"),
    (dict(), {}, "null handle"), (dict(), dict(out=OK_PTR * 2), "null handle"),
    (dict(post=0), dict(x=None, out=None), "null handle"),
])
def test_block_norm_forward_refusals(kw, io, msg):
    assert _block(rt.load(), io, **kw) < 0
    import re
    assert re.search(msg, rt.last_error()), rt.last_error()


@pytest.mark.parametrize("kw,io,ws,msg", [
    (dict(), dict(grad_out=None, grad_y=None), {}, "neither"),
    (dict(pre=0), {}, {}, "without a pre"), (dict(), dict(grad_gate=FAR), {}, "without a gate"),
    (dict(post=0), dict(grad_w_post=FAR), {}, "without a post"),
    (dict(pre=0), dict(grad_y=None, grad_b_pre=FAR), {}, "without a pre"),
    (dict(), dict(grad_x=None, grad_residual=None), {}, "no gradient"),
    (dict(post=0), dict(x=None, grad_x=None), {}, "without x"),
    (dict(), {}, dict(ws=None), "workspace"), (dict(), {}, dict(ws_bytes=16), "workspace"),
    (dict(), {}, dict(ws=OK_PTR * 64 + 8), "256-byte"),
    (dict(), dict(grad_x=OK_PTR * 3), {}, "overlaps"),
    (dict(), dict(grad_x=OK_PTR * 6), {}, "two outputs"),
    (dict(), {}, dict(ws=OK_PTR), "overlaps"), (dict(), {}, {}, "null handle"),
])
def test_block_norm_backward_refusals(kw, io, ws, msg):
    assert _block(rt.load(), io, fwd=False, **ws, **kw) < 0
    assert msg in rt.last_error()


@pytest.mark.parametrize("post,pre,gate", [("layer", "layer", 3), ("rms", "layer", 2),
                                           (None, "rms", 3), ("layer", None, 0)])
def test_block_oracle_gradients_against_differences(post, pre, gate):
    """The oracle's autograd gradients against central differences (float64 gradcheck)."""
    import torch
    g = torch.Generator().manual_seed(1)
    B, P, C = 2, 3, 5
    t = {"x": torch.randn(B, P, C, generator=g, dtype=torch.float64),
         "residual": torch.randn(B, P, C, generator=g, dtype=torch.float64),
         "scale": torch.rand(C, generator=g, dtype=torch.float64) + 0.5}
    if gate:
        t["gate"] = torch.randn(*((B, P, C) if gate == 3 else (B, C)), generator=g,
                                dtype=torch.float64)
    for k, on in (("w_post", post), ("b_post", post == "layer"), ("w_pre", pre),
                  ("b_pre", pre == "layer")):
        if on:
            t[k] = torch.randn(C, generator=g, dtype=torch.float64)
    f = torch.from_numpy(BO.drop_factor(B * P * C, 1, 0.3, 1, 2)).reshape(B, P, C)
    names = list(t)

    def fn(*v):
        o, y = BO.block_forward(dict(zip(names, v)), post=post, pre=pre, act="silu", factor=f)
        return (o, y) if pre else o

    assert torch.autograd.gradcheck(fn, [t[k].requires_grad_() for k in names])


# ---- 8-bit products
def test_fp8_rounding_is_the_nearest():
    """fp8_round picks, for each value, a nearest multiple the byte format holds."""
    g = np.random.default_rng(3)
    v = g.standard_normal((4, 256)) * np.exp2(g.integers(-12, 9, (4, 256)))
    v[0, :128] = 0
    q, e = BO.fp8_round(v, 1, 128)
    grid = np.unique(BO.e4m3_decode(np.arange(256))[~np.isnan(BO.e4m3_decode(np.arange(256)))])
    s = np.ldexp(v, -np.repeat(e, 128, 1))
    assert np.isin(q, grid).all() and np.abs(s).max() <= 448
    assert np.array_equal(np.abs(s - q), np.abs(s[..., None] - grid).min(-1))
    assert e[0, 0] == -126 and all(448 * 2.0 ** (e[i, 1] - 1) < np.abs(v[i, 128:]).max()
                                   for i in range(4))


A = OK_PTR


@pytest.mark.parametrize("kw,ptr,msg", [
    (dict(B=0), {}, "positive"), (dict(dtype=5), {}, "dtype"), (dict(layout=3), {}, "layout"),
    (dict(), dict(s_tok=None), "come together"), (dict(), dict(q_ch=A * 9), "come together"),
    (dict(), dict(q_tok=A * 2 + 8), "16-byte"), (dict(), dict(s_tok=A * 3 + 2), "4-byte"),
    (dict(), dict(q_tok=None, s_tok=None), "null tensor"), (dict(), dict(v=None), "null tensor"),
    (dict(), dict(v=A + 2), "aligned"), (dict(), dict(q_tok=A + 16), "overlaps"),
    (dict(), dict(s_tok=A * 2), "two outputs"), (dict(B=1 << 20, P=1 << 20), {}, "too large"),
    (dict(), {}, "null handle"),
])
def test_fp8_quantize_refusals(kw, ptr, msg):
    d = rt.Fp8Desc(**{**dict(B=2, C=8, P=6, layout=0, dtype=0), **kw})
    p = {**dict(v=A, q_tok=A * 2, s_tok=A * 3, q_ch=None, s_ch=None), **ptr}
    assert rt.load().dcn_fp8_quantize(None, ctypes.byref(d), *p.values()) < 0
    assert msg in rt.last_error()


@pytest.mark.parametrize("kw,msg", [
    (dict(O=0), "positive"), (dict(C=-3), "positive"), (dict(dtype=2), "dtype"),
    (dict(w=None), "null tensor"), (dict(q=None, s=None), "null tensor"),
    (dict(s=None), "come together"), (dict(qT=A * 5), "come together"),
    (dict(q=A + 64), "overlaps"), (dict(w=A + 1), "aligned"), (dict(O=1 << 30, C=1 << 30), "large"),
    (dict(), "null handle"),
])
def test_fp8_quantize_weight_refusals(kw, msg):
    p = {**dict(O=20, C=30, dtype=0, w=A, q=A * 2, s=A * 3, qT=None, sT=None), **kw}
    assert rt.load().dcn_fp8_quantize_weight(None, *p.values()) < 0
    assert msg in rt.last_error()


@pytest.mark.parametrize("kw,ptr,msg", [
    (dict(M=0), {}, "positive"), (dict(K=-128), {}, "positive"), (dict(K=100), {}, "multiple of 128"),
    (dict(a_block=64), {}, "1 or 128"), (dict(b_block=0), {}, "1 or 128"),
    (dict(layout=2), {}, "layout"), (dict(layout=0, P=0), {}, "multiple of P"),
    (dict(layout=0, P=7), {}, "multiple of P"), (dict(out_dtype=9), {}, "dtype"),
    (dict(M=1 << 26, N=1 << 26), {}, "2^24 tiles"), (dict(M=(1 << 26) + 1, N=1), {}, "2^26"),
    (dict(), dict(a=None), "null tensor"), (dict(), dict(sb=None), "come together"),
    (dict(), dict(b=A * 3 + 4), "16-byte"), (dict(), dict(sa=A * 2 + 1), "4-byte"),
    (dict(), dict(out=A * 5 + 2), "aligned"), (dict(), dict(out=A * 3), "overlaps"),
    (dict(), dict(ws=A * 6 + 16), "256-byte"), (dict(), {}, "null handle"),
])
def test_fp8_matmul_refusals(kw, ptr, msg):
    d = rt.Fp8MatmulDesc(**{**dict(M=16, N=24, K=256, a_block=1, b_block=128, layout=1, P=0,
                                   out_dtype=0), **kw})
    p = {**dict(a=A, sa=A * 2, b=A * 3, sb=A * 4, out=A * 5, ws=None, n=0), **ptr}
    assert rt.load().dcn_fp8_matmul(None, ctypes.byref(d), *p.values()) < 0
    assert msg in rt.last_error()


def _pointwise(L, fwd, **kw):
    d = rt.Fp8PointwiseDesc(**{**dict(B=2, C=20, P=6, O=30, layout=0, dtype=0),
                               **{k: kw.pop(k) for k in list(kw) if k in "BCPO" or k in ("layout", "dtype")}})
    if fwd:
        p = {**dict(grads=0, x=A, w=A * 2, q=None, s=None, y=A * 3, saved=None, ns=0, ws=A * 4,
                    n=1 << 19), **kw}
        return L.dcn_fp8_pointwise_fwd(None, ctypes.byref(d), *p.values())
    p = {**dict(grads=3, gy=A, saved=A * 2, ns=1 << 19, gx=A * 3, gw=A * 4, ws=A * 5, n=1 << 19), **kw}
    return L.dcn_fp8_pointwise_bwd(None, ctypes.byref(d), *p.values())


@pytest.mark.parametrize("fwd,kw,msg", [
    (1, dict(O=0), "positive"), (1, dict(dtype=4), "dtype"), (1, dict(layout=5), "layout"),
    (1, dict(grads=4), "unknown gradient"), (1, dict(x=None), "null tensor"),
    (1, dict(w=None), "null tensor"), (1, dict(q=A * 7, s=A * 8), "one weight"),
    (1, dict(w=None, q=A * 7), "come together"),
    (1, dict(w=None, q=A * 7, s=A * 8, grads=1), "no gradients"),
    (1, dict(n=100), "too small"), (1, dict(ws=A * 4 + 16), "256-byte"),
    (1, dict(grads=1), "saved buffer too small"), (1, dict(y=A + 64), "overlaps"),
    (1, dict(y=A * 3 + 2), "aligned"), (1, dict(ws=A * 3), "two outputs"),
    (1, dict(B=1 << 15, P=1 << 16), "too large"), (1, {}, "null handle"),
    (1, dict(w=None, q=A * 7, s=A * 8), "null handle"),
    (1, dict(grads=8), "one weight"), (1, dict(grads=9, w=None, q=A * 7, s=A * 8), "unknown"),
    (1, dict(grads=8, w=None, q=A * 7, s=A * 8, n=100), "too small"),
    (1, dict(grads=8, w=None, q=A * 7, s=A * 8), "null handle"),
    (1, dict(grads=8, w=None, q=A * 7, s=A * 8, layout=1, ws=None, n=0), "null handle"),
    (0, dict(grads=8), "kept nothing"),
    (1, dict(grads=3, saved=A * 9, ns=1 << 19), "null handle"),
    (0, dict(gx=None, gw=None), "null tensor"), (0, dict(gy=None), "null tensor"),
    (0, dict(grads=1), "kept nothing"), (0, dict(ns=4), "saved buffer too small"),
    (0, dict(n=4), "too small"), (0, dict(gx=A), "overlaps"), (0, dict(gw=A * 3), "two outputs"),
    (0, dict(gx=A * 3 + 1), "aligned"), (0, {}, "null handle"), (0, dict(gx=None), "null handle"),
])
def test_fp8_pointwise_refusals(fwd, kw, msg):
    assert _pointwise(rt.load(), fwd, **dict(kw)) < 0
    assert msg in rt.last_error()
