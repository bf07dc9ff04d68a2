"""GPU: block norms where an argument is absent, a value is not finite or a channel count leaves
a vector half filled, against the 64-bit oracle with the bounds of test_gpu_block_norm.py."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import block_oracle as BO  # noqa: E402
import test_gpu_block_norm as N  # noqa: E402

U, SEED, OFF = N.U, N.SEED, N.OFF
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def tb():
    import torch_block
    return torch_block


NEUTRAL = {"scale": 1.0, "w_post": 1.0, "b_post": 0.0, "w_pre": 1.0, "b_pre": 0.0}


def absent_equals_neutral(tb, layout, B, C, P, dt, post, pre, gate, act, keep=(), p=0.0):
    """A call without the parameters that are not in `keep` gives the bits, results and gradients,
    of one with ones for scale and weights and zeros for biases (which other tests hold against
    the oracle)."""
    t, go, gy = N.tensors(layout, B, C, P, dt, post, pre, gate, shift=3.0, seed=C)
    got = []
    for absent in (True, False):
        u = {}
        for k, v in t.items():
            if k not in NEUTRAL or k in keep:
                u[k] = v.clone()
            elif not absent:
                u[k] = torch.full_like(v, NEUTRAL[k])
        for v in u.values():
            v.requires_grad_()
        out = N.call(tb, u, post, pre, act, p=p)
        out = [(v, g) for v, g in zip(out, (go, gy)) if v is not None]
        grads = torch.autograd.grad([v for v, _ in out], list(u.values()), [g for _, g in out])
        got.append({**dict(zip(u, grads)), **dict(zip(("out", "y"), (v for v, _ in out)))})
    for k, v in got[0].items():
        assert torch.equal(v, got[1][k]), k


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("post,pre", [("layer", "rms"), ("layer", "layer"), ("layer", None),
                                      ("rms", "layer"), ("rms", "rms"), (None, "layer")])
@pytest.mark.parametrize("gate,act", [("none", "linear"), ("image", "sigmoid"), ("full", "sigmoid")])
@pytest.mark.parametrize("keep", [(), ("scale",), ("w_post",), ("b_post",), ("w_pre", "b_pre")])
def test_absent_parameters(tb, dt, layout, post, pre, gate, act, keep):
    """50 channels, no whole number of vectors, and means that are not zero: a NULL weight is 1 for
    the channels there are and adds nothing past the last."""
    absent_equals_neutral(tb, layout, 3, 50, 13, dt, post, pre, gate, act, keep)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("C", [1, 3, 9, 33, 50, 100, 130, 257, 515, 1001, 2049, 4097, 8197, 16383,
                               16387])
@pytest.mark.parametrize("gate,p", [("none", 0.0), ("full", 0.0), ("image", 0.25)])
def test_absent_parameters_at_every_row_variant(tb, dt, C, gate, p):
    absent_equals_neutral(tb, "rows", 2, C, 3, dt, "layer", "layer", gate, "sigmoid", p=p)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("C", [3, 33, 65, 130, 257, 513, 1025, 2049])
def test_absent_parameters_at_every_map_variant(tb, dt, C):
    absent_equals_neutral(tb, "nchw", 2, C, 11, dt, "layer", "layer", "full", "sigmoid")
    absent_equals_neutral(tb, "nchw", 5, C, 1, dt, "layer", "rms", "none", "linear")


@pytest.mark.parametrize("dt", DTYPES)
def test_image_draws_of_flat_features(tb, dt):
    """drop="image" on [N, C] draws once per row, as DropPath does."""
    n, C = 40, 36
    t, go, gy = N.tensors("rows", n, C, 1, dt, "rms", "layer", "none")
    t = {k: v.reshape(n, C) if v.dim() == 3 else v for k, v in t.items()}
    f = torch.from_numpy(BO.drop_factor(n, 1, 0.5, SEED, OFF)).cuda()
    assert (f == 0).any() and (f > 0).any()
    out, y = N.call(tb, t, "rms", "layer", "linear", p=0.5, drop="image")
    assert torch.equal(out[f == 0], t["residual"][f == 0])
    kept = N.call(tb, t, "rms", "layer", "linear", alpha=2.0)  # (the factor of p = 1/2)
    assert torch.equal(out[f > 0], kept[0][f > 0]) and torch.equal(y[f > 0], kept[1][f > 0])
    d = tb.dropout(t["x"], 0.5, (SEED, OFF), group="image")
    assert torch.equal((d != 0).any(1), f > 0)
    g = torch.randn(1, C, device="cuda").to(dt).requires_grad_()
    u = {**t, "gate": g}
    o2, _ = N.call(tb, u, "rms", "layer", "silu", p=0.5, drop="image")
    gg, = torch.autograd.grad(o2, g, go.reshape(n, C))
    assert gg.shape == (1, C) and bool(torch.isfinite(gg).all())


@pytest.mark.parametrize("act", ["linear", "sigmoid", "silu"])
@pytest.mark.parametrize("p", [0.5, 1.0])
@pytest.mark.parametrize("layout,C", [("nchw", 48), ("nchw", 300), ("nchw", 2100), ("rows", 48),
                                      ("rows", 300), ("rows", 3000), ("rows", 8000),
                                      ("rows", 16500)])
def test_an_image_gate_of_dropped_elements(tb, layout, C, p, act):
    """A gate[b, c] whose elements are all dropped reaches nothing, NaN and infinities neither:
    the bits that 0 gives there, in the results and in every gradient."""
    B, P = 6, 3
    t, go, gy = N.tensors(layout, B, C, P, torch.float32, "layer", "layer", "image")
    f = torch.from_numpy(BO.drop_factor(B * C * P, 1, p, SEED, OFF))
    f = f.reshape(B, C, P).transpose(1, 2) if layout == "nchw" else f.reshape(B, P, C)
    gone = (f == 0).all(1).cuda()
    assert gone.any() and (p == 1.0 or not gone.all())
    results = []
    for bad in (0.0, float("nan"), float("inf"), float("-inf")):
        u = {k: v.clone() for k, v in t.items()}
        u["gate"][gone] = bad
        for v in u.values():
            v.requires_grad_()
        o, y = N.call(tb, u, "layer", "layer", act, p=p)
        results.append([o, y, *torch.autograd.grad((o, y), list(u.values()), (go, gy))])
    assert all(torch.isfinite(v).all() for v in results[0])
    for r in results[1:]:
        for k, a, b in zip(["out", "y", *t], results[0], r):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("layout,C", [("nchw", 16), ("nchw", 2064), ("rows", 16), ("rows", 16400)])
@pytest.mark.parametrize("gate", ["full", "image"])
def test_gate_values(tb, dt, act, layout, C, gate):
    """act(g) and act'(g) alone (x = 1, nothing else) over the whole range of g.

    With u = 2^-24: e = exp(-|g|) to 1 ulp (2 u) and 1 / (1 + e) to 2 u of a sum rounded once;
    sigmoid = e or 1 times that: 2 + 2 + 1 + 2 + 1 = 8 u of its value, 1 - sigmoid the same; silu
    one product more. sigmoid' = s (1 - s): 17 u. silu' = s (1 + g (1 - s)): 8 + 8 + 4 u of s (1 +
    |g| (1 - s)). Each product with x, the scale of 1 and the incoming gradient of 1 is exact.
    Results below 2^-126 are multiples of 2^-149, half of one off in each of up to four steps, the
    silu's multiplied by |g| <= 110 after the first. In bf16 e's argument is a rounded product with a
    rounded constant, 2 |g| u more in each of its two uses, the result has its half step, and what
    lies below 110 times the smallest normal may be 0."""
    n = C * 64
    g = torch.cat([torch.linspace(-110, 110, n // 2), torch.linspace(-9, 9, n - n // 2)])
    g = g[torch.randperm(n, generator=torch.Generator().manual_seed(1))]
    if gate == "image":
        B, P, gsh = 64, 1, (64, C)
    else:
        B, P, gsh = 1, 64, (1, C, 64, 1) if layout == "nchw" else (1, 64, C)
    shape = (B, C, P, 1) if layout == "nchw" else (B, P, C)
    x = torch.ones(shape, device="cuda", dtype=dt)
    g = g.reshape(gsh).to("cuda", dt).requires_grad_()
    out, _ = tb.block_norm(x, gate=g, gate_act=act)
    d, = torch.autograd.grad(out, g, torch.ones_like(out))
    G = g.detach().cpu().double()
    s, t = torch.sigmoid(G), torch.sigmoid(-G)
    bf = dt == torch.bfloat16
    more, half, tiny = (2 * G.abs(), 2.0 ** -8, 110 * 2.0 ** -126) if bf else (0, 0, 110 * 2.0 ** -147)
    want, slope = (s, s * t) if act == "sigmoid" else (G * s, s * (1 + G * t))
    mag = s * t if act == "sigmoid" else s * (1 + G.abs() * t)
    got = out.detach().cpu().double().reshape(G.shape)
    err = (got - want).abs() / (((9 + more) * U + half) * want.abs() + tiny)
    assert float(err.max()) <= 1, (float(err.max()), float(G.flatten()[err.argmax()]))
    err = (d.cpu().double() - slope).abs() / ((20 + 2 * more) * U * mag + half * slope.abs() + tiny)
    assert float(err.max()) <= 1, (float(err.max()), float(G.flatten()[err.argmax()]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("gate", ["none", "full", "image"])
@pytest.mark.parametrize("layout,B,C,P", [
    ("rows", 1, 4096, 1), ("rows", 3, 4096, 300), ("rows", 5, 24, 7), ("rows", 2, 300, 2000),
    ("rows", 1, 8192, 3), ("rows", 2, 6000, 700), ("rows", 2, 16384, 300), ("rows", 3, 16390, 5),
    ("nchw", 2, 64, 5), ("nchw", 3, 48, 113), ("nchw", 70, 16, 130), ("nchw", 2, 256, 4000),
    ("nchw", 3, 1500, 60), ("nchw", 2, 2050, 9), ("nchw", 9, 70, 1)])
def test_backward_stays_in_its_workspace(tb, dt, gate, layout, B, C, P):
    """With exactly dcn_block_norm_workspace bytes: what lies behind them stays, and the gradients are
    those of a workspace of any contents."""
    import ctypes

    import dcn_runtime as rt
    t, go, gy = N.tensors(layout, B, C, P, dt, "layer", "rms", gate, seed=P)
    kind = {"none": rt.DCN_GATE_NONE, "full": rt.DCN_GATE_FULL, "image": rt.DCN_GATE_IMAGE}[gate]
    d = rt.BlockDesc(B, C, P, rt.DCN_NCHW if layout == "nchw" else rt.DCN_NHWC, tb._DT[dt], 2, 1,
                     kind, rt.DCN_ACT_SILU, 1e-6, 1e-6, 1.0, 0.0, 0, 0, 0)
    n = ctypes.c_size_t()
    rt.check(rt.load().dcn_block_norm_workspace(d, n))
    behind, results = 1 << 22, []
    for fill in (0, 255):
        ws = torch.full((n.value + behind,), fill, dtype=torch.uint8, device="cuda")
        g = {k: torch.empty_like(v) for k, v in t.items()}
        io = rt.BlockIO(**{k: v.data_ptr() for k, v in t.items()}, grad_out=go.data_ptr(),
                        grad_y=gy.data_ptr(), **{"grad_" + k: v.data_ptr() for k, v in g.items()})
        tb._call(ws.device, "dcn_block_norm_bwd", d, io, ws.data_ptr(), n.value)
        assert bool((ws[n.value:] == fill).all())
        results.append(g)
    for k, v in results[0].items():
        assert torch.equal(v, results[1][k]) and bool(torch.isfinite(v).all()), k


# ---- the sums in 32 bits
@pytest.mark.parametrize("layout,C,P", [("nchw", 64, 50), ("nchw", 256, 196), ("nchw", 512, 49),
                                        ("nchw", 1024, 49), ("nchw", 2048, 33), ("rows", 64, 50),
                                        ("rows", 256, 196), ("rows", 1024, 60), ("rows", 4096, 40),
                                        ("rows", 8192, 24), ("rows", 16384, 24)])
@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms")])
def test_sums_keep_fp32(tb, layout, C, P, post, pre):
    """fp32 all the way: bounds of a few dozen roundings whatever the length (1e-4 of the magnitudes),
    which half a bf16 step (2e-3) would pass many times over.

    A sum over n values that each kernel takes as chains of at most m terms, joined by a tree
    and a few partial sums, is off by at most (m + depth) u of its magnitudes: m <= 32 channels
    of a thread, depth <= 6 lane steps + 16 waves. A parameter's gradient: at most 64 positions of a
    thread here (4 images of P over the workgroups), the fold's 64 partials and 4 steps. So 96 u and
    176 u of a sum's magnitudes in place of n u; two norms forward and two backward chain at most a
    dozen such sums and products (16)."""
    B = 4
    t, go, gy = N.tensors(layout, B, C, P, torch.float32, post, pre, "full", seed=C)
    for v in t.values():
        v.requires_grad_()
    out, y = N.call(tb, t, post, pre, "silu")
    grads = torch.autograd.grad((out, y), list(t.values()), (go, gy))
    ref = {k: N.rows(v, layout).requires_grad_() for k, v in t.items()}
    kw = dict(post=post, pre=pre, act="silu")
    ro, ry = BO.block_forward(ref, **kw)
    rg = torch.autograd.grad((ro, ry), list(ref.values()), (N.rows(go, layout), N.rows(gy, layout)))
    with torch.no_grad():
        b = BO.block_bounds({k: v.detach() for k, v in ref.items()}, N.rows(go, layout),
                            N.rows(gy, layout), **kw)
    full = {"x", "residual", "gate"}
    for k, a, r in [("out", out, ro), ("y", y, ry), *zip(t, grads, rg)]:
        n = 96 if k in full or k in ("out", "y") else 176
        err = (N.rows(a, layout) - r.detach()).abs() / (16 * n * U * b[k] + 1e-37)
        assert float(err.max()) <= 1, (k, float(err.max()))
