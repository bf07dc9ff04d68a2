"""GPU: the block norms (torch_block.block_norm, dcn_block_norm_*) against the 64-bit oracle.

Tolerances: with M the output's formula in magnitudes (block_oracle.block_bounds), n the number
of terms of its longest sum and u = 2^-24, |Δ| <= 16 n' u M + eps/2 |ref|, n' = n + 64. A sum of
n fp32 terms is off by at most n u of its magnitudes whatever its order; two norms forward and
two backward chain at most a dozen such sums and products of them (16), 64 covers the
elementwise roundings, eps/2 the store in the tensor's type."""
import itertools

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import block_oracle as BO  # noqa: E402

SEED, OFF = 77, 0x123456789A
U = 2.0 ** -24


@pytest.fixture(scope="module")
def tb():
    import torch_block
    return torch_block


def tensors(layout, B, C, P, dt, post, pre, gate, seed=0, x=True, residual=True, params=True,
            shift=0.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)
    shape = (B, C, P, 1) if layout == "nchw" else (B, P, C)
    t = {}
    if x:
        t["x"] = rnd(*shape) * 0.7 + shift
        if gate == "full":
            t["gate"] = rnd(*shape)
        elif gate == "image":
            t["gate"] = rnd(B, C)
        if params:
            t["scale"] = rnd(C) * 0.1 + 0.5
            if post:
                t["w_post"] = 1 + 0.2 * rnd(C)
            if post == "layer":
                t["b_post"] = 0.2 * rnd(C)
    if residual:
        t["residual"] = rnd(*shape) * 2 + shift
    if params and pre:
        t["w_pre"] = 1 + 0.2 * rnd(C)
        if pre == "layer":
            t["b_pre"] = 0.2 * rnd(C)
    t = {k: v.to(dt).cuda() for k, v in t.items()}
    return t, rnd(*shape).to(dt).cuda(), rnd(*shape).to(dt).cuda()


def rows(v, layout):
    """float64 on the CPU, [B][P][C] for a map tensor."""
    if v is None:
        return None
    v = v.detach().cpu().double()
    return v[..., 0].transpose(1, 2) if layout == "nchw" and v.dim() == 4 else v


def call(tb, t, post, pre, act, p=0.0, drop="element", rng=(SEED, OFF), **kw):
    return tb.block_norm(t.get("x"), t.get("residual"), gate=t.get("gate"), gate_act=act,
                         scale=t.get("scale"), post=post, post_weight=t.get("w_post"),
                         post_bias=t.get("b_post"), pre=pre, pre_weight=t.get("w_pre"),
                         pre_bias=t.get("b_pre"), drop_p=p, drop=drop, rng=rng, **kw)


def run_and_check(tb, layout, B, C, P, dt, post, pre, gate="none", act="linear", p=0.0,
                  drop="element", alpha=1.0, eps=1e-6, use=("out", "y"), **mk):
    t, go, gy = tensors(layout, B, C, P, dt, post, pre, gate, **mk)
    for v in t.values():
        v.requires_grad_()
    out, y = call(tb, t, post, pre, act, p, drop, alpha=alpha, eps=eps)
    ref = {k: rows(v, layout).requires_grad_() for k, v in t.items()}
    factor = None
    if p > 0:
        n = B * C * P
        f = torch.from_numpy(BO.drop_factor(n, C * P if drop == "image" else 1, p, SEED, OFF))
        factor = f.reshape(B, C, P).transpose(1, 2) if layout == "nchw" else f.reshape(B, P, C)
    kw = dict(post=post, pre=pre, act=act, alpha=alpha, eps=eps, factor=factor)
    rout, ry = BO.block_forward(ref, **kw)
    use = [u for u in use if not (u == "y" and not pre) and not (u == "out" and "x" not in t)]
    g64 = {"out": rows(go, layout), "y": rows(gy, layout)}
    pick = {"out": (out, go, rout), "y": (y, gy, ry)}
    grads = torch.autograd.grad([pick[u][0] for u in use], list(t.values()),
                                [pick[u][1] for u in use], allow_unused=True)
    refg = torch.autograd.grad([pick[u][2] for u in use], list(ref.values()),
                               [g64[u] for u in use], allow_unused=True)
    with torch.no_grad():
        bounds = BO.block_bounds({k: v.detach() for k, v in ref.items()},
                                 g64["out"] if "out" in use else None,
                                 g64["y"] if "y" in use else None, **kw)
    half = torch.finfo(dt).eps / 2 if dt == torch.bfloat16 else 0.0
    got = {"out": (out, rout, C)} if "x" in t else {}
    if pre:
        got["y"] = (y, ry, C)
    for k, a, r in zip(t, grads, refg):
        if r is None:  # a gradient that no output reaches
            assert a is None or not a.any()
            continue
        n = C if k in ("x", "residual") or (k == "gate" and gate == "full") else \
            (P if k == "gate" else B * P) + C
        got["grad " + k] = (a, r, n)
    for name, (a, r, n) in got.items():
        m = bounds[name.replace("grad ", "")]
        a, r = rows(a, layout), r.detach()
        assert a.shape == r.shape, name
        tol = 16 * (n + 64) * U * m + half * r.abs() + 1e-37
        err = (a - r).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (f"{name}: {int(bad.sum())} / {bad.numel()} off, worst "
                               f"{float((err / tol).max()):.2f} x tolerance")


NORMS = [None, "rms", "layer"]
DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("post,pre", [p for p in itertools.product(NORMS, NORMS)])
@pytest.mark.parametrize("gate,act", [("none", "linear"), ("full", "silu"), ("image", "sigmoid")])
def test_variants(tb, dt, layout, post, pre, gate, act):
    run_and_check(tb, layout, 3, 40, 29, dt, post, pre, gate, act, p=0.1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("C", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129,
                               255, 256, 257, 511, 513, 1000, 1023, 1025])
def test_channel_counts(tb, dt, layout, C):
    run_and_check(tb, layout, 2, C, 11, dt, "layer", "rms", "full", "silu", p=0.25, seed=C)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout,B,C,P", [
    ("rows", 1, 64, 1), ("rows", 1, 4096, 1), ("nchw", 1, 64, 1), ("nchw", 5, 33, 1),
    ("rows", 5, 33, 1), ("rows", 1, 2047, 3), ("rows", 2, 2048, 5), ("rows", 1, 4097, 4),
    ("rows", 1, 8192, 3), ("rows", 1, 16384, 2), ("rows", 1, 16385, 2), ("rows", 1, 20000, 2),
    ("nchw", 1, 2048, 7), ("nchw", 1, 2049, 9), ("nchw", 1, 4099, 8), ("nchw", 2, 600, 49),
    ("nchw", 300, 8, 4), ("rows", 300, 8, 4), ("nchw", 2, 256, 784), ("rows", 2, 256, 784),
    ("nchw", 3, 64, 31), ("nchw", 3, 64, 32), ("nchw", 3, 64, 33), ("nchw", 2, 16, 3137),
    ("rows", 3, 24, 1601)])
@pytest.mark.parametrize("gate", ["none", "image"])
def test_shapes(tb, dt, layout, B, C, P, gate):
    run_and_check(tb, layout, B, C, P, dt, "rms", "layer", gate, "silu", seed=C + P)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout,B,C,P", [
    ("nchw", 16, 256, 784), ("nchw", 24, 128, 1003), ("nchw", 8, 512, 300), ("nchw", 300, 16, 260),
    ("nchw", 2, 64, 8193), ("rows", 16, 256, 784), ("rows", 700, 40, 5), ("rows", 3, 1024, 700)])
@pytest.mark.parametrize("gate", ["none", "image"])
def test_many_tiles(tb, dt, layout, B, C, P, gate):
    """Enough tiles that workgroups take several, in turn, over image borders: every workgroup's
    share of the parameter and gate gradients has to arrive once."""
    run_and_check(tb, layout, B, C, P, dt, "layer", "rms", gate, "silu", seed=B + P)


@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("C", [48, 300, 3000])
def test_backward_without_kept_statistics(tb, layout, C):
    """dcn_block_norm_bwd computes the statistics again where it gets none: the kept ones are the
    same numbers up to the summation order of the same kernel, so the gradients agree to fp32
    rounding (16 (C + 64) u of their magnitudes on either side)."""
    import ctypes

    import dcn_runtime as rt
    t, go, gy = tensors(layout, 3, C, 70, torch.float32, "layer", "rms", "full")
    names = list(t)
    for v in t.values():
        v.requires_grad_()
    want = torch.autograd.grad(call(tb, t, "layer", "rms", "silu"), list(t.values()), (go, gy))
    d = rt.BlockDesc(3, C, 70, 0 if layout == "nchw" else 1, rt.DCN_F32, 2, 1, 1, 2, 1e-6, 1e-6,
                     1.0, 0.0, 0, 0, 0)
    n = ctypes.c_size_t()
    rt.check(rt.load().dcn_block_norm_workspace(d, n))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    got = {k: torch.full_like(v, float("nan")) for k, v in t.items()}
    io = rt.BlockIO(**{k: v.data_ptr() for k, v in t.items()}, grad_out=go.data_ptr(),
                    grad_y=gy.data_ptr(), **{"grad_" + k: v.data_ptr() for k, v in got.items()})
    tb._call(ws.device, "dcn_block_norm_bwd", d, io, ws.data_ptr(), n.value)
    ref = {k: rows(v, layout) for k, v in t.items()}
    b = BO.block_bounds(ref, rows(go, layout), rows(gy, layout), post="layer", pre="rms", act="silu")
    for k, w in zip(names, want):
        terms = C if k in ("x", "residual", "gate") else 3 * 70 + C
        err = (rows(got[k], layout) - rows(w, layout)).abs()
        assert bool((err <= 2 * 16 * (terms + 64) * U * b[k] + 1e-37).all()), k


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_parts(tb, dt, layout):
    """Absent pieces: the pre norm alone, no residual, no parameters, no pre norm, a gradient of
    one output only, per-image dropout, another alpha and eps."""
    base = (tb, layout, 4, 50, 37, dt)
    for pre in ("rms", "layer"):
        run_and_check(*base, None, pre, x=False)
        run_and_check(*base, None, pre, x=False, params=False)
    run_and_check(*base, "layer", "layer", residual=False)
    run_and_check(*base, "rms", "layer", params=False, gate="full", act="linear")
    run_and_check(*base, "rms", None, p=0.5)
    run_and_check(*base, None, None, gate="image", act="silu")
    run_and_check(*base, "layer", "rms", use=("out",))
    run_and_check(*base, "layer", "rms", use=("y",), gate="full", act="sigmoid")
    run_and_check(*base, "layer", "rms", p=0.4, drop="image", alpha=-0.5, eps=1e-2)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_large_mean(tb, dt, layout):
    """Means far above the spread: the variance is taken about the mean."""
    run_and_check(tb, layout, 2, 300, 21, dt, "layer", "layer", shift=64.0)


@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_zero_rows_and_non_finite(tb, layout):
    """A row of zeros normalises to zero; a NaN or infinity stays in its own position."""
    t, _, _ = tensors(layout, 2, 48, 10, torch.float32, "rms", "rms", "none")
    x, res = t["x"], t["residual"]
    put = (lambda v, b, p, c, w: v.__setitem__((b, c, p, 0), w)) if layout == "nchw" else \
        (lambda v, b, p, c, w: v.__setitem__((b, p, c), w))
    clean_out, clean_y = call(tb, t, "rms", "rms", "linear")
    for c in range(48):
        put(x, 0, 3, c, 0.0)
        put(res, 0, 3, c, 0.0)
    put(x, 1, 5, 7, float("nan"))
    put(res, 1, 8, 2, float("inf"))
    out, y = call(tb, t, "rms", "rms", "linear")
    ro, rc, ry, rcy = (rows(v, layout) for v in (out, clean_out, y, clean_y))
    assert not ro[0, 3].any() and not ry[0, 3].any()
    assert torch.isnan(ro[1, 5]).all() and torch.isnan(ry[1, 5]).all()
    assert torch.isinf(ro[1, 8, 2]) and torch.isnan(ry[1, 8, 2])
    keep = torch.ones(2, 10, dtype=torch.bool)
    keep[0, 3] = keep[1, 5] = keep[1, 8] = False
    assert torch.equal(ro[keep], rc[keep]) and torch.equal(ry[keep], rcy[keep])


@pytest.mark.parametrize("drop", ["element", "image"])
@pytest.mark.parametrize("gate", ["none", "full", "image"])
@pytest.mark.parametrize("layout,C", [("nchw", 48), ("nchw", 2100), ("rows", 48), ("rows", 3000),
                                      ("rows", 8000), ("rows", 16500)])
def test_dropped_values_reach_nothing(tb, layout, C, gate, drop):
    """NaN and infinities where dropout drops give the bits that zeros there give. (Per element
    without a norm after the block: with one, a NaN spreads over its position.)"""
    B, P, p = 4, 6, 0.5
    post = "layer" if drop == "image" else None
    t, go, gy = tensors(layout, B, C, P, torch.float32, post, "layer", gate)
    f = torch.from_numpy(BO.drop_factor(B * C * P, C * P if drop == "image" else 1, p, SEED, OFF))
    f = f.reshape(B, C, P, 1) if layout == "nchw" else f.reshape(B, P, C)
    dropped = (f == 0).cuda()
    assert dropped.any() and not dropped.all()
    names = ["x"] + (["gate"] if gate == "full" or (gate == "image" and drop == "image") else [])
    results = []
    for bad in (0.0, float("nan"), float("-inf")):
        u = {k: v.clone() for k, v in t.items()}
        for k in names:
            m = dropped if u[k].shape == dropped.shape else dropped.flatten(1)[:, :1].expand(B, C)
            u[k][m] = bad
        for v in u.values():
            v.requires_grad_()
        o, y = call(tb, u, post, "layer", "silu", p=p, drop=drop)
        results.append([o, y, *torch.autograd.grad((o, y), list(u.values()), (go, gy))])
    assert all(torch.isfinite(v).all() for v in results[0])
    for r in results[1:]:
        for k, a, b in zip(["out", "y", *t], results[0], r):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("layout,C", [("nchw", 48), ("nchw", 2100), ("rows", 48), ("rows", 3000),
                                      ("rows", 8000), ("rows", 16500)])
def test_a_bad_gate_stays_in_its_image(tb, layout, C):
    """A NaN gate of a kept image leaves the dropped images' gate gradients 0 and their results
    the residual's."""
    B, P, p = 6, 5, 0.5
    t, go, gy = tensors(layout, B, C, P, torch.float32, "rms", "rms", "image")
    f = torch.from_numpy(BO.drop_factor(B * C * P, C * P, p, SEED, OFF)).reshape(B, -1)[:, 0]
    assert (f > 0).any() and (f == 0).any()
    t["gate"][f.cuda() > 0] = float("nan")
    for v in t.values():
        v.requires_grad_()
    o, y = call(tb, t, "rms", "rms", "silu", p=p, drop="image")
    gx, gg = torch.autograd.grad((o, y), (t["x"], t["gate"]), (go, gy))
    gone = (f == 0).cuda()
    assert torch.equal(o[gone], t["residual"][gone]) and torch.isfinite(y[gone]).all()
    assert not gx[gone].any() and not gg[gone].any()
    assert torch.isnan(gg[~gone]).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_layouts_and_strides_agree(tb, dt):
    """Channels-last memory, transposed and sliced inputs give the results of dense copies (no
    dropout, whose elements count in memory order), each gradient in its input's shape."""
    t, go, gy = tensors("nchw", 3, 24, 35, dt, "layer", "rms", "full")
    t = {k: v.reshape(3, 24, 5, 7) if v.dim() == 4 else v for k, v in t.items()}
    go, gy = go.reshape(3, 24, 5, 7), gy.reshape(3, 24, 5, 7)

    def run(conv, names):
        u = {k: (conv(v) if k in names else v.clone()).requires_grad_() for k, v in t.items()}
        o, y = call(tb, u, "layer", "rms", "silu")
        g = torch.autograd.grad((o, y), list(u.values()), (go, gy))
        return [o, y, *g]

    cl = lambda v: v.contiguous(memory_format=torch.channels_last) if v.dim() == 4 else v

    def odd(v):  # one element off the allocation's start
        w = torch.empty(v.numel() + 1, dtype=v.dtype, device=v.device)[1:].view(v.shape)
        return w.copy_(v)

    def wide(v):  # every second column of a larger tensor
        w = torch.zeros(*v.shape[:-1], 2 * v.shape[-1], dtype=v.dtype, device=v.device)
        w[..., ::2] = v
        return w[..., ::2]

    want = run(torch.clone, ())
    for conv, names in ((wide, list(t)), (odd, list(t)), (cl, ["residual", "gate"])):
        got = run(lambda v: conv(v.detach()).detach(), names)
        for a, b in zip(got, want):
            assert a.shape == b.shape and torch.equal(a, b)
    got = run(lambda v: cl(v.detach()), list(t))  # runs as token rows: another summation order
    tol = 2.0 ** -7 if dt == torch.bfloat16 else 1e-4
    for a, b in zip(got, want):
        assert a.shape == b.shape
        assert float((a - b).abs().max()) <= tol * float(b.abs().max())


@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_bitwise_reproducible_and_graph(tb, layout):
    t, go, gy = tensors(layout, 8, 96, 333, torch.bfloat16, "layer", "layer", "image")
    for v in t.values():
        v.requires_grad_()
    rng = torch.tensor([3, 4], dtype=torch.int64, device="cuda")

    def step():
        o, y = call(tb, t, "layer", "layer", "sigmoid", p=0.2, rng=rng)
        return [o.detach(), y.detach(), *torch.autograd.grad((o, y), list(t.values()), (go, gy))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = step()
        b = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = step()
    with torch.cuda.graph(g2):
        r2 = step()
    for off in (4, 9, 4):
        rng.copy_(torch.tensor([3, off]))
        g1.replay()
        e1 = step()
        g2.replay()
        torch.cuda.synchronize()
        for u, v, w in zip(r1, r2, e1):
            assert torch.equal(u, w) and torch.equal(v, w)


@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_more_than_2_31_elements(tb, layout):
    """The last image of a large tensor gives the bits that it gives alone; its mask, drawn once per
    image with p = 1/2, is an exact factor 2."""
    B, C, P = 4, 256, 2_100_003
    shape = (B, C, P, 1) if layout == "nchw" else (B, P, C)
    assert B * C * P > 2 ** 31
    make = lambda *s: torch.randn(s, device="cuda", dtype=torch.bfloat16)
    t = {"x": make(*shape), "residual": make(*shape), "gate": make(*shape)}
    vec = {"w_post": make(C), "w_pre": make(C)}
    g = make(*shape)
    seed = next(s for s in range(100) if BO.drop_factor(4, 1, 0.5, s, OFF)[3] > 0)

    def step(t, g, **kw):
        for v in t.values():
            v.requires_grad_()
        o, y = call(tb, {**t, **vec}, "rms", "rms", "silu", rng=(seed, OFF), **kw)
        return [o.detach(), y.detach(), *torch.autograd.grad((o, y), list(t.values()), (g, g))]

    whole = step(t, g, p=0.5, drop="image")
    last = {k: v.detach()[3:].contiguous() for k, v in t.items()}
    alone = step(last, g[3:].contiguous(), alpha=2.0)
    for k, a, b in zip(("out", "y", *t), whole, alone):
        assert torch.equal(a[3:], b), k


@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_image_gate_sums_over_2_31_elements(tb, layout):
    """Small integers: every partial sum is exact in fp32, the result is rounded once."""
    B, C, P = 3, 260, 2_800_001
    shape = (B, C, P, 1) if layout == "nchw" else (B, P, C)
    assert B * C * P > 2 ** 31
    ints = lambda n, *s: torch.randint(-n, n + 1, s, device="cuda", dtype=torch.int8).bfloat16()
    x, go, gate = ints(2, *shape), ints(1, *shape), ints(3, B, C).requires_grad_()
    out, _ = tb.block_norm(x, gate=gate)
    got, = torch.autograd.grad(out, gate, go)
    dim = 2 if layout == "nchw" else 1
    for b in range(B):
        want = sum((x[b:b + 1].narrow(dim, i, min(700_000, P - i)).double() *
                    go[b:b + 1].narrow(dim, i, min(700_000, P - i)).double()).sum(dim).reshape(C)
                   for i in range(0, P, 700_000))
        assert float(want.abs().max()) < 2 ** 24
        assert torch.equal(got[b], want.bfloat16()), b


def test_two_threads_two_streams(tb):
    """Calls from two threads, each on its own stream, give the bits of one after the other."""
    import threading
    sets = []
    for i in range(2):
        t, go, gy = tensors("nchw" if i else "rows", 4, 128, 500 + i, torch.bfloat16, "layer",
                            "rms", "full", seed=i)
        for v in t.values():
            v.requires_grad_()
        sets.append((t, go, gy))

    def step(i):
        t, go, gy = sets[i]
        o, y = call(tb, t, "layer", "rms", "silu", p=0.2)
        return [o.detach(), y.detach(), *torch.autograd.grad((o, y), list(t.values()), (go, gy))]

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = step(i)
            s.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))


def test_in_place_out(tb):
    """dcn_block_norm_fwd with out = residual gives the bits of separate tensors."""
    import dcn_runtime as rt
    for layout in ("nchw", "rows"):
        for C in (96, 5000, 20000):
            t, _, _ = tensors(layout, 2, C, 7, torch.bfloat16, "rms", "layer", "none")
            out, y = call(tb, t, "rms", "layer", "linear")
            d = rt.BlockDesc(2, C, 7, 0 if layout == "nchw" else 1, rt.DCN_BF16, 1, 2, 0, 0,
                             1e-6, 1e-6, 1.0, 0.0, 0, 0, 0)
            r, y2 = t["residual"].clone(), torch.empty_like(y)
            io = rt.BlockIO(x=t["x"].data_ptr(), residual=r.data_ptr(),
                            scale=t["scale"].data_ptr(), w_post=t["w_post"].data_ptr(),
                            w_pre=t["w_pre"].data_ptr(), b_pre=t["b_pre"].data_ptr(),
                            out=r.data_ptr(), y=y2.data_ptr())
            tb._call(r.device, "dcn_block_norm_fwd", d, io)
            assert torch.equal(r, out) and torch.equal(y2, y)


def test_directional_difference(tb):
    """Gradients against central differences of the operator itself (fp32): the sum of the
    outputs along go, gy changes by the gradients along a direction. The oracle's difference
    with the same step has the same truncation; the operator's own rounding is below
    16 (C + 64) u of the outputs' magnitudes, divided by the step."""
    layout, B, C, P = "nchw", 2, 24, 15
    t, go, gy = tensors(layout, B, C, P, torch.float32, "layer", "rms", "image")
    d = {k: torch.randn(v.shape, generator=torch.Generator().manual_seed(9)).cuda()
         for k, v in t.items()}
    u = {k: v.clone().requires_grad_() for k, v in t.items()}
    grads = torch.autograd.grad(call(tb, u, "layer", "rms", "silu"), list(u.values()), (go, gy))
    along = sum(float((g.double() * d[k].double()).sum()) for g, k in zip(grads, u))
    h, s = 2.0 ** -8, []
    mag = 0.0
    for sign in (1, -1):
        v = {k: t[k] + sign * h * d[k] for k in t}
        o, y = call(tb, v, "layer", "rms", "silu")
        s.append(float((o.double() * go).sum() + (y.double() * gy).sum()))
        b = BO.block_bounds({k: rows(w, layout) for k, w in v.items()}, None, None, post="layer",
                            pre="rms", act="silu")
        mag += float((b["out"] * rows(go, layout).abs()).sum() +
                     (b["y"] * rows(gy, layout).abs()).sum())
    diff = (s[0] - s[1]) / (2 * h)

    def oracle(sign):
        v = {k: rows(t[k], layout) + sign * h * rows(d[k], layout) for k in t}
        o, y = BO.block_forward(v, post="layer", pre="rms", act="silu")
        return float((o * rows(go, layout)).sum() + (y * rows(gy, layout)).sum())

    trunc = abs((oracle(1) - oracle(-1)) / (2 * h) - along)
    assert abs(diff - along) <= trunc + 16 * (C + 64) * U * mag / (2 * h)
    assert trunc <= 0.02 * abs(along) + 0.05


def test_refusals(tb):
    t, _, _ = tensors("nchw", 2, 8, 6, torch.float32, "rms", "rms", "full")
    ok = dict(x=t["x"], residual=t["residual"])
    tb.block_norm(**ok, pre="rms")
    for kw, err in [(dict(pre="batch"), ValueError), (dict(gate_act="relu"), ValueError),
                    (dict(drop="row", drop_p=0.1), ValueError), (dict(drop_p=1.1), ValueError),
                    (dict(drop_p=0.1), ValueError), (dict(scale=t["x"]), ValueError),
                    (dict(gate=t["x"][:1]), ValueError),
                    (dict(pre_weight=torch.ones(8, device="cuda")), RuntimeError),
                    (dict(post_weight=torch.ones(8, device="cuda"), pre="rms"), RuntimeError),
                    (dict(pre="rms", eps=float("nan")), RuntimeError),
                    (dict(pre="rms", eps=-1.0), RuntimeError),
                    (dict(scale=torch.ones(8, device="cuda").bfloat16()), ValueError)]:
        with pytest.raises(err):
            tb.block_norm(**ok, **kw)
    with pytest.raises(ValueError):
        tb.block_norm()
    with pytest.raises(ValueError):
        tb.block_norm(t["x"], t["residual"].bfloat16())
    with pytest.raises(RuntimeError):
        tb.block_norm(None, t["residual"])


def test_empty_and_modules(tb):
    m = tb.BlockNorm(16, post="layer", pre="layer", layer_scale=0.5, drop_p=0.3).cuda()
    x = torch.randn(4, 16, 6, 6, device="cuda", requires_grad=True)
    out, y = m(x, x * 2)
    (out.sum() + (y * y).sum()).backward()
    assert all(p.grad is not None for p in m.parameters()) and x.grad is not None
    m.eval()
    a, b = m(x, x), m(x, x)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    e = x.detach()[:0].requires_grad_()
    out, y = m(e, e)
    assert out.shape == y.shape == (0, 16, 6, 6)
    for p in m.parameters():
        p.grad = None
    y.sum().backward()
    assert not m.pre_weight.grad.any()
