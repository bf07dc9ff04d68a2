"""GPU: the block operators together, as a network uses them (torch_block.DeformBlock): every
stage of a training step, forward and backward, against the 64-bit oracles fed with that
stage's own inputs and upstream gradient, so each is held to its own operator's tolerance (the
bounds of test_gpu_block_norm.py, test_gpu_fp8.py, and 1e-3 of the largest value for
DeformConv2d in fp32 as in test_gpu_ednet.py; in bf16 its offsets are rounded, a sample may fall
on the other side of a pixel than the oracle's and its derivative jump, which no bound on a largest
difference covers: test_gpu_bf16.py holds that operator against its own oracle)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import block_oracle as BO  # noqa: E402
from test_gpu_fp8 import by_channel, close, np64, tok  # noqa: E402

U = 2.0 ** -24
SEED = 5


@pytest.fixture(scope="module")
def tb():
    import torch_block
    return torch_block


def make_block(tb, C, dt, drop, seed=0):
    torch.manual_seed(seed)
    rng = tuple(torch.tensor([SEED, i], dtype=torch.int64, device="cuda") for i in (1, 2))
    m = tb.DeformBlock(C, expand=2, layer_scale=0.5, drop_path=drop, rng=rng)
    with torch.no_grad():
        m.dcn.offset_conv.weight.normal_(0, 0.02)
        m.dcn.offset_conv.bias.uniform_(-0.4, 0.4)
        for n, p in m.named_parameters():
            if "post" in n or "pre" in n or n.endswith("scale"):
                p.add_(0.1 * torch.randn_like(p))
    return m.to("cuda", dt)


def run(m, x, go):
    """One step with every intermediate and its gradient kept."""
    t = {"x": x.detach().requires_grad_()}
    _, t["y0"] = m.norm(None, t["x"])
    t["h0"] = m.dcn(t["y0"])
    t["x1"], t["y1"] = m.join(t["h0"], t["x"])
    t["u"] = m.fc1(t["y1"])
    t["a"] = m.act(t["u"])
    t["v"] = m.fc2(t["a"])
    t["out"] = m.leave(t["v"], t["x1"])[0]
    for v in t.values():
        v.retain_grad()
    t["out"].backward(go)
    return t


def pos(v):
    """[B][P][C] float64 of a map."""
    return v.detach().cpu().double().flatten(2).transpose(1, 2)


def norm_stage(t, params, ins, outs, factor=None, **kw):
    """One block-norm stage: ins {oracle name: (tensor, gradient or None)}, outs {name: tensor}."""
    leaf = {k: pos(v).requires_grad_() for k, (v, _) in ins.items()}
    leaf.update({k: p.detach().cpu().double().requires_grad_() for k, p in params.items()})
    o, y = BO.block_forward(leaf, factor=factor, **kw)
    got = {"out": o, "y": y}
    up = {k: pos(v.grad) for k, v in outs.items()}
    names = list(leaf)
    ref = dict(zip(names, torch.autograd.grad([got[k] for k in outs], [leaf[k] for k in names],
                                              [up[k] for k in outs], allow_unused=True)))
    with torch.no_grad():
        b = BO.block_bounds({k: v.detach() for k, v in leaf.items()}, up.get("out"), up.get("y"),
                            factor=factor, **kw)
    half = 2.0 ** -8 if next(iter(outs.values())).dtype == torch.bfloat16 else 0.0
    B, P, C = next(iter(leaf.values())).shape

    def check(a, r, m, n, what):
        tol = 16 * (n + 64) * U * m + half * r.abs() + 1e-37
        assert bool(((a - r).abs() <= tol).all()), what

    for k, v in outs.items():
        check(pos(v), got[k].detach(), b[k], C, k)
    for k, (_, g) in ins.items():
        if g is not None:
            check(pos(g), ref[k], b[k], C, "grad " + k)
    for k, p in params.items():
        check(p.grad.cpu().double(), ref[k], b[k], B * P + C, "grad " + k)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C,B,H,W,drop", [(64, 3, 9, 11, 0.4), (36, 2, 14, 14, 0.0)])
def test_training_step_stage_by_stage(tb, dt, C, B, H, W, drop):
    from test_gpu_ednet import OracleDCN
    m = make_block(tb, C, dt, drop)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, C, H, W, generator=g).to(dt).cuda()
    go = torch.randn(B, C, H, W, generator=g).to(dt).cuda()
    t = run(m, x, go)
    assert torch.equal(m(x), t["out"])

    def factor(i):
        if drop == 0:
            return None
        f = BO.drop_factor(B * C * H * W, C * H * W, drop, SEED, i)
        return torch.from_numpy(f).reshape(B, C, H * W).transpose(1, 2)

    eps = dict(eps=1e-6)
    # the residual's gradient at x and at x1 sums two uses: taken apart below
    norm_stage(t, {"w_pre": m.norm.pre_weight, "b_pre": m.norm.pre_bias},
               {"residual": (t["x"], None)}, {"y": t["y0"]}, pre="layer", **eps)
    norm_stage(t, {"scale": m.join.scale, "w_post": m.join.post_weight,
                   "w_pre": m.join.pre_weight, "b_pre": m.join.pre_bias},
               {"x": (t["h0"], t["h0"].grad), "residual": (t["x"], None)},
               {"out": t["x1"], "y": t["y1"]}, factor(1), post="rms", pre="layer", **eps)
    norm_stage(t, {"scale": m.leave.scale, "w_post": m.leave.post_weight},
               {"x": (t["v"], t["v"].grad), "residual": (t["x1"], t["x1"].grad)},
               {"out": t["out"]}, factor(2), post="rms", **eps)
    for fc, i, o in ((m.fc1, t["y1"], t["u"]), (m.fc2, t["a"], t["v"])):
        w = BO.fp8_value(np64(fc.weight), 128, 128)
        close(tok(o), BO.fp8_value(tok(i), 1, 128), w, dt, "product")
        close(tok(i.grad), BO.fp8_value(tok(o.grad), 1, 128), w.T, dt, "product's grad x")
        close(np64(fc.weight.grad), by_channel(o.grad), by_channel(i), dt, "product's grad w")
    if dt == torch.bfloat16:
        return
    ref = OracleDCN(C, C, 3, 1, 1).double()
    with torch.no_grad():
        for p, q in zip(ref.parameters(), (m.dcn.weight, m.dcn.bias, m.dcn.offset_conv.weight,
                                           m.dcn.offset_conv.bias)):
            assert p.shape == q.shape
            p.copy_(q.cpu().double())
    y0 = t["y0"].detach().cpu().double().requires_grad_()
    h0 = ref(y0)
    h0.backward(t["h0"].grad.cpu().double())
    for a, r in ((t["h0"], h0), (t["y0"].grad, y0.grad), (m.dcn.weight.grad, ref.weight.grad),
                 (m.dcn.bias.grad, ref.bias.grad)):
        a, r = a.detach().cpu().double(), r.detach()
        assert float((a - r).abs().max()) <= 1e-3 * float(r.abs().max())


def test_gradient_of_the_residual_stream(tb):
    """x feeds the first norm and the residual: its gradient is the sum of the two stages'."""
    m = make_block(tb, 32, torch.float32, 0.0)
    x = torch.randn(2, 32, 8, 8, device="cuda")
    t = run(m, x, torch.randn(2, 32, 8, 8, device="cuda"))
    via_norm, = torch.autograd.grad(tb.block_norm(None, (x0 := x.clone().requires_grad_()),
                                                  pre="layer", pre_weight=m.norm.pre_weight,
                                                  pre_bias=m.norm.pre_bias)[1], x0, t["y0"].grad)
    h0, x1 = t["h0"].detach(), x.clone().requires_grad_()
    o, y = m.join(h0, x1)
    via_res, = torch.autograd.grad((o, y), x1, (t["x1"].grad, t["y1"].grad))
    assert torch.equal(t["x"].grad, via_norm + via_res)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_serving_equals_evaluation(tb, dt):
    """serve() keeps the MLP's weights in the 8 bits that training rounds them to."""
    m = make_block(tb, 40, dt, 0.3).eval()
    for shape in ((1, 40, 2, 2), (5, 40, 7, 9)):
        x = torch.randn(*shape, device="cuda").to(dt)
        with torch.no_grad():
            a = m(x)
            b = m.serve()(x)
            m.train().eval()
        assert torch.equal(a, b)


def test_short_training_runs(tb):
    """Steps of Adam on two stacked blocks run, and every parameter gets a finite gradient."""
    net = torch.nn.Sequential(make_block(tb, 24, torch.float32, 0.2, 1),
                              make_block(tb, 24, torch.float32, 0.2, 2))
    opt = torch.optim.Adam(net.parameters(), lr=1e-3)
    x, y = torch.randn(4, 24, 10, 10, device="cuda"), torch.randn(4, 24, 10, 10, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        ((net(x) - y) ** 2).mean().backward()
        for n, p in net.named_parameters():
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
        opt.step()


def test_captured_training_step(tb):
    """The block's second half (join, channel MLP, leave) captured forward and backward in one
    graph: every replay gives the eager step's bits, with the rng tensors' masks of the moment."""
    m = make_block(tb, 32, torch.float32, 0.5)
    x, h, g = (torch.randn(6, 32, 9, 7, device="cuda") for _ in range(3))
    h.requires_grad_()
    leaves = [h, *(p for k in ("join", "fc1", "fc2", "leave") for p in getattr(m, k).parameters())]

    def step():
        x1, y = m.join(h, x)
        out = m.leave(m.fc2(m.act(m.fc1(y))), x1)[0]
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    seen = []
    for off in (5, 11, 23, 5):
        for r in (m.join.rng, m.leave.rng):
            r[1] = off
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), off
        seen.append(got[0].clone())
    assert torch.equal(seen[0], seen[3])
    assert not (torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2]))
