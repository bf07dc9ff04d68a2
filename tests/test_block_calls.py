"""torch_block's handling of arguments, on the CPU: the library call is replaced by one that
multiplies (block norms: out = alpha x, dropout: y = 2 x), so what reaches it shows."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import dcn_runtime as rt  # noqa: E402


@pytest.fixture
def tb(monkeypatch):
    import torch_block as tb

    def view(ptr, n):
        return torch.frombuffer((ctypes.c_float * n).from_address(ptr), dtype=torch.float32)

    def call(dev, name, d, *a):
        calls.append((name, d, a))
        if name == "dcn_dropout_fwd":
            view(a[2], d.n).copy_(2 * view(a[0], d.n))
        elif name == "dcn_block_norm_fwd":
            n = d.B * d.C * d.P
            view(a[0].out, n).copy_(d.alpha * view(a[0].x, n))

    calls = []
    tb.real_call = tb._call
    monkeypatch.setattr(tb, "_call", call)
    monkeypatch.setattr(tb, "_dtype", lambda x, what: tb._DT[x.dtype])
    tb.calls = calls
    yield tb
    del tb.calls, tb.real_call
    tb._block_desc.cache_clear()


def test_alpha_follows_its_tensor(tb):
    """A factor given as a tensor counts with the value it has at the call."""
    x, a = torch.ones(2, 4), torch.tensor(2.0)
    assert float(tb.block_norm(x, alpha=a)[0][0, 0]) == 2.0
    a.fill_(5.0)
    assert float(tb.block_norm(x, alpha=a)[0][0, 0]) == 5.0
    e = torch.tensor(0.5)
    for want in (0.5, 0.25):
        e.fill_(want)
        tb.block_norm(x, pre="rms", eps=(1e-6, e))
        assert tb.calls[-1][1].eps_pre == want
    p = torch.tensor(0.5)
    tb.block_norm(x, drop_p=p, rng=(1, 2))
    assert tb.calls[-1][1].drop_p == 0.5


def test_a_learnable_alpha_is_refused(tb):
    """alpha, eps and drop_p have no gradient: one that wants it is an error, not a number that
    stays as it is."""
    x = torch.ones(2, 4)
    for kw in (dict(alpha=torch.nn.Parameter(torch.tensor(2.0))),
               dict(pre="rms", eps=torch.tensor(1e-6, requires_grad=True)),
               dict(drop_p=torch.tensor(0.5, requires_grad=True), rng=(1, 2))):
        with pytest.raises(TypeError, match="no gradient"):
            tb.block_norm(x, **kw)
    with pytest.raises(TypeError, match="no gradient"):
        tb.dropout(x, torch.tensor(0.5, requires_grad=True), (1, 2))
    with torch.no_grad():  # nothing to lose there
        a = torch.nn.Parameter(torch.tensor(3.0))
        assert float(tb.block_norm(x, alpha=a)[0][0, 0]) == 3.0
    m = tb.BlockNorm(4, post=None, pre=None, alpha=torch.nn.Parameter(torch.tensor(2.0)))
    with pytest.raises(TypeError, match="no gradient"):
        m(x)


def test_forward_mode_is_refused(tb):
    """A tangent is never dropped: the operators have no forward-mode derivative and say so."""
    import torch.autograd.forward_ad as fa
    x = torch.ones(2, 4)
    with fa.dual_level():
        dual = fa.make_dual(x, torch.ones(2, 4))
        for f in (lambda: tb.dropout(dual, 0.5, (1, 2)),
                  lambda: tb.dropout(x, 0.5, (1, 2), residual=dual),
                  lambda: tb.block_norm(dual), lambda: tb.block_norm(x, dual),
                  lambda: tb.block_norm(x, scale=fa.make_dual(torch.ones(4), torch.ones(4))),
                  lambda: tb.fp8_pointwise(dual, torch.ones(3, 4))):
            with pytest.raises(NotImplementedError, match="jvp"):
                f()
        assert float(tb.dropout(x, 0.5, (1, 2))[0, 0]) == 2.0  # no tangent, nothing to refuse


def _served(tb, o, c):
    w = tb.Fp8Weight.__new__(tb.Fp8Weight)
    w.q = torch.zeros(o, 128, dtype=torch.uint8)
    w.exponents = torch.zeros(1, 1, dtype=torch.uint8)
    w.out_features, w.in_features = o, c
    return w


def test_forward_mode_of_a_served_product_is_refused(tb):
    import torch.autograd.forward_ad as fa
    with fa.dual_level():
        dual = fa.make_dual(torch.ones(2, 4), torch.ones(2, 4))
        with pytest.raises(RuntimeError, match="inference"):
            tb.fp8_pointwise(dual, _served(tb, 3, 4))


@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused(tb, monkeypatch):
    """torch.jit.trace and make_fx record torch's operations: they would keep the empty result that a
    call fills, or the call with the sizes of the traced tensors. Nothing is recorded instead."""
    from torch.fx.experimental.proxy_tensor import make_fx
    monkeypatch.setattr(tb, "_call", tb.real_call)
    x, w = torch.ones(2, 4), torch.ones(3, 4)
    for f, args in ((lambda x: tb.dropout(x, 0.5, (1, 2)) + 1, (x,)),
                    (lambda x: tb.dropout(x, 0.5, (1, 2)) + 1, (x.clone().requires_grad_(),)),
                    (lambda x: tb.block_norm(x, alpha=3.0)[0] + 1, (x,)),
                    (lambda x: tb.block_norm(x, alpha=3.0)[0] + 1, (x.clone().requires_grad_(),)),
                    (lambda x: tb.fp8_pointwise(x, w), (x,)),
                    (lambda x: tb.fp8_pointwise(x, _served(tb, 3, 4)), (x,)),
                    (lambda x: tb.fp8_quantize(x)[0], (x,)),
                    (lambda w: tb._quantize_weight(w, True, False)[0], (w,))):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, args, check_trace=False)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(*args)


def test_image_draws_of_flat_features(tb):
    """drop="image" draws once per x[b], for features [N, C] too, as dropout(group="image")."""
    x = torch.ones(6, 4)
    tb.block_norm(x, drop_p=0.5, drop="image", rng=(1, 2))
    d = tb.calls[-1][1]
    assert (d.B, d.C, d.P, d.drop_image) == (6, 4, 1, 1)
    tb.block_norm(x, drop_p=0.5, rng=(1, 2))  # per element: one run of tokens, as before
    assert (tb.calls[-1][1].B, tb.calls[-1][1].P) == (1, 6)
    tb.block_norm(x, torch.ones(6, 4), gate=torch.ones(1, 4), drop_p=0.5, drop="image", rng=(1, 2))
    d = tb.calls[-1][1]
    assert (d.B, d.P, d.gate) == (6, 1, rt.DCN_GATE_FULL)


def test_dropout_groups_of_any_size(tb):
    """A group above the element count is one draw; it never wraps around in 64 bits."""
    x = torch.ones(2, 4)
    for g in (8, 9, 2 ** 63, 2 ** 64 + 1, 10 ** 30):
        tb.dropout(x, 0.5, (1, 2), group=g)
        assert tb.calls[-1][1].group >= 8
    with pytest.raises(ValueError, match="group"):
        tb.dropout(x, 0.5, (1, 2), group=2.5)
    with pytest.raises(ValueError, match="group"):
        tb.dropout(x, 0.5, (1, 2), group=0)


def _workspace(**kw):
    d = rt.BlockDesc(**{**dict(B=1, C=64, P=1, layout=rt.DCN_NHWC, dtype=rt.DCN_F32, post=1, pre=1,
                               alpha=1.0), **kw})
    n = ctypes.c_size_t()
    rt.check(rt.load().dcn_block_norm_workspace(d, n))
    return n.value


@pytest.mark.parametrize("kw,floats", [
    (dict(C=4096), 5 * 4096), (dict(C=4096, P=100), 100 * 5 * 4096),
    (dict(C=4096, P=10000), 512 * 5 * 4096), (dict(C=8192), 64 + 5 * 8192),
    (dict(C=16384, P=512, dtype=rt.DCN_BF16), 6 * 512 + 32 * 5 * 16384),
    (dict(C=16384, P=512), 6 * 512 + 16 * 5 * 16384),
    (dict(C=8192, P=512, dtype=rt.DCN_BF16, gate=rt.DCN_GATE_FULL), 6 * 512 + 256 * 5 * 8192),
    (dict(B=2, C=256, P=49, layout=rt.DCN_NCHW), 8 * 5 * 256),
    (dict(B=64, C=256, P=784, layout=rt.DCN_NCHW, gate=rt.DCN_GATE_IMAGE),
     (1024 * 6 + 64 * 8) * 256)])
def test_block_norm_workspace_holds_what_is_launched(kw, floats):
    """Partials of no more workgroups than the call has tiles or its kernel launches."""
    assert _workspace(**kw) == 4 * floats
