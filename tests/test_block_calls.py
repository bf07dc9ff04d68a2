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
    monkeypatch.setattr(tb, "_call", call)
    monkeypatch.setattr(tb, "_dtype", lambda x, what: tb._DT[x.dtype])
    tb.calls = calls
    yield tb
    del tb.calls
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
