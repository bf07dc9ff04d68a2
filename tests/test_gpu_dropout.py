"""GPU: dropout (torch_block.dropout, dcn_dropout_*) against the 64-bit oracle.

Tolerances: t = x * s takes two fp32 roundings (s itself and the product), r + t one more, the
store to the tensor's type one: |Δ| <= 2^-24 (2 |t| + |y|) + eps/2 |y|, the higher-order terms
covered by a factor 1.01. Which elements are dropped must agree exactly."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import block_oracle as BO  # noqa: E402

SEED, OFF = 0x9E3779B97F4A7C15, 0x0123456789ABCDEF


@pytest.fixture(scope="module")
def tb():
    import torch_block
    return torch_block


def make(shape, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dt).cuda()


def group_of(shape, group):
    n = int(np.prod(shape))
    return {"element": 1, "channel": int(np.prod(shape[2:])), "image": n // max(shape[0], 1)}.get(
        group, group)


def check(y, x, p, group, residual=None, seed=SEED, off=OFF):
    f = torch.from_numpy(BO.drop_factor(x.numel(), group, p, seed, off)).reshape(x.shape)
    t = x.cpu().double() * f
    t = torch.where(f == 0, torch.zeros((), dtype=torch.float64), t)
    ref = t if residual is None else residual.cpu().double() + t
    eps = torch.finfo(x.dtype).eps / 2 if x.dtype == torch.bfloat16 else 0.0
    tol = 1.01 * (2.0 ** -24 * (2 * t.abs() + ref.abs()) + eps * ref.abs())
    err = (y.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    if residual is None:
        assert torch.equal(y.cpu() == 0, (ref == 0))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,group", [
    ((1, 1), "element"), ((7,), 1), ((8,), 1), ((9,), 1), ((3, 5, 7, 11), "element"),
    ((4, 16, 28, 28), "element"), ((3, 5, 7, 7), "channel"), ((5, 3, 7, 9), "image"),
    ((2, 33, 1, 1), "channel"), ((64, 3), "image"), ((1, 4099), 3), ((1, 4099), 13),
    ((2, 70, 3, 3), "channel"), ((1, 100003), 99991), ((17, 1023), 1023)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_forward_backward(tb, dt, shape, group, p):
    x, r, gy = make(shape, dt).requires_grad_(), make(shape, dt, 1).requires_grad_(), \
        make(shape, dt, 2)
    n = group_of(shape, group)
    y = tb.dropout(x, p, (SEED, OFF), group=group)
    check(y.detach(), x.detach(), p, n)
    gx, = torch.autograd.grad(y, x, gy)
    check(gx, gy, p, n)
    y = tb.dropout(x, p, (SEED, OFF), group=group, residual=r)
    check(y.detach(), x.detach(), p, n, r.detach())
    gx, gr = torch.autograd.grad(y, (x, r), gy)
    check(gx, gy, p, n)
    assert torch.equal(gr, gy)


@pytest.mark.parametrize("p,kept", [(0.0, True), (1.0, False), (2.0 ** -18, True)])
def test_probability_ends(tb, p, kept):
    x = make((3, 1000), torch.float32)
    y = tb.dropout(x, p, (1, 2))
    assert torch.equal(y, x if kept else torch.zeros_like(x))


def test_dropped_nan_is_zero(tb):
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    y = tb.dropout(x, 0.5, (SEED, OFF)).cpu()
    f = torch.from_numpy(BO.drop_factor(4096, 1, 0.5, SEED, OFF))
    assert torch.equal(y == 0, f == 0)
    assert torch.equal(torch.isnan(y), (f != 0) & torch.isnan(x.cpu()))


def test_draws_beyond_32_bits(tb):
    """Elements past 2^32 draw from their own counters: a group of one element, the tail of a
    2^32 + 40 element tensor (bf16, 8.6 GB)."""
    n = (1 << 32) + 40
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = tb.dropout(x, 0.5, (SEED, OFF))
    tail = y[-80:].cpu().double().numpy()
    want = np.where(BO.draws(n - 80, 80, SEED, OFF) < 32768, 0.0, 2.0)
    assert np.array_equal(tail, want)
    del x, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(tb, dt):
    """Transposed, sliced at an odd element, expanded and channels-last inputs give the bits of
    their contiguous copies."""
    base = make((6, 10, 14, 18), dt)
    flat = make((10001,), dt)
    for x in (base.transpose(1, 3), flat[1:], flat[3:4000], base[:, :1].expand(6, 10, 14, 18),
              base.contiguous(memory_format=torch.channels_last), base[::2, 1::3]):
        a, b = (tb.dropout(t, 0.3, (5, 6), group="element") for t in (x, x.contiguous()))
        assert torch.equal(a, b)


def test_in_place_through_the_c_entry(tb):
    import dcn_runtime as rt
    x = make((5000,), torch.bfloat16)
    want = tb.dropout(x, 0.25, (9, 9))
    d = rt.DropoutDesc(5000, 1, 9, 9, rt.DCN_BF16, 0.25)
    y = x.clone()
    tb._call(y.device, "dcn_dropout_fwd", d, y.data_ptr(), None, y.data_ptr(), None)
    assert torch.equal(y, want)


def test_rng_tensor_and_graph(tb):
    """A device rng gives the host rng's bits; a captured step draws anew when it is updated,
    forward and backward from the same draws, with eager work between the replays."""
    x, gy = make((3, 999), torch.float32).requires_grad_(), make((3, 999), torch.float32, 1)
    rng = torch.tensor([11, 5], dtype=torch.int64, device="cuda")
    assert torch.equal(tb.dropout(x, 0.4, rng), tb.dropout(x, 0.4, (11, 5)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(tb.dropout(x, 0.4, rng), x, gy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = tb.dropout(x, 0.4, rng)
        gx, = torch.autograd.grad(y, x, gy)
    for off in (5, 6, 7, 5):
        rng.copy_(torch.tensor([11, off]))
        g.replay()
        eager = tb.dropout(x.detach(), 0.4, (11, off))
        assert torch.equal(y.detach(), eager)
        assert torch.equal(gx, tb.dropout(gy, 0.4, (11, off)))
        torch.cuda.synchronize()
    assert not torch.equal(tb.dropout(x, 0.4, (11, 6)), tb.dropout(x, 0.4, (11, 5)))


def test_rng_changed_before_backward_is_refused(tb):
    x = make((64,), torch.float32).requires_grad_()
    rng = torch.tensor([1, 2], dtype=torch.int64, device="cuda")
    y = tb.dropout(x, 0.5, rng)
    rng.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_side_stream(tb):
    x = make((1 << 20,), torch.float32)
    want = tb.dropout(x, 0.5, (3, 4))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tb.dropout(x * 1.0, 0.5, (3, 4))
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(tb):
    x = make((4, 4), torch.float32)
    with pytest.raises(TypeError):
        tb.dropout(x.half(), 0.5, (1, 2))
    with pytest.raises(RuntimeError):
        tb.dropout(x.cpu(), 0.5, (1, 2))
    with pytest.raises(ValueError):
        tb.dropout(x, 1.5, (1, 2))
    with pytest.raises(ValueError):
        tb.dropout(x, 0.5, None)
    with pytest.raises(ValueError):
        tb.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        tb.dropout(x, 0.5, (1, 2), residual=x[:2])
    with pytest.raises(ValueError):
        tb.dropout(x[0], 0.5, (1, 2), group="channel")


def test_modules(tb):
    x = make((8, 4, 5, 5), torch.float32)
    m = tb.Dropout(0.5)
    torch.manual_seed(3)
    a = m(x)
    torch.manual_seed(3)
    assert torch.equal(a, m(x)) and not torch.equal(a, m(x))
    m.eval()
    assert m(x) is x and torch.equal(m(x, x), x + x)
    y = tb.DropPath(0.5)(torch.ones(64, 3, 2, 2, device="cuda"))
    assert set(y.flatten(1).unique(dim=1).flatten().tolist()) == {0.0, 2.0}
    assert tb.dropout(x[:0], 0.5, (1, 2)).shape == (0, 4, 5, 5)
