"""GPU: 8-bit pointwise products (torch_block.fp8_*, dcn_fp8_*) against the 64-bit oracle.

The rounding to 8 bits is exact arithmetic, so bytes (as values) and exponents must be the
oracle's. Products: each e4m3 product and its power-of-two scale are exact in fp32 and a sum of K
fp32 terms is off by at most K u of its magnitudes, u = 2^-24: |Δ| <= (K + 128) u Σ|a b| +
eps/2 |ref|, the 128 for sums over parts of K joined later and a step of the result's exponent.
That is the bound of fp32 results. bf16 results come from the 8-bit MFMA, which cuts the products
of 8 neighbouring k's below 2^-13 of the largest one's power of two (measured on the instruction
with single pairs of products): each of the other 7 loses less than 2^-13 max|a b|, so a group
loses less than 7 2^-13 of its Σ|a b|, and so does the whole sum; that is added for bf16."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import block_oracle as BO  # noqa: E402

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def tb():
    import torch_block
    return torch_block


def make(shape, dt, seed=0, spread=1.0):
    """Normal values whose magnitudes vary by 2^±(4 spread) between the elements."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(shape, generator=g) * torch.exp2(4 * spread * torch.randn(shape, generator=g))
    return v.to(dt).cuda()


def up(n):
    return -(-n // 128) * 128


def np64(t):
    return t.detach().cpu().double().numpy()


def check_blocks(v, q, e, K):
    """Bytes q [R][Kp] and exponents e [Kp/128][>= R] of v [R][K'] (oracle layout: K' = Kp)."""
    R = v.shape[0]
    want, we = BO.fp8_round(v, 1, 128)
    got = BO.e4m3_decode(q.cpu().numpy())
    assert np.array_equal(e.cpu().numpy()[:, :R].T.astype(int) - 127, we)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got), np.nan_to_num(want))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("B,C,P", [(1, 1, 1), (2, 3, 5), (1, 128, 128), (2, 127, 129), (3, 129, 127),
                                   (2, 260, 49), (2, 64, 784), (1, 1000, 77), (5, 16, 1),
                                   (1, 256, 300)])
def test_quantize(tb, dt, layout, B, C, P):
    shape = (B, C, P, 1) if layout == "nchw" else (B, P, C)
    x = make(shape, dt, seed=C + P)
    if P > 4:  # an infinity, a NaN, a block of zeros and values far below the block's largest
        f = x.view(-1)
        f[0], f[min(7, f.numel() - 1)] = float("inf"), float("nan")
        f[f.numel() // 2:f.numel() // 2 + 40] = 0.0
    q, e, qc, ec = tb.fp8_quantize(x, True, True)
    img = np64(x).reshape(B, C, P) if layout == "nchw" else np64(x).reshape(B, P, C).transpose(0, 2, 1)
    tok = np.zeros((B * P, up(C)))
    tok[:, :C] = img.transpose(0, 2, 1).reshape(B * P, C)
    check_blocks(tok, q, e, up(C))
    if layout == "nchw":
        ch = np.zeros((C, B, up(P)))
        ch[:, :, :P] = img.transpose(1, 0, 2)
        ch = ch.reshape(C, -1)
    else:
        ch = np.zeros((C, up(B * P)))
        ch[:, :B * P] = tok[:, :C].T
    check_blocks(ch, qc, ec, ch.shape[1])
    # either alone gives the same bytes
    assert torch.equal(tb.fp8_quantize(x, True, False)[0], q)
    assert torch.equal(tb.fp8_quantize(x, False, True)[2], qc)


def test_rounding_of_every_half_step(tb):
    """Every e4m3 value, the midpoints between neighbours (ties to even) and their neighbours in
    fp32, under a block maximum of 448, 1.75 * 2^k and just above it."""
    grid = np.unique(np.abs(BO.e4m3_decode(np.arange(256)))[~np.isnan(BO.e4m3_decode(np.arange(256)))])
    mid = (grid[:-1] + grid[1:]) / 2
    vals = np.concatenate([grid, mid, np.nextafter(mid.astype(np.float32), np.float32(1e9)),
                           np.nextafter(mid.astype(np.float32), np.float32(0))])
    vals = np.concatenate([vals, -vals]).astype(np.float32)
    rows = []
    for top in (448.0, np.nextafter(np.float32(448), np.float32(1e9)), 449.0, 1.75 * 2.0 ** -20,
                2.0 ** -126, 2.0 ** -140, 3e38):
        for i in range(0, len(vals), 127):
            r = np.zeros(128, np.float32)
            part = vals[i:i + 127] * np.float32(top / 448.0 if top < 1 else 1.0)
            r[:len(part)] = np.clip(part, -top, top)
            r[127] = top
            rows.append(r)
    v = torch.from_numpy(np.stack(rows)).cuda()
    q, e, _, _ = tb.fp8_quantize(v)
    check_blocks(np64(v), q, e, 128)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("O,C", [(1, 1), (5, 130), (128, 128), (127, 300), (300, 127), (640, 256)])
def test_quantize_weight(tb, dt, O, C):
    w = make((O, C), dt, seed=O)
    q, e, qt, et = tb._quantize_weight(w, True, True)
    p = np.zeros((up(O), up(C)))
    p[:O, :C] = np64(w)
    want, we = BO.fp8_round(p, 128, 128)
    assert np.array_equal(e.cpu().numpy().astype(int) - 127, we.T)
    assert np.array_equal(et.cpu().numpy().astype(int) - 127, we)
    assert np.array_equal(BO.e4m3_decode(q.cpu().numpy()), want[:O])
    assert np.array_equal(BO.e4m3_decode(qt.cpu().numpy()), want[:, :C].T)


def tok(v):
    """[tokens][channels] float64 of a map tensor."""
    v = np64(v)
    return v.reshape(*v.shape[:2], -1).transpose(0, 2, 1).reshape(-1, v.shape[1]) if v.ndim == 4 \
        else v.reshape(-1, v.shape[-1])


def by_channel(v):
    """The values of v's blocks of 128 tokens, [channels][tokens]."""
    a = np64(v)
    if a.ndim != 4:
        return BO.fp8_value(a.reshape(-1, a.shape[-1]).T, 1, 128)
    B, C = a.shape[:2]
    return np.concatenate([BO.fp8_value(a[i].reshape(C, -1), 1, 128) for i in range(B)], 1)


def close(got, a, b, dt, what):
    """got against a · bᵀ in 64 bits."""
    ref, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    half, cut = (2.0 ** -8, 7 * 2.0 ** -13) if dt == torch.bfloat16 else (0.0, 0.0)
    tol = ((a.shape[1] + 128) * U + cut) * mag + half * np.abs(ref) + 1e-37
    err = np.abs(got - ref)
    assert got.shape == ref.shape, what
    assert (err <= tol).all(), f"{what}: {(err / tol).max():.2f} x tolerance"


def run_pointwise(tb, x, w, gy, dt):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = tb.fp8_pointwise(x, w)
    assert y.dtype == dt and y.shape == gy.shape
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    xt, wq, gt = (BO.fp8_value(tok(x), 1, 128), BO.fp8_value(np64(w).reshape(w.shape[0], -1), 128, 128),
                  BO.fp8_value(tok(gy), 1, 128))
    close(tok(y), xt, wq, dt, "y")
    close(tok(gx), gt, wq.T, dt, "grad x")
    close(np64(gw).reshape(w.shape[0], -1), by_channel(gy), by_channel(x), dt, "grad w")
    return y, gx, gw


SIZES = [(1, 1, 1, 1), (1, 1, 128, 128), (1, 5, 130, 70), (2, 49, 100, 300), (3, 128, 256, 129),
         (1, 1, 1000, 500), (1, 17, 4096, 33), (2, 333, 65, 64), (1, 130, 257, 640),
         (64, 1, 40, 24), (2, 784, 256, 1024), (1, 16, 300, 2050), (1, 33, 520, 40),
         (1, 65, 128, 260), (1, 2000, 16, 16)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("B,P,C,O", SIZES)
def test_pointwise(tb, dt, layout, B, P, C, O):
    sh = lambda c: (B, c, P, 1) if layout == "nchw" else (B, P, c)
    x, w, gy = make(sh(C), dt, 1, 0.3), make((O, C), dt, 2, 0.1), make(sh(O), dt, 3, 0.3)
    y, gx, gw = run_pointwise(tb, x, w, gy, dt)
    # the same bits again, and from a kept weight
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    y2 = tb.fp8_pointwise(xr, wr)
    g2 = torch.autograd.grad(y2, (xr, wr), gy)
    assert torch.equal(y2, y) and torch.equal(g2[0], gx) and torch.equal(g2[1], gw)
    with torch.no_grad():
        assert torch.equal(tb.fp8_pointwise(x, tb.fp8_quantize_weight(w)), y)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout,B,P,C,O", [("rows", 1, 3601, 200, 3503), ("nchw", 5, 723, 129, 3330),
                                            ("nchw", 4, 900, 384, 3588), ("rows", 1, 3700, 520, 3396)])
def test_large_tiles(tb, dt, layout, B, P, C, O):
    """Results of about 200 tiles of 256 x 256 and more, with ragged edges, an odd and an even
    number of k blocks; forward only (the gradients run the same kernels)."""
    sh = lambda c: (B, c, P, 1) if layout == "nchw" else (B, P, c)
    x, w = make(sh(C), dt, 1, 0.3), make((O, C), dt, 2, 0.1)
    with torch.no_grad():
        y = tb.fp8_pointwise(x, w)
    close(tok(y), BO.fp8_value(tok(x), 1, 128), BO.fp8_value(np64(w), 128, 128), dt, "y")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (70, 300, 256), (200, 65, 1024), (300, 40, 384),
                                   (129, 131, 2304)])
@pytest.mark.parametrize("ab,bb", [(1, 1), (1, 128), (128, 1), (128, 128)])
def test_matmul_blocks(tb, dt, M, N, K, ab, bb):
    """Either operand with an exponent per row or per 128 rows, tile and few-row kernels."""
    def operand(rows, block, seed):
        v = make((rows, K), torch.float32, seed, 0.3)
        if block == 1:
            q, e, _, _ = tb.fp8_quantize(v)
        else:
            w = tb.fp8_quantize_weight(v)
            q, e = w.q, w.exponents
        return q, e, BO.fp8_value(np64(v), block, 128)

    (a, ea, va), (b, eb, vb) = operand(M, ab, 1), operand(N, bb, 2)
    close(np64(tb.fp8_matmul(a, ea, b, eb, dt)), va, vb, dt, "product")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("K", [128, 256, 384, 1152])
@pytest.mark.parametrize("ab,bb", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("M,N", [(100, 49500), (200, 49000)])
def test_wide_and_flat(tb, dt, M, N, K, ab, bb):
    """One row of tiles, at 200 x 49000 of the largest (fewer than 768 of 128 x 128), any number of
    stages; small integers, so that the sums are exact."""
    g = torch.Generator(device="cuda").manual_seed(K)
    v = [torch.randint(-4, 5, (rows, K), generator=g, device="cuda").float() for rows in (M, N)]
    ops = []
    for t, block in zip(v, (ab, bb)):
        if block == 1:
            ops += tb.fp8_quantize(t)[:2]
        else:
            w = tb.fp8_quantize_weight(t)
            ops += [w.q, w.exponents]
    assert torch.equal(tb.fp8_matmul(*ops, dt), (v[0].double() @ v[1].double().t()).to(dt))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("layout", ["nchw", "rows"])
@pytest.mark.parametrize("C,O,B,P", [(40, 24, 5, 4000), (70, 130, 3, 20001), (16, 7, 1, 60000),
                                     (300, 64, 40, 900), (64, 64, 9, 1024)])
def test_few_channels_many_tokens(tb, dt, layout, C, O, B, P):
    """Few tiles of a long K, many splits of a small result; small integers, sums exact."""
    g = torch.Generator(device="cuda").manual_seed(C)
    ints = lambda n, *s: torch.randint(-n, n + 1, s, generator=g, device="cuda").to(dt)
    sh = lambda c: (B, c, P, 1) if layout == "nchw" else (B, P, c)
    x, w, gy = ints(2, *sh(C)).requires_grad_(), ints(2, O, C).requires_grad_(), ints(1, *sh(O))
    y = tb.fp8_pointwise(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    flat = lambda t: (t[..., 0].transpose(1, 2) if layout == "nchw" else t).detach().double().reshape(B * P, -1)
    X, W, G = flat(x), w.detach().double(), flat(gy)
    assert torch.equal(flat(y), (X @ W.t()).to(dt).double())
    assert torch.equal(flat(gx), (G @ W).to(dt).double())
    assert torch.equal(gw, (G.t() @ X).to(dt))


def test_k_beyond_the_tiles_offsets(tb):
    """K above 2^22: rows too long for the 32-bit offsets of the large tiles. A few columns hold
    values, the rest is zero."""
    M, K = 3500, 2 ** 22 + 128
    cols = torch.tensor([0, 127, 128, 2 ** 21, 2 ** 22 - 1, 2 ** 22, K - 1], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    ops, vals = [], []
    for _ in range(2):
        v = torch.randint(-4, 5, (M, len(cols)), generator=g, device="cuda").float()
        q = torch.zeros(M, K, dtype=torch.uint8, device="cuda")
        q[:, cols] = v.to(torch.float8_e4m3fn).view(torch.uint8)
        ops += [q, torch.full((K // 128, -(-M // 128) * 128), 127, dtype=torch.uint8, device="cuda")]
        vals.append(v.double())
    out = tb.fp8_matmul(*ops, torch.bfloat16)
    assert torch.equal(out.double(), vals[0] @ vals[1].t())


def test_only_one_gradient(tb):
    """The gradient of one input alone is the one of both."""
    x, w = make((50, 200), torch.bfloat16, 1, 0.2), make((70, 200), torch.bfloat16, 2, 0.2)
    gy = make((50, 70), torch.bfloat16, 3, 0.2)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(tb.fp8_pointwise(xr, wr), (xr, wr), gy)
    assert torch.equal(torch.autograd.grad(tb.fp8_pointwise(xr, w), xr, gy)[0], gx)
    assert torch.equal(torch.autograd.grad(tb.fp8_pointwise(x, wr), wr, gy)[0], gw)
    assert torch.equal(torch.autograd.grad(tb.fp8_pointwise(xr, wr), wr, gy)[0], gw)


@pytest.mark.parametrize("dt", DTYPES)
def test_few_tokens_equal_many(tb, dt):
    """The first tokens of a long batch and the same tokens alone: another kernel, which rounds
    them inside the product; with weights and values that make every partial sum exact."""
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-4, 5, (300, 1000), generator=g).to(dt).cuda()
    w = torch.randint(-2, 3, (130, 1000), generator=g).to(dt).cuda()
    want = (x.double() @ w.double().t())
    for n in (1, 2, 15, 16, 17, 32, 33, 64, 65, 300):
        assert torch.equal(tb.fp8_pointwise(x[:n], w).double(), want[:n].to(dt).double())


def test_asymmetric_identity(tb):
    """Each weight row picks one channel: every output element is one input value, so a row, a
    column or an exponent out of place shows at once."""
    T, C, O = 200, 384, 300
    x = torch.arange(T * C, dtype=torch.float32).reshape(T, C) % 13 + 1
    x = (x * torch.exp2((torch.arange(T) % 9 - 4).float())[:, None] *
         torch.exp2((torch.arange(C) // 128 * 3).float())).cuda()
    pick = (torch.arange(O) * 7) % C
    w = torch.zeros(O, C)
    w[torch.arange(O), pick] = torch.exp2((torch.arange(O) // 128).float())
    y = tb.fp8_pointwise(x, w.cuda())
    want = x[:, pick.cuda()] * torch.exp2((torch.arange(O) // 128).float()).cuda()
    assert torch.equal(y, want)


@pytest.mark.parametrize("dt", DTYPES)
def test_channels_last_and_strides(tb, dt):
    x, w, gy = make((2, 70, 6, 9), dt, 1), make((50, 70, 1, 1), dt, 2, 0.1), make((2, 50, 6, 9), dt, 3)
    y, gx, gw = run_pointwise(tb, x, w, gy, dt)
    cl = torch.channels_last
    xl, wl = x.contiguous(memory_format=cl).requires_grad_(), w.clone().requires_grad_()
    yl = tb.fp8_pointwise(xl, wl)
    assert yl.is_contiguous(memory_format=cl) and torch.equal(yl, y)
    gl = torch.autograd.grad(yl, (xl, wl), gy)
    assert torch.equal(gl[0], gx) and gl[1].shape == gw.shape
    flat = make((10001,), dt, 5)[1:1 + 100 * 70].view(100, 70)
    wt = w.flatten(1).t().contiguous().t()
    with torch.no_grad():
        assert torch.equal(tb.fp8_pointwise(flat, wt), tb.fp8_pointwise(flat.clone(), w))


@pytest.mark.parametrize("T", [12, 40, 200])
@pytest.mark.parametrize("dt", DTYPES)
def test_nan_stays_in_its_row(tb, dt, T):
    x, w = make((T, 300), dt, 1), make((90, 300), dt, 2, 0.1)
    clean = tb.fp8_pointwise(x, w)
    x[7, 200], x[10, 3] = float("nan"), float("-inf")
    y = tb.fp8_pointwise(x, w)
    bad = torch.zeros(T, dtype=torch.bool)
    bad[7] = bad[10] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


def test_graph_and_side_stream(tb):
    x, w, gy = (make(s, torch.bfloat16, i, 0.2) for i, s in enumerate(((300, 520), (200, 520), (300, 200))))
    x.requires_grad_(), w.requires_grad_()

    def step():
        y = tb.fp8_pointwise(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), gy)]

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = step()
    with torch.cuda.graph(g2):
        r2 = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(1.5)
        g1.replay()
        eager = step()
        g2.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(r1, r2, eager):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_gradient_against_differences(tb):
    """The 8-bit product is piecewise constant, so differences are taken of the oracle: with
    inputs that e4m3 holds exactly, the gradients are the exact bilinear form's."""
    g = torch.Generator().manual_seed(4)
    x = torch.randint(-8, 9, (70, 140), generator=g).float().cuda().requires_grad_()
    w = torch.randint(-8, 9, (60, 140), generator=g).float().cuda().requires_grad_()
    gy = torch.randint(-8, 9, (70, 60), generator=g).float().cuda()
    y = tb.fp8_pointwise(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    xd, wd, gd = x.detach().double(), w.detach().double(), gy.double()
    f = lambda a, b: float(((a @ b.t()) * gd).sum())
    assert torch.equal(y.double(), xd @ wd.t())
    for i, j in ((0, 0), (13, 139), (69, 70)):
        d = torch.zeros_like(xd)
        d[i, j] = 1.0
        assert float(gx[i, j]) == (f(xd + d, wd) - f(xd - d, wd)) / 2
    for i, j in ((0, 0), (59, 139), (31, 128)):
        d = torch.zeros_like(wd)
        d[i, j] = 1.0
        assert float(gw[i, j]) == (f(xd, wd + d) - f(xd, wd - d)) / 2


def test_refusals_and_modules(tb):
    x, w = make((4, 10), torch.float32), make((6, 10), torch.float32)
    for bad in (w.bfloat16(), w[:, :9], w.cpu(), w[None]):
        with pytest.raises(ValueError):
            tb.fp8_pointwise(x, bad)
    with pytest.raises(TypeError):
        tb.fp8_pointwise(x.half(), w)
    with pytest.raises(RuntimeError):
        tb.fp8_pointwise(x.cpu(), w)
    qw = tb.fp8_quantize_weight(w)
    with pytest.raises(RuntimeError):
        tb.fp8_pointwise(x.clone().requires_grad_(), qw)
    with pytest.raises(ValueError):
        tb.fp8_pointwise(make((4, 11), torch.float32), qw)
    with pytest.raises(ValueError):
        tb.Fp8Weight(qw.q, qw.exponents, 200)
    q, e, _, _ = tb.fp8_quantize(x)
    for args in ((q, e, q[:, :64], e), (q, e[:, :4], q, e), (q.int(), e, q, e), (q, e, q.cpu(), e)):
        with pytest.raises(ValueError):
            tb.fp8_matmul(*args)
    with pytest.raises(ValueError):
        tb.fp8_quantize_weight(x[0])
    assert tb.fp8_pointwise(x[:0], w).shape == (0, 6)
    assert tb.fp8_pointwise(make((2, 10, 3, 0), torch.float32), w).shape == (2, 6, 3, 0)
    e = x[:0].requires_grad_()
    wr = w.clone().requires_grad_()
    tb.fp8_pointwise(e, wr).sum().backward()
    assert not wr.grad.any() and e.grad.shape == (0, 10)
    m = tb.Fp8Pointwise(10, 6).cuda()
    y = m(x)
    y.sum().backward()
    assert m.weight.grad is not None
    with torch.no_grad():
        assert torch.equal(m.eval().serve()(x), y)
        m.load_state_dict({"weight": m.weight * 2})
        assert torch.equal(m(x), y * 2)
        m.serve().bfloat16()
        assert m.weight8 is None
    assert m.eval().serve().train().weight8 is None
    m.serve()  # a call that wants the weight's gradient gets it
    m.weight.grad = None
    m(x.to(m.weight.dtype)).sum().backward()
    assert m.weight.grad is not None
    for bad in (x[0, 0], x[:, :0]):
        with pytest.raises(ValueError):
            tb.fp8_pointwise(bad, w)
        with pytest.raises(ValueError):
            tb.fp8_quantize(bad)


@pytest.mark.parametrize("layout", ["nchw", "rows"])
def test_more_than_2_31_elements(tb, layout):
    """Small integers, so that every product and sum is exact whatever its order."""
    C, O = 2048, 130
    n = 1_050_001
    x = torch.randint(-2, 3, (3, C, 1000, 351) if layout == "nchw" else (n, C), device="cuda",
                      dtype=torch.int8).float()
    g = torch.Generator().manual_seed(1)
    w = torch.randint(-2, 3, (O, C), generator=g).float().cuda()
    assert x.numel() > 2 ** 31
    x.requires_grad_(), w.requires_grad_()
    y = tb.fp8_pointwise(x, w)
    gy = torch.randint(-1, 2, y.shape, device="cuda", dtype=torch.int8).float()
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    tok = lambda t: t.detach().permute(0, 2, 3, 1).flatten(0, 2) if layout == "nchw" else t.detach()
    x, y, gy, gx, w = tok(x), tok(y), tok(gy), tok(gx), w.detach().double()
    want = torch.zeros(O, C, dtype=torch.float64, device="cuda")
    for i in range(0, x.shape[0], 150_000):
        part = slice(i, i + 150_000)
        a, b = x[part].double().contiguous(), gy[part].double().contiguous()
        assert torch.equal(y[part].double(), a @ w.t()), i
        assert torch.equal(gx[part].double(), b @ w), i
        want += b.t() @ a
    assert torch.equal(gw.double(), want)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T", [8, 300])
@pytest.mark.parametrize("p", [-110, -118, -124, -126, -130, -134])
def test_smallest_values(tb, dt, T, p):
    """Blocks near the smallest exponent against a large weight: fp32 results take the values to
    multiples of 2^-133 (half of one off), bf16 results as they are."""
    g = torch.Generator().manual_seed(0)
    x = (torch.rand((T, 256), generator=g) + 0.5) * \
        torch.exp2(torch.randint(-8, 1, (T, 256), generator=g).float() + p)
    x, w = x.to(dt), (torch.rand((200, 256), generator=g) * 2.0 ** 90).to(dt)
    got = np64(tb.fp8_pointwise(x.cuda(), w.cuda()))
    a, b = BO.fp8_value(np64(x), 1, 128), BO.fp8_value(np64(w), 128, 128)
    if dt == torch.bfloat16:
        return close(got, a, b, dt, "y")
    ref, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    tol = (256 + 128) * U * mag + 2.0 ** -134 * np.abs(b).sum(1)
    assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("T", [8, 300])
def test_largest_values(tb, T):
    """The type's largest magnitude is worth 2^128 in e4m3 (its neighbour below it is 240 / 256 of
    that): infinite in fp32's products, finite in bf16's; what rounds down stays finite in both."""
    w = torch.eye(128)[:100] * 0.25
    x = torch.full((T, 128), torch.finfo(torch.float32).min)
    y = tb.fp8_pointwise(x.cuda(), w.cuda())
    assert not bool(torch.isfinite(y[:, :100]).any())
    x = torch.full((T, 128), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16)
    y = tb.fp8_pointwise(x.cuda(), w.bfloat16().cuda())
    assert bool((y == -2.0 ** 126).all())
    for dt in DTYPES:
        x = torch.full((T, 128), -247.0 * 2.0 ** 120, dtype=dt)
        assert bool((tb.fp8_pointwise(x.cuda(), w.to(dt).cuda()) == -240.0 * 2.0 ** 118).all())
