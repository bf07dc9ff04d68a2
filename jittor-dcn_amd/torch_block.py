"""What stands around a DeformConv2d in a residual block, for PyTorch callers: libdcn's
block operators (include/dcn.h, "residual block around a DeformConv2d") as autograd functions
and modules.

The reference's network is DeformConv2d + BatchNorm + ReLU (train.py:304-337); blocks of
larger networks put norms over the channels, gates, residual scales, dropout and pointwise
products around the operator. Everything here runs on torch's current stream of the tensors'
device in libdcn's kernels, takes float32 and bfloat16 CUDA tensors of any strides (copied to
a dense layout where they have another), and has no CPU fallback.

Random numbers are arguments: `rng` is (seed, offset), or an int64 CUDA tensor of those two
that is read when the kernel runs (a captured graph then draws a new mask per replay when the
tensor is updated between replays). The backward draws the same mask again.

Forward and backward may be captured into a graph. As with every torch operator, let go of the
results of earlier eager passes over the same leaf tensors (and of their losses) first: a leaf's
accumulation node lives as long as a graph that holds it and stays on the stream it was made on.
Refused are forward-mode derivatives (there are none), torch.jit.trace and make_fx.
"""
from __future__ import annotations

import ctypes
import functools
import threading

import torch
import torch.autograd.forward_ad as forward_ad
from torch.autograd.function import once_differentiable

import dcn_runtime as rt

_DT = {torch.float32: rt.DCN_F32, torch.bfloat16: rt.DCN_BF16}
_handles = {}
_lock = threading.Lock()  # a handle takes one caller at a time: stream and launch belong together
_fns = {}
_is_tracing, _mode = torch._C._is_tracing, torch._C._get_dispatch_mode
_PROXY = torch._C._TorchDispatchModeKey.PROXY  # the mode under which torch.fx's make_fx records


def _fn(name):
    """The entry point, bound so that the call keeps the GIL: these calls only enqueue, and
    giving the GIL up and taking it back around each costs more than the call itself (a
    backward runs beside the thread that waits for it)."""
    f = _fns.get(name)
    if f is None:
        lib = rt.load()
        f = getattr(ctypes.PyDLL(lib._name, handle=lib._handle), name)
        f.argtypes, f.restype = rt.SIGNATURES[name], ctypes.c_int
        _fns[name] = f
    return f


def _call(dev: torch.device, name: str, *args):
    """One libdcn call on torch's current stream of `dev`, whatever device is current."""
    if _is_tracing() or _mode(_PROXY) is not None:
        raise RuntimeError("torch_block's calls cannot be traced: a trace would keep their empty "
                           "results, or their sizes for tensors of others (capture a graph)")
    idx = dev.index
    if idx != torch._C._cuda_getDevice():
        with torch.cuda.device(idx):
            return _call(dev, name, *args)
    stream = torch._C._cuda_getCurrentRawStream(idx)
    with _lock:
        h = _handles.get(idx)
        if h is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"torch_block: make one call on cuda:{idx} before capturing "
                                   "(the library's handle is created by the first)")
            h = _handles[idx] = rt.Handle(idx)
            h.bound = None
        if h.bound != stream:
            h.set_stream(stream)
            h.bound = stream
        rc = _fn(name)(h.h, *args)
    if rc:
        rt.check(rc, name)


def _wants_grad(*tensors):
    """Autograd has to see the call: for a gradient, or inside a forward-mode level, where it refuses
    a tensor with a tangent (there are no forward-mode derivatives)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _number(v, what):
    """v as it is now, as a float: the library takes numbers, and descriptors are kept by them."""
    if type(v) is float:
        return v
    if isinstance(v, torch.Tensor):
        if v.requires_grad and torch.is_grad_enabled():
            raise TypeError(f"{what} is a number, which gets no gradient (a learnable factor per "
                            "channel is block_norm's scale)")
        v = v.detach()
    return float(v)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dtype(x: torch.Tensor, what: str) -> int:
    if x.dtype not in _DT:
        raise TypeError(f"{what} takes float32 or bfloat16 tensors, not {x.dtype}")
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on the GPU only; the tensor is on {x.device}")
    return _DT[x.dtype]


def _same(x, t, what, name, shape=None):
    """t is of x's dtype, on its device, and of `shape` (None: x's)."""
    if t is None:
        return
    shape = x.shape if shape is None else shape
    if t.shape != shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what}: {name} must be {tuple(shape)} {x.dtype} on {x.device}, not "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


def _rng(rng, dev, what):
    """(seed, offset, device tensor or None) of an rng argument."""
    if isinstance(rng, torch.Tensor):
        if rng.dtype not in (torch.int64, torch.uint64) or rng.numel() != 2 or \
                rng.device != dev or not rng.is_contiguous():
            raise ValueError(f"{what}: rng must be 2 contiguous int64 on {dev}")
        return 0, 0, rng
    if rng is None:
        raise ValueError(f"{what}: rng = (seed, offset) is needed where p > 0")
    seed, offset = rng
    mask = (1 << 64) - 1
    return int(seed) & mask, int(offset) & mask, None


def _fresh_rng(rng):
    """The rng of a module's call: its own tensor, or a new seed from torch's generator."""
    if rng is not None:
        return rng
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a captured dropout needs an rng tensor (its seed would be frozen)")
    return int(torch.randint(1 << 62, ()).item()), 0


def _ints(what, *sizes):
    """The entry points count in 32-bit integers."""
    if max(sizes) > 0x7fffffff:
        raise ValueError(f"{what}: a size above 2^31 - 1")


# ---------------------------------------------------------------------------- dropout
def _drop(x, residual, p, rng, group):
    seed, offset, dev_rng = _rng(rng, x.device, "dropout") if p > 0 else (0, 0, None)
    d = rt.DropoutDesc(x.numel(), group, seed, offset, _DT[x.dtype], p)
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    y = torch.empty_like(x)
    if d.n:
        _call(x.device, "dcn_dropout_fwd", d, _ptr(x), _ptr(residual), _ptr(y), _ptr(dev_rng))
    return y, d, dev_rng


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, group):
        y, ctx.desc, dev_rng = _drop(x, residual, p, rng, group)
        ctx.save_for_backward(dev_rng)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        gx = None
        if ctx.needs_input_grad[0]:
            dev_rng, = ctx.saved_tensors
            g = gy.contiguous()
            gx = torch.empty_like(g)
            if g.numel():
                _call(g.device, "dcn_dropout_bwd", ctx.desc, _ptr(g), _ptr(gx), _ptr(dev_rng))
        return gx, gy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, rng, group="element", residual=None):
    """residual + drop(x), or drop(x): each draw of `group` elements is zeroed with
    probability p and scaled by 1 / (1 - p) otherwise (p to the nearest 1/65536).

    group: "element"; "channel", one draw per x[b, c] (whole maps of an NCHW tensor); "image",
    one per x[b] (stochastic depth); or a number of neighbouring elements. Elements count in
    x's logical order, whatever its strides."""
    _dtype(x, "dropout")
    _same(x, residual, "dropout", "residual")
    p = _number(p, "dropout: p")
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout: p must be between 0 and 1")
    if isinstance(group, str):
        skip = {"element": x.dim(), "channel": 2, "image": 1}.get(group)
        if skip is None or x.dim() < min(skip, 2):
            raise ValueError(f"dropout: group {group!r} does not fit a {x.dim()}-d tensor")
        group = 1
        for s in x.shape[skip:]:
            group *= s
    if group != int(group) or (group < 1 and x.numel()):
        raise ValueError("dropout: group must be a whole number of elements")
    args = (x, residual, p, rng, max(min(int(group), x.numel()), 1))  # (all of them: one draw)
    return _Dropout.apply(*args) if _wants_grad(x, residual) else _drop(*args)[0]


class Dropout(torch.nn.Module):
    """dropout() in training, x (+ residual) in evaluation. Each call draws a new seed from
    torch's generator, unless `rng` (an int64 CUDA tensor the caller advances) is given."""

    def __init__(self, p=0.5, group="element", rng=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError("Dropout: p must be between 0 and 1")
        self.p, self.group, self.rng = p, group, rng

    def forward(self, x, residual=None):
        if not self.training or self.p == 0:
            return x if residual is None else residual + x
        return dropout(x, self.p, _fresh_rng(self.rng), self.group, residual)


class DropPath(Dropout):
    """Stochastic depth: one draw per image."""

    def __init__(self, p=0.1, rng=None):
        super().__init__(p, "image", rng)


# ---------------------------------------------------------------------------- block norms
_NORM = {None: rt.DCN_NORM_NONE, "rms": rt.DCN_NORM_RMS, "layer": rt.DCN_NORM_LAYER}
_ACT = {"linear": rt.DCN_ACT_LINEAR, "sigmoid": rt.DCN_ACT_SIGMOID, "silu": rt.DCN_ACT_SILU}


def _layout(x):
    """(layout, B, C, P, memory format) of a map tensor: [B, C, H, W] (channels-last memory
    stays channels-last) or token rows [..., C]."""
    if x.dim() == 0 or x.shape[1 if x.dim() == 4 else -1] == 0:
        raise ValueError("torch_block: a tensor without channels")
    if x.dim() == 4:
        B, C, H, W = x.shape
        _ints("a map tensor", B, C, H * W)
        if not x.is_contiguous() and x.is_contiguous(memory_format=torch.channels_last):
            return rt.DCN_NHWC, B, C, H * W, torch.channels_last
        return rt.DCN_NCHW, B, C, H * W, torch.contiguous_format
    C = x.shape[-1]
    B = x.shape[0] if x.dim() > 2 else 1
    P = x.numel() // max(B * C, 1)
    _ints("token rows", B, C, P)
    return rt.DCN_NHWC, B, C, P, torch.contiguous_format


@functools.lru_cache(maxsize=1024)
def _block_desc(*fields):
    """The descriptor of a call without dropout (not written to by anyone)."""
    return rt.BlockDesc(*fields)


@functools.lru_cache(maxsize=1024)
def _block_ws(*geometry):
    """Bytes of workspace of a backward, by the descriptor's fields up to `gate`."""
    nbytes = ctypes.c_size_t()
    rt.check(_fn("dcn_block_norm_workspace")(rt.BlockDesc(*geometry), nbytes),
             "dcn_block_norm_workspace")
    return nbytes.value


def _dense(t, mf):
    return t if t is None else t.contiguous(memory_format=mf)


def _block(tensors, desc, mf, dev_rng, keep=False):
    """(out, y), the dense tensors behind them and, with keep, the norms' statistics."""
    x, residual, gate, *vectors = tensors
    x, residual = _dense(x, mf), _dense(residual, mf)
    gate = _dense(gate, mf if desc.gate == rt.DCN_GATE_FULL else torch.contiguous_format)
    tensors = (x, residual, gate, *[t if t is None else t.contiguous() for t in vectors])
    ref = residual if x is None else x
    out = None if x is None else torch.empty_like(x)  # as dense as x: in its memory format
    y = torch.empty_like(ref) if desc.pre else None
    stats = None
    if ref.numel():
        if keep and (desc.post or desc.pre):
            stats = torch.empty(4 * desc.B * desc.P, dtype=torch.float32, device=ref.device)
        _call(ref.device, "dcn_block_norm_fwd", desc,
              rt.BlockIO(*[t if t is None else t.data_ptr()
                           for t in (*tensors, dev_rng, out, y)], stats=_ptr(stats)))
    return out, y, tensors, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, desc, mf, dev_rng, *tensors):
        out, y, tensors, stats = _block(tensors, desc, mf, dev_rng, keep=True)
        ctx.desc, ctx.mf = desc, mf
        ctx.save_for_backward(*tensors, dev_rng, stats)
        ctx.set_materialize_grads(False)
        return out, y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_y):
        *inputs, dev_rng, stats = ctx.saved_tensors
        need = ctx.needs_input_grad[3:]
        if grad_out is None and grad_y is None:
            return (None,) * 11
        mf, d = ctx.mf, ctx.desc
        grad_out, grad_y = _dense(grad_out, mf), _dense(grad_y, mf)
        ref = inputs[0] if inputs[0] is not None else inputs[1]
        if not ref.numel():
            return (None, None, None,
                    *(torch.zeros_like(t) if n else None for t, n in zip(inputs, need)))
        grads = [torch.empty_like(t) if n else None for t, n in zip(inputs, need)]
        nbytes = _block_ws(d.B, d.C, d.P, d.layout, d.dtype, d.post, d.pre, d.gate)
        ws = _bytes(ref.device, nbytes)
        io = rt.BlockIO(*[t if t is None else t.data_ptr() for t in (
            *inputs, dev_rng, None, None, grad_out, grad_y, *grads, stats)])
        _call(ref.device, "dcn_block_norm_bwd", d, io, ws.data_ptr(), nbytes)
        return (None, None, None, *grads)


def block_norm(x=None, residual=None, *, gate=None, gate_act="linear", scale=None, alpha=1.0,
               post=None, post_weight=None, post_bias=None, pre=None, pre_weight=None,
               pre_bias=None, eps=1e-6, drop_p=0.0, drop="element", rng=None):
    """The operator between two residual blocks: returns (out, y),

        t = dropout(alpha * scale * act(gate) * N_post(x));  out = residual + t;  y = N_pre(out)

    with the norms over the channels: dim 1 of a 4-d tensor (NCHW, or channels-last memory as
    it is), else the last. post / pre: None, "rms" or "layer" (None: no norm after the block;
    no y); eps: one number, or (post, pre). gate: of x's shape, or [B, C] for one per image
    and channel, through gate_act "linear", "sigmoid" or "silu". scale, *_weight, *_bias: [C].
    drop: "element" (elements count in memory order) or "image", one draw per x[b] (stochastic
    depth; a row of a 2-d tensor, as in dropout). Without a residual out = t; without x the
    operator is the pre norm alone and out is the residual. All tensors have x's dtype;
    everything but the rounding of the results is fp32. alpha, eps and drop_p are numbers: a
    tensor there counts with its value at the call, and one that wants a gradient is refused."""
    ref = residual if x is None else x
    if ref is None:
        raise ValueError("block_norm: neither x nor a residual")
    dt = _dtype(ref, "block_norm")
    if post not in _NORM or pre not in _NORM or gate_act not in _ACT:
        raise ValueError("block_norm: norms are None, 'rms' or 'layer'; gate_act is 'linear', "
                         "'sigmoid' or 'silu'")
    drop_p = _number(drop_p, "block_norm: drop_p")
    if drop not in ("element", "image") or not 0.0 <= drop_p <= 1.0:
        raise ValueError("block_norm: drop is 'element' or 'image' and 0 <= drop_p <= 1")
    layout, B, C, P, mf = _layout(ref)
    if drop == "image" and drop_p > 0 and ref.dim() == 2:  # an image of one position per row
        if gate is not None and gate.shape == (1, C):
            gate = gate.expand(ref.shape)
        B, P = P, 1
    kind = rt.DCN_GATE_NONE
    if gate is not None:
        image = gate.dim() == 2 and tuple(gate.shape) == (B, C) and gate.shape != ref.shape
        kind = rt.DCN_GATE_IMAGE if image else rt.DCN_GATE_FULL
        _same(ref, gate, "block_norm", "gate", (B, C) if image else None)
    if x is not None:
        _same(x, residual, "block_norm", "residual")
    shape = (C,)
    _same(ref, scale, "block_norm", "scale", shape)
    _same(ref, post_weight, "block_norm", "post_weight", shape)
    _same(ref, post_bias, "block_norm", "post_bias", shape)
    _same(ref, pre_weight, "block_norm", "pre_weight", shape)
    _same(ref, pre_bias, "block_norm", "pre_bias", shape)
    e1, e2 = eps if isinstance(eps, (tuple, list)) else (eps, eps)
    fields = (B, C, P, layout, dt, _NORM[post], _NORM[pre], kind, _ACT[gate_act],
              _number(e1, "block_norm: eps"), _number(e2, "block_norm: eps"),
              _number(alpha, "block_norm: alpha"))
    dev_rng = None
    if drop_p > 0:
        seed, offset, dev_rng = _rng(rng, ref.device, "block_norm")
        desc = rt.BlockDesc(*fields, drop_p, int(drop == "image"), seed, offset)
    else:
        desc = _block_desc(*fields)
    tensors = (x, residual, gate, scale, post_weight, post_bias, pre_weight, pre_bias)
    if _wants_grad(*tensors):
        out, y = _BlockNorm.apply(desc, mf, dev_rng, *tensors)
    else:
        out, y, _, _ = _block(tensors, desc, mf, dev_rng)
    return (residual if x is None else out), y


class BlockNorm(torch.nn.Module):
    """block_norm() with its parameters: (x, residual, gate=None) -> (out, y).

    post / pre: None, "rms" (weight) or "layer" (weight and bias); layer_scale: the residual
    scale's initial value per channel, or None for no scale; alpha: a fixed factor; drop_p:
    dropout of the block's result in training, per element or per image ("image": stochastic
    depth), seeded like Dropout."""

    def __init__(self, channels, post="rms", pre="rms", layer_scale=None, alpha=1.0, gate_act="linear",
                 drop_p=0.0, drop="element", eps=1e-6, rng=None):
        super().__init__()
        self.channels, self.post, self.pre, self.alpha, self.gate_act = (channels, post, pre,
                                                                         alpha, gate_act)
        self.drop_p, self.drop, self.eps, self.rng = drop_p, drop, eps, rng

        def vec(on, value):
            return torch.nn.Parameter(torch.full((channels,), float(value))) if on else None

        self.scale = vec(layer_scale is not None, layer_scale or 0.0)
        self.post_weight, self.post_bias = vec(post, 1.0), vec(post == "layer", 0.0)
        self.pre_weight, self.pre_bias = vec(pre, 1.0), vec(pre == "layer", 0.0)

    def forward(self, x, residual=None, gate=None):
        p = self.drop_p if self.training else 0.0
        return block_norm(x, residual, gate=gate, gate_act=self.gate_act, scale=self.scale,
                          alpha=self.alpha, post=self.post, post_weight=self.post_weight,
                          post_bias=self.post_bias, pre=self.pre, pre_weight=self.pre_weight,
                          pre_bias=self.pre_bias, eps=self.eps, drop_p=p, drop=self.drop,
                          rng=_fresh_rng(self.rng) if p > 0 else None)


# ---------------------------------------------------------------------------- 8-bit products
def _up(n, m=128):
    return (n + m - 1) // m * m


def _bytes(dev, *shape):
    return torch.empty(shape, dtype=torch.uint8, device=dev)


class Fp8Weight:
    """A weight [O, C] kept in 8 bits: q [O, C up to 128s] e4m3 bytes and exponents
    [C / 128, O / 128] (each up; bias 127), one per 128 x 128 block (include/dcn.h). What a
    server keeps instead of the weight; fp8_quantize_weight makes one."""

    def __init__(self, q, exponents, in_features):
        O, C = q.shape[0], int(in_features)
        for t, shape in ((q, (O, _up(C))), (exponents, (_up(C) // 128, -(-O // 128)))):
            if t.dtype != torch.uint8 or not t.is_cuda or tuple(t.shape) != shape or \
                    t.device != q.device:
                raise ValueError(f"Fp8Weight: expected uint8 {shape} on a GPU, not "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        self.q, self.exponents = _at16(q), _at16(exponents)
        self.out_features, self.in_features = O, C


def _at16(t):
    """Dense and 16-byte aligned (a slice of a larger buffer may not be)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _quantize_weight(w, plain, transposed):
    O, C = w.shape
    w, dev = w.contiguous(), w.device
    q = e = qt = et = None
    if plain:
        q, e = _bytes(dev, O, _up(C)), _bytes(dev, _up(C) // 128, -(-O // 128))
    if transposed:
        qt, et = _bytes(dev, C, _up(O)), _bytes(dev, _up(O) // 128, -(-C // 128))
    _call(dev, "dcn_fp8_quantize_weight", O, C, _DT[w.dtype], _ptr(w), _ptr(q), _ptr(e),
          _ptr(qt), _ptr(et))
    return q, e, qt, et


def fp8_quantize_weight(w):
    """Fp8Weight of a float32 or bfloat16 weight [O, C] (or [O, C, 1, 1])."""
    _dtype(w, "fp8_quantize_weight")
    if w.dim() == 4 and w.shape[2:] == (1, 1):
        w = w.flatten(1)
    if w.dim() != 2 or not w.numel():
        raise ValueError(f"fp8_quantize_weight: a weight is [O, C], not {tuple(w.shape)}")
    _ints("fp8_quantize_weight", *w.shape)
    q, e, _, _ = _quantize_weight(w.detach(), True, False)
    return Fp8Weight(q, e, w.shape[1])


def fp8_quantize(x, tokens=True, channels=False):
    """(bytes, exponents, bytes, exponents) of a map tensor by token and by channel (None where
    not wanted), in the layouts of dcn_fp8_quantize (include/dcn.h)."""
    dt = _dtype(x, "fp8_quantize")
    layout, B, C, P, mf = _layout(x)
    if not x.numel():
        raise ValueError("fp8_quantize: an empty tensor")
    x, T, dev = x.contiguous(memory_format=mf), B * P, x.device
    kt = B * _up(P) if layout == rt.DCN_NCHW else _up(T)
    q = e = qc = ec = None
    if tokens:
        q, e = _bytes(dev, T, _up(C)), _bytes(dev, _up(C) // 128, _up(T))
    if channels:
        qc, ec = _bytes(dev, C, kt), _bytes(dev, kt // 128, _up(C))
    _call(dev, "dcn_fp8_quantize", rt.Fp8Desc(B, C, P, layout, dt), _ptr(x), _ptr(q), _ptr(e),
          _ptr(qc), _ptr(ec))
    return q, e, qc, ec


def fp8_matmul(a, a_exponents, b, b_exponents, dtype=torch.float32):
    """a · bᵀ of two matrices in 8 bits (fp8_quantize's or Fp8Weight's layouts; either may have
    an exponent per row or per 128 rows), as [a's rows, b's rows] of `dtype`. float32: products and
    sums in 32 bits. bfloat16: by the 8-bit matrix instruction, whose sums keep 13 bits below the
    largest product of each 8 neighbouring k's (off by up to 8.5e-4 of Σ|a b|; include/dcn.h); where
    that matters, take float32 and round it."""
    if dtype not in _DT:
        raise TypeError(f"fp8_matmul gives float32 or bfloat16, not {dtype}")
    K, blocks = a.shape[-1], []
    for t, e in ((a, a_exponents), (b, b_exponents)):
        if t.dim() != 2 or t.shape[1] != K or K % 128 or t.dtype != torch.uint8 or not t.is_cuda:
            raise ValueError("fp8_matmul: operands are uint8 [rows, K] on a GPU, K a multiple of 128")
        rows = t.shape[0]
        shape = {(K // 128, _up(rows)): 1, (K // 128, -(-rows // 128)): 128}
        if e.dtype != torch.uint8 or e.device != t.device or tuple(e.shape) not in shape:
            raise ValueError(f"fp8_matmul: exponents of {rows} rows are uint8 {list(shape)}")
        blocks.append(shape[tuple(e.shape)])
    if b.device != a.device or not a.numel() or not b.numel():
        raise ValueError("fp8_matmul: non-empty operands on one device")
    _ints("fp8_matmul", a.shape[0], b.shape[0], K)
    a, a_exponents, b, b_exponents = (_at16(t) for t in (a, a_exponents, b, b_exponents))
    out = torch.empty((a.shape[0], b.shape[0]), dtype=dtype, device=a.device)
    d = rt.Fp8MatmulDesc(a.shape[0], b.shape[0], K, *blocks, rt.DCN_NHWC, 0, _DT[dtype])
    n = ctypes.c_size_t()
    rt.check(_fn("dcn_fp8_matmul_workspace")(d, n), "dcn_fp8_matmul_workspace")
    ws = _bytes(out.device, n.value) if n.value else None
    _call(out.device, "dcn_fp8_matmul", d, _ptr(a), _ptr(a_exponents), _ptr(b),
          _ptr(b_exponents), _ptr(out), _ptr(ws), n.value)
    return out


@functools.lru_cache(maxsize=1024)
def _pointwise_plan(B, C, P, O, layout, dtype, grads):
    """Descriptor and buffer sizes (forward workspace, kept, backward workspace) of a product."""
    d = rt.Fp8PointwiseDesc(B, C, P, O, layout, dtype)
    n = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    rt.check(_fn("dcn_fp8_pointwise_workspace")(d, grads, *n), "dcn_fp8_pointwise_workspace")
    return d, *(v.value for v in n)


def _pointwise(x, w, kept, geo, grads):
    """(y, what the backward needs) of x and a weight w [O, C] or an Fp8Weight `kept`."""
    layout, B, C, P, mf = geo
    x, dev = x.contiguous(memory_format=mf), x.device
    O = kept.out_features if w is None else w.shape[0]
    w = None if w is None else w.contiguous()
    d, n_ws, n_saved, n_bwd = _pointwise_plan(B, C, P, O, layout, _DT[x.dtype], grads)
    if x.dim() == 4:
        y = torch.empty((B, O, *x.shape[2:]), dtype=x.dtype, device=dev, memory_format=mf)
    else:
        y = x.new_empty((*x.shape[:-1], O))
    ws = _bytes(dev, n_ws) if n_ws else None
    saved = _bytes(dev, n_saved) if n_saved else None
    q, e = (None, None) if kept is None else (kept.q.data_ptr(), kept.exponents.data_ptr())
    _call(dev, "dcn_fp8_pointwise_fwd", d, grads, x.data_ptr(), _ptr(w), q, e, y.data_ptr(),
          _ptr(saved), n_saved, _ptr(ws), n_ws)
    return y, (d, saved, n_saved, n_bwd)


class _Fp8Pointwise(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, geo):
        need_x, need_w = ctx.needs_input_grad[:2]
        grads = rt.DCN_FP8_GRAD_X * need_x | rt.DCN_FP8_GRAD_W * need_w
        y, (d, saved, n_saved, n_bwd) = _pointwise(x, w, None, geo, grads)
        ctx.args = d, grads, n_saved, n_bwd, geo[-1], x.shape, w.shape
        ctx.save_for_backward(saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        d, grads, n_saved, n_bwd, mf, xshape, wshape = ctx.args
        saved, = ctx.saved_tensors
        gy = gy.contiguous(memory_format=mf)
        new = lambda shape, **kw: torch.empty(shape, dtype=gy.dtype, device=gy.device, **kw)
        gx = new(xshape, memory_format=mf) if grads & rt.DCN_FP8_GRAD_X else None
        gw = new(wshape) if grads & rt.DCN_FP8_GRAD_W else None
        ws = _bytes(gy.device, n_bwd)
        _call(gy.device, "dcn_fp8_pointwise_bwd", d, grads, gy.data_ptr(), saved.data_ptr(),
              n_saved, _ptr(gx), _ptr(gw), ws.data_ptr(), n_bwd)
        return gx, gw, None


def fp8_pointwise(x, weight):
    """x · weightᵀ over the channels (dim 1 of a 4-d tensor, else the last): a linear layer of
    token rows or a 1x1 convolution of maps, its products in 8 bits with one power-of-two scale
    per 128 channels of a token (128 tokens of a channel in the weight's gradient, a map's blocks
    ending with its image; 128 x 128 of the weight). Its sums are fp32 for float32 tensors, the
    8-bit matrix instruction's for bfloat16 ones (fp8_matmul).

    weight: [O, C] (or [O, C, 1, 1]) of x's dtype, rounded in the call, gradients for both; or an
    Fp8Weight (no gradients), as a server keeps it."""
    dt = _dtype(x, "fp8_pointwise")
    geo = _layout(x)
    C = geo[2]
    if isinstance(weight, Fp8Weight):
        if weight.in_features != C or weight.q.device != x.device:
            raise ValueError(f"fp8_pointwise: the weight takes {weight.in_features} channels on "
                             f"{weight.q.device}, x has {C} on {x.device}")
        if torch.is_grad_enabled() and x.requires_grad or \
                forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("fp8_pointwise: an Fp8Weight is for inference (no gradients)")
        O = weight.out_features
    else:
        O = weight.shape[0] if weight.dim() else 0
        if weight.dim() == 4 and tuple(weight.shape[2:]) == (1, 1):
            weight = weight.flatten(1)
        _same(x, weight, "fp8_pointwise", "weight", (O, C))
        if O == 0:
            raise ValueError("fp8_pointwise: no output channels")
    _ints("fp8_pointwise", O)
    if not x.numel():  # no tokens
        shape = (x.shape[0], O, *x.shape[2:]) if x.dim() == 4 else (*x.shape[:-1], O)
        y = x.new_empty(shape)
        return y if isinstance(weight, Fp8Weight) else y + 0 * (x.sum() + weight.sum())
    if isinstance(weight, Fp8Weight):
        return _pointwise(x, None, weight, geo, rt.DCN_FP8_SERVED)[0]
    if _wants_grad(x, weight):
        return _Fp8Pointwise.apply(x, weight, geo)
    return _pointwise(x, weight, None, geo, 0)[0]


class Fp8Pointwise(torch.nn.Module):
    """fp8_pointwise with its weight [out, in] (no bias: a norm or a residual scale follows it in
    a block). serve() makes calls that want no gradient use the weight's 8-bit form, as it is at
    that moment, until train(), a move or a load of other weights; call it again after changing
    the weight. A call that wants a gradient, of x or of the weight, rounds the weight itself."""

    def __init__(self, in_channels, out_channels):
        super().__init__()
        self.in_channels, self.out_channels = in_channels, out_channels
        self.weight = torch.nn.Parameter(torch.randn(out_channels, in_channels) *
                                         in_channels ** -0.5)
        self.weight8 = None

    def serve(self):
        self.weight8 = fp8_quantize_weight(self.weight)
        return self

    def train(self, mode=True):
        if mode:
            self.weight8 = None
        return super().train(mode)

    def _apply(self, fn, *args, **kw):
        self.weight8 = None
        return super()._apply(fn, *args, **kw)

    def _load_from_state_dict(self, *args, **kw):
        self.weight8 = None
        super()._load_from_state_dict(*args, **kw)

    def forward(self, x):
        if self.weight8 is not None and not _wants_grad(x, self.weight):
            return fp8_pointwise(x, self.weight8)
        return fp8_pointwise(x, self.weight)


# ---------------------------------------------------------------------------- a block
class DeformBlock(torch.nn.Module):
    """A residual block around torch_dcn.DeformConv2d and a channel MLP in 8 bits:

        x1, y1 = block_norm(dcn(N(x)), x)      # norm after, layer scale, stochastic depth, norm
        out    = x1 + drop(scale * N(fc2(act(fc1(y1)))))

    on [B, C, H, W] maps, C as torch_dcn.DeformConv2d takes it (bfloat16: a multiple of 4 up
    to 256). `rng`: as in Dropout (two tensors, one per join) for captured steps."""

    def __init__(self, channels, expand=4, layer_scale=0.1, drop_path=0.0, kernel_size=3,
                 act=torch.nn.functional.silu, rng=(None, None)):
        super().__init__()
        import torch_dcn
        pad = kernel_size // 2
        self.norm = BlockNorm(channels, post=None, pre="layer")
        self.dcn = torch_dcn.DeformConv2d(channels, channels, kernel_size, 1, pad)
        self.join = BlockNorm(channels, post="rms", pre="layer", layer_scale=layer_scale,
                              drop_p=drop_path, drop="image", rng=rng[0])
        self.fc1 = Fp8Pointwise(channels, expand * channels)
        self.fc2 = Fp8Pointwise(expand * channels, channels)
        self.act = act
        self.leave = BlockNorm(channels, post="rms", pre=None, layer_scale=layer_scale,
                               drop_p=drop_path, drop="image", rng=rng[1])

    def serve(self):
        """For inference: the MLP's weights in 8 bits."""
        self.fc1.serve()
        self.fc2.serve()
        return self

    def forward(self, x):
        _, y = self.norm(None, x)
        x, y = self.join(self.dcn(y), x)
        return self.leave(self.fc2(self.act(self.fc1(y))), x)[0]
