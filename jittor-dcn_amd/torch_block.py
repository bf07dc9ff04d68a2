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
"""
from __future__ import annotations

import contextlib
import ctypes
import threading

import torch
from torch.autograd.function import once_differentiable

import dcn_runtime as rt

_DT = {torch.float32: rt.DCN_F32, torch.bfloat16: rt.DCN_BF16}
_handles = {}
_lock = threading.Lock()  # a handle takes one caller at a time: stream and launch belong together
_null = contextlib.nullcontext()


def _call(dev: torch.device, fn: str, *args):
    """One libdcn call on torch's current stream of `dev`, whatever device is current."""
    here = torch.cuda.current_device()
    idx = dev.index if dev.index is not None else here
    with (_null if idx == here else torch.cuda.device(idx)), _lock:
        h = _handles.get(idx)
        if h is None:
            h = _handles[idx] = rt.Handle(idx)
        stream = torch.cuda.current_stream(idx).cuda_stream
        if getattr(h, "bound", -1) != stream:
            h.set_stream(stream)
            h.bound = stream
        rt.check(getattr(h.lib, fn)(h.h, *args), fn)


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
    shape = tuple(x.shape if shape is None else shape)
    if t.dtype != x.dtype or t.device != x.device or tuple(t.shape) != shape:
        raise ValueError(f"{what}: {name} must be {shape} {x.dtype} on {x.device}, not "
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


# ---------------------------------------------------------------------------- dropout
class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, group):
        seed, offset, dev_rng = _rng(rng, x.device, "dropout")
        d = rt.DropoutDesc(x.numel(), group, seed, offset, _DT[x.dtype], p)
        x = x.contiguous()
        residual = residual.contiguous() if residual is not None else None
        y = torch.empty_like(x)
        if x.numel():
            _call(x.device, "dcn_dropout_fwd", d, _ptr(x), _ptr(residual), _ptr(y), _ptr(dev_rng))
        ctx.desc = d
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
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout: p must be between 0 and 1")
    if isinstance(group, str):
        skip = {"element": x.dim(), "channel": 2, "image": 1}.get(group)
        if skip is None or x.dim() < min(skip, 2):
            raise ValueError(f"dropout: group {group!r} does not fit a {x.dim()}-d tensor")
        group = 1
        for s in x.shape[skip:]:
            group *= s
    if group < 1 and x.numel():
        raise ValueError("dropout: group must be positive")
    return _Dropout.apply(x, residual, float(p), rng, max(int(group), 1))


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
