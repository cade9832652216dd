"""Layer norm and RMS norm over the last dimension, forward and backward, with 8-bit results and checkpoints, alone or with
the residual stream's addition in the same pass.

The forward pass reads x once and can write, in that pass, y in 8 bits (``y8``: the operand of ``linear8.matmul``) and the
8-bit rows of x (``checkpoint``), which the backward pass then takes in x's place, so that x itself need not be kept.
Statistics are fp32, taken about the mean.  y in 8 bits is rounded from its fp32 value: one within fp32's own rounding of the
middle between two e4m3 values, or a block's largest of where its scale steps, may go either way.

``add_layer_norm`` and ``add_rms_norm`` add a sublayer's output x to the residual stream, h = x + residual rounded to their
type, and return h with the norm of it; their gradients take dh, what reaches h past the norm, and return one dx, which is x's
and the residual's alike.

``layer_norm_train``, ``rms_norm_train``, ``add_layer_norm_train`` and ``add_rms_norm_train`` are differentiable; the others
compute values only, and no gradient passes through them (torch warns in a backward pass that reaches one).
"""
import torch
from torch.autograd.function import once_differentiable

from . import act8, library  # noqa: F401  (library registers the operators)
from .act8 import Act8

_norm_forward = torch.ops.yoco_z1.norm_forward.default
_norm_backward = torch.ops.yoco_z1.norm_backward.default
_add_norm_forward = torch.ops.yoco_z1.add_norm_forward.default
_add_norm_backward = torch.ops.yoco_z1.add_norm_backward.default


def _results(out, x, y8, checkpoint):
    d = x.shape[-1]
    y, stats = (Act8(out[0], out[1], d), out[2:]) if y8 else (out[0] if x.dim() == 2 else out[0].view(x.shape), out[1:])
    if checkpoint:
        return (y, *stats[:-2], Act8(stats[-2], stats[-1], d))
    return (y, *stats)


def _forward(x, weight, bias, eps, center, y8, checkpoint):
    return _results(_norm_forward(act8.rows_of(x), weight, bias, eps, center, y8, checkpoint), x, y8, checkpoint)


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, y8=False, checkpoint=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x (fp32, bf16 or fp16; weight and bias in
    its type or fp32, or None).  Returns (y, mean, rstd): y in x's type and shape, or an Act8 of its rows where y8; mean
    and rstd fp32 [rows].  checkpoint adds the Act8 of x's rows."""
    return _forward(x, weight, bias, eps, True, y8, checkpoint)


def rms_norm(x, weight=None, eps=1e-5, *, y8=False, checkpoint=False):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension of x.  Returns (y, rstd), and with checkpoint the Act8 of
    x's rows; otherwise as layer_norm."""
    return _forward(x, weight, None, eps, False, y8, checkpoint)


def _add_forward(x, residual, weight, bias, eps, center, y8, checkpoint):
    if x.shape != residual.shape:
        raise RuntimeError(f'add_norm: x of {tuple(x.shape)} and a residual of {tuple(residual.shape)}')
    out = _add_norm_forward(act8.rows_of(x), act8.rows_of(residual), weight, bias, eps, center, y8, checkpoint)
    h = out[0] if x.dim() == 2 else out[0].view(x.shape)
    return (h, *_results(out[1:], x, y8, checkpoint))


def add_layer_norm(x, residual, weight=None, bias=None, eps=1e-5, *, y8=False, checkpoint=False):
    """h = x + residual (one shape and type) and layer_norm(h): (h, y, mean, rstd), and with checkpoint the Act8 of h's
    rows."""
    return _add_forward(x, residual, weight, bias, eps, True, y8, checkpoint)


def add_rms_norm(x, residual, weight=None, eps=1e-5, *, y8=False, checkpoint=False):
    """h = x + residual (one shape and type) and rms_norm(h): (h, y, rstd), and with checkpoint the Act8 of h's rows."""
    return _add_forward(x, residual, weight, None, eps, False, y8, checkpoint)


def _backward(dy, x, mean, rstd, weight, center, need_weight, need_bias, grad_dtype=None, dh=None):
    r = act8.rows_of(dy)
    if isinstance(x, Act8):
        if x.dim != dy.shape[-1]:
            raise RuntimeError(f'norm_backward: a checkpoint of {x.dim} columns, gradient rows of {dy.shape[-1]}')
        x = (None, x.q, x.s)
    else:
        x = (act8.rows_of(x), None, None)
    if dh is None:
        out = _norm_backward(r, *x, mean, rstd, weight, center, need_weight, need_bias, grad_dtype)
    else:
        if dh.shape != dy.shape:
            raise RuntimeError(f'add_norm_backward: dy of {tuple(dy.shape)} and dh of {tuple(dh.shape)}')
        out = _add_norm_backward(r, act8.rows_of(dh), *x, mean, rstd, weight, center, need_weight, need_bias, grad_dtype)
    if dy.dim() != 2:
        return (out[0].view(dy.shape), *out[1:])
    return tuple(out)


def layer_norm_backward(dy, x, mean, rstd, weight=None, *, bias=False, grad_dtype=None):
    """The gradients of layer_norm from dy, its input x (dy's type, or the Act8 of its rows) and the forward's mean and
    rstd: (dx, dw) where weight is given, with db where bias is True; dw and db in grad_dtype, else in the weight's type, else
    in dy's (fp32 for an fp32 bias without a weight)."""
    return _backward(dy, x, mean, rstd, weight, True, weight is not None, bias, grad_dtype)


def rms_norm_backward(dy, x, rstd, weight=None):
    """The gradients of rms_norm: (dx,), with dw where weight is given."""
    return _backward(dy, x, None, rstd, weight, False, weight is not None, False)


def add_layer_norm_backward(dy, dh, h, mean, rstd, weight=None, *, bias=False, grad_dtype=None):
    """The gradients of add_layer_norm from dy, dh (dy's shape and type) and h (or its Act8): (dx, dw, db) as
    layer_norm_backward, dx with dh added; it is x's and the residual's."""
    return _backward(dy, h, mean, rstd, weight, True, weight is not None, bias, grad_dtype, dh)


def add_rms_norm_backward(dy, dh, h, rstd, weight=None):
    """The gradients of add_rms_norm: (dx,), with dw where weight is given."""
    return _backward(dy, h, None, rstd, weight, False, weight is not None, False, None, dh)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, center, checkpoint):
        out = _forward(x, weight, bias, eps, center, False, checkpoint)
        mean, rstd = (out[1], out[2]) if center else (None, out[1])
        kept = (out[-1].q, out[-1].s) if checkpoint else (x, None)
        ctx.save_for_backward(*kept, mean, rstd, weight)
        ctx.center, ctx.checkpoint, ctx.bias = center, checkpoint, None if bias is None else bias.dtype
        return out[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        kept, s, mean, rstd, weight = ctx.saved_tensors
        x = Act8(kept, s, dy.shape[-1]) if ctx.checkpoint else kept
        need_w = weight is not None and ctx.needs_input_grad[1]
        need_b = ctx.bias is not None and ctx.needs_input_grad[2]
        out = list(_backward(dy, x, mean, rstd, weight, ctx.center, need_w, need_b, ctx.bias))
        dx = out.pop(0)
        dw = out.pop(0) if need_w else None
        return dx, dw, out.pop(0) if need_b else None, None, None, None


def layer_norm_train(x, weight=None, bias=None, eps=1e-5, *, checkpoint=False):
    """layer_norm's y, differentiable; with checkpoint the 8-bit rows of x are kept for the backward pass, not x."""
    return _Norm.apply(x, weight, bias, eps, True, checkpoint)


def rms_norm_train(x, weight=None, eps=1e-5, *, checkpoint=False):
    """rms_norm's y, differentiable; with checkpoint the 8-bit rows of x are kept for the backward pass, not x."""
    return _Norm.apply(x, weight, None, eps, False, checkpoint)


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, center, checkpoint):
        out = _add_forward(x, residual, weight, bias, eps, center, False, checkpoint)
        mean, rstd = (out[2], out[3]) if center else (None, out[2])
        kept = (out[-1].q, out[-1].s) if checkpoint else (out[0], None)
        ctx.save_for_backward(*kept, mean, rstd, weight)
        ctx.center, ctx.checkpoint, ctx.bias = center, checkpoint, None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return out[0], out[1]

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dy):
        kept, s, mean, rstd, weight = ctx.saved_tensors
        if dy is None:                                 # only h was used
            return dh, dh, None, None, None, None, None
        h = Act8(kept, s, dy.shape[-1]) if ctx.checkpoint else kept
        need_w = weight is not None and ctx.needs_input_grad[2]
        need_b = ctx.bias is not None and ctx.needs_input_grad[3]
        out = list(_backward(dy, h, mean, rstd, weight, ctx.center, need_w, need_b, ctx.bias, dh))
        dx = out.pop(0)
        dw = out.pop(0) if need_w else None
        return dx, dx, dw, out.pop(0) if need_b else None, None, None, None


def add_layer_norm_train(x, residual, weight=None, bias=None, eps=1e-5, *, checkpoint=False):
    """add_layer_norm's (h, y), differentiable; with checkpoint the 8-bit rows of h are kept for the backward pass, not h."""
    return _AddNorm.apply(x, residual, weight, bias, eps, True, checkpoint)


def add_rms_norm_train(x, residual, weight=None, eps=1e-5, *, checkpoint=False):
    """add_rms_norm's (h, y), differentiable; with checkpoint the 8-bit rows of h are kept for the backward pass, not h."""
    return _AddNorm.apply(x, residual, weight, None, eps, False, checkpoint)
