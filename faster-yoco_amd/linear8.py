"""Linear maps on 8-bit operands: the forward product, the input's gradient and the weight's gradient.

    a = act8.pack(x)                          # or norm.layer_norm(..., y8=True): the operand, and the checkpoint
    w = linear8.pack_weight(weight)           # after each optimizer update
    y = linear8.matmul(a, w)                  # x @ weight.T
    dx = linear8.matmul(act8.pack(dy), w, transposed=True)        # dy @ weight
    dw = linear8.weight_grad(dy, a)           # dy.T @ x, from the checkpoint

``linear`` is the three of them as one differentiable function; the others compute values only, and no gradient passes
through them (torch warns in a backward pass that reaches one).  Products read e4m3 values and their scales, which bf16 holds
exactly, and sum in fp32 for every result type; the weight's gradient reads dy in bf16 and the checkpoint's values.  (A value that
rounded up to 2^128, past fp32's largest, multiplies as an infinity.)
"""
import torch
from torch.autograd.function import once_differentiable

from . import act8, library  # noqa: F401  (library registers the operators)
from .act8 import Act8

_pack = torch.ops.yoco_z1.weight8_pack.default
_product = torch.ops.yoco_z1.product8.default
_weight_grad = torch.ops.yoco_z1.weight_grad8.default


class Weight8:
    """A weight [N, K] in 128 x 128 blocks of one power-of-two scale each, in both orders: ``q`` float8_e4m3fn [N, K
    rounded up to 128] with ``s`` float8_e8m0fnu [ceil(N / 128), blocks of K rounded up to 4], and ``qt`` [K, N rounded up
    to 128] with ``st`` for the input's gradient (None: forward only).  ``shape`` is (N, K)."""
    __slots__ = ('q', 's', 'qt', 'st', 'shape')

    def __init__(self, q, s, qt, st, shape):
        self.q, self.s, self.qt, self.st, self.shape = q, s, qt, st, shape

    def nbytes(self):
        return sum(t.numel() for t in (self.q, self.s, self.qt, self.st) if t is not None)


def pack_weight(w, transposed=True):
    """The 8-bit form of a weight [N, K] (fp32, bf16 or fp16), with its other order unless transposed is False."""
    if w.dim() != 2:
        raise RuntimeError('linear8.pack_weight: expected a weight [N, K]')
    out = _pack(act8.rows_of(w), transposed)
    return Weight8(*(out if transposed else (*out, None, None)), tuple(w.shape))


def matmul(a, w, dtype=torch.bfloat16, transposed=False):
    """8-bit rows a [M, K] times the transpose of w [N, K]: [M, N] in `dtype`; transposed: a [M, N] times w: [M, K]."""
    N, K = w.shape
    if a.dim != (N if transposed else K):
        raise RuntimeError(f'linear8.matmul: rows of {a.dim} columns do not fit a weight {N} x {K}'
                           f'{" from the left" if transposed else ""}')
    if transposed:
        if w.qt is None:
            raise RuntimeError('linear8.matmul: the weight was packed without its other order')
        return _product(a.q, a.s, w.qt, w.st, N, dtype)
    return _product(a.q, a.s, w.q, w.s, K, dtype)


def weight_grad(dy, a, dtype=torch.bfloat16):
    """dy^T x, [N, K] in `dtype`, from bf16 gradient rows dy [..., N] and the 8-bit rows a of x [..., K]."""
    return _weight_grad(act8.rows_of(dy), a.q, a.s, a.dim, dtype)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, w8):
        a = act8.pack(x)
        need_x, need_w = ctx.needs_input_grad[:2]
        if need_x and w8.qt is None:
            raise RuntimeError('linear8.linear: the weight was packed without its other order, which the gradient of x needs')
        ctx.save_for_backward(*((w8.qt, w8.st) if need_x else (None, None)), *((a.q, a.s) if need_w else (None, None)))
        ctx.shape, ctx.dim, ctx.x_shape, ctx.dtype, ctx.w_dtype = w8.shape, a.dim, x.shape, x.dtype, weight.dtype
        return matmul(a, w8, x.dtype).view(*x.shape[:-1], w8.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = dw = None
        qt, st, q, s = ctx.saved_tensors
        if ctx.needs_input_grad[0]:
            w8 = Weight8(None, None, qt, st, ctx.shape)
            dx = matmul(act8.pack(dy), w8, ctx.dtype, transposed=True).view(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            dw = weight_grad(dy, Act8(q, s, ctx.dim), ctx.w_dtype)
        return dx, dw, None


def linear(x, weight, w8):
    """x @ weight.T for bf16 x [..., K], differentiable: w8 is pack_weight(weight), packed again whenever the weight
    changes.  What is kept for the backward pass is the 8-bit rows of x and w8's other order; w8's tensors may be replaced
    before it, not written."""
    if x.dtype != torch.bfloat16:
        raise RuntimeError('linear8.linear: expected bf16 rows')
    if tuple(weight.shape) != tuple(w8.shape):
        raise RuntimeError(f'linear8.linear: a weight of {tuple(weight.shape)} and 8-bit blocks of {tuple(w8.shape)}')
    return _Linear.apply(x, weight, w8)
