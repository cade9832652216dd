"""8-bit activations: rows in blocks of 128 columns, e4m3 values with a power-of-two scale for each block.

An ``Act8`` is what a layer keeps of an activation for its backward pass (half the bytes of bf16), and at the same time
the operand of an 8-bit product: pack it once -- alone (``pack``) or in the pass of the norm that makes it
(``norm.layer_norm(..., y8=True)``) -- multiply it (``linear8.matmul``), keep it, and let the weight's gradient
(``linear8.weight_grad``) or the norm's backward pass (``norm.layer_norm_backward``) read it in the activation's place.

The scale of a block is the least 2^e (e >= -127) with max |x| <= 448 * 2^e over its finite elements, so that scaling is
exact and an element has one rounding, to the nearest e4m3 value (relative error up to 2^-4; below 2^-6 of its scale, up
to 2^-10 of the scale).  Infinities and NaN become NaN and do not count for the scale.  No gradient
passes through ``pack`` and ``unpack``.
"""
import torch

from . import library  # noqa: F401  (registers the operators)

# the overloads themselves: a call through the packet looks one up first (0.5 us)
_pack = torch.ops.yoco_z1.act8_pack.default
_unpack = torch.ops.yoco_z1.act8_unpack.default

BLOCK = 128


class Act8:
    """8-bit rows: ``q`` float8_e4m3fn [rows, dim rounded up to 128], zero past ``dim``; ``s`` float8_e8m0fnu [rows,
    blocks rounded up to 4], one past the last block; ``dim`` the columns that count.  Both tensors are contiguous."""
    __slots__ = ('q', 's', 'dim')

    def __init__(self, q, s, dim):
        self.q, self.s, self.dim = q, s, dim

    @property
    def rows(self):
        return self.q.shape[0]

    @property
    def device(self):
        return self.q.device

    def nbytes(self):
        return self.q.numel() + self.s.numel()


def rows_of(x):
    """x [..., dim] as rows whose elements are neighbours: a view where its strides allow, else a copy."""
    if x.dim() == 2:
        if x.stride(1) == 1 and x.stride(0) >= 0:
            return x
        r = x
    elif x.dim() == 0:
        raise RuntimeError('yoco_z1: expected a tensor with at least one dimension')
    elif x.dim() == 1:
        r = x[None]
    else:
        n = 1
        for k in x.shape[:-1]:
            n *= k
        r = x.reshape(n, x.shape[-1])
    d = r.shape[1]
    if (d > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < 0):
        r = r.contiguous()
    return r


def pack(x):
    """The 8-bit rows of x [..., dim] (fp32, bf16 or fp16; leading dimensions become rows)."""
    q, s = _pack(rows_of(x))
    return Act8(q, s, x.shape[-1])


def unpack(a, dtype=torch.bfloat16):
    """The values that 8-bit rows stand for, [rows, dim] in `dtype`.  A finite value stays finite: one past the type's
    largest becomes the largest."""
    return _unpack(a.q, a.s, a.dim, dtype)
