"""The orthogonalised update of matrices: momentum, Newton-Schulz steps that bring its singular values near 1, decoupled decay.

    q = muon.orthogonalize(x)                              # matrices [..., m, n], their singular values near 1
    muon.step_(params, grads, momenta, copies, lr=3e-4)    # one update of fp32 master matrices and their BF16 copies
    opt = muon.MuonShardOptimizer(shard, lr=3e-4)          # a shard: its matrices by this, its other tensors by Adam

X = u / max(|u|_F, eps), then for each step's (a, b, c): X <- a X + b (X X^T) X + c (X X^T)^2 X.  The default coefficients
take singular values from 1e-3 of the norm up to between 0.7 and 1.2 in five steps.  The products run on fp16 operands with
fp32 sums, X kept in 22 bits and the diagonals of both symmetric products in fp32.  ``precise``: the operands are pairs of fp16,
which leaves the result as fp32 products do, 1e-6 to 3e-5 off the exact iterate (2-norm, relative; 1e-4 to 4e-4 where the input
has few directions).  Without it, 4e-4 to 1e-3 mostly and up to 2e-3 whatever the spectrum, about a bf16 result's rounding
(1.7e-3) at the most, at two fifths of the work; matrices whose shorter side is at most 64 have pairs in any case.  The products
of a call's matrices share launches, whose tiles are chosen by how much there is in all: the same call gives the same bits, but
the last bits of a matrix may differ with the matrices beside it.  None of it is differentiable.
"""
import math

import torch

from . import library, ops, shard as shard_mod  # noqa: F401  (library registers the operators)

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 64
MAX_SIDE = 1 << 20

_orthogonalize = torch.ops.yoco_z1.orthogonalize.default
_step = torch.ops.yoco_z1.muon_step_.default


def _coefficients(coefficients, steps):
    """[a, b, c] of each step, in a row: one triple for all of them, or a triple for each."""
    if not 1 <= steps <= MAX_STEPS:
        raise RuntimeError(f'muon: expected 1 to {MAX_STEPS} steps, got {steps}')
    c = list(coefficients)
    if len(c) == 3 and not any(hasattr(v, '__len__') for v in c):
        return [float(v) for v in c] * int(steps)
    if len(c) != steps or any(not hasattr(v, '__len__') or len(v) != 3 for v in c):
        raise RuntimeError(f'muon: expected one triple of coefficients or {steps} of them, got {coefficients!r}')
    return [float(v) for t in c for v in t]


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=None, precise=None):
    """The matrices of x [..., m, n] (fp32, bf16 or fp16, m and n from 1 to 2^20), each orthogonalised by `steps` steps, in
    `dtype` (x's own where None) and contiguous.  coefficients: one (a, b, c), or one for each step; they must keep singular
    values that start in [0, 1] below 4.  A matrix of zeros stays one; an infinity or NaN makes its whole matrix NaN.  precise:
    None for what `dtype` holds (bf16: no, fp16 and fp32: yes)."""
    if x.dim() < 2:
        raise RuntimeError('muon.orthogonalize: expected matrices [..., m, n]')
    dtype = x.dtype if dtype is None else dtype
    m, n = x.shape[-2:]
    r = x if x.dim() == 3 else x.reshape(math.prod(x.shape[:-2]), m, n)
    if (n > 1 and r.stride(2) != 1) or any(r.shape[i] > 1 and r.stride(i) < 0 for i in (0, 1)):
        r = r.contiguous()
    out = _orthogonalize(r, int(steps), _coefficients(coefficients, steps), float(eps), dtype,
                         dtype != torch.bfloat16 if precise is None else bool(precise))
    return out if x.dim() == 3 else out.view(x.shape)


def rate(lr, shape, adjust):
    """The rate of a matrix: lr times 0.2 sqrt(max(m, n)) for 'rms' (the update's elements are then as large as Adam's), times
    sqrt(max(1, m / n)) for 'shape', or times a number."""
    m, n = shape
    if adjust == 'rms':
        return lr * 0.2 * math.sqrt(max(m, n))
    if adjust == 'shape':
        return lr * math.sqrt(max(1.0, m / n)) if n else lr
    if isinstance(adjust, str):
        raise RuntimeError(f"muon: adjust is 'rms', 'shape' or a number, not {adjust!r}")
    return lr * float(adjust)


def step_(params, grads, momenta, copies=None, *, lr, momentum=0.95, nesterov=True, weight_decay=0.1, adjust='rms', factor=None,
          steps=5, coefficients=COEFFICIENTS, eps=1e-7, precise=None):
    """One update, in place, of matrices `params` (fp32, contiguous) with `momenta` (alike) and their BF16 `copies` (or None):

        momentum_i = momentum * momentum_i + (1 - momentum) * factor * g_i
        u_i = momentum * momentum_i + (1 - momentum) * factor * g_i  (nesterov), or momentum_i
        p_i = p_i * (1 - lr * weight_decay) - rate(lr, p_i.shape, adjust) * orthogonalize(u_i)

    Sides from 1 to 2^20; a call that is refused has written nothing.  momentum is taken in fp32, and 1 - momentum from it.
    grads: fp32, bf16 or fp16, with rows of neighbouring elements.  factor: None or a one-element fp32 device tensor, as the
    clip leaves it.  Nothing that is written may overlap another of the call's tensors.  precise: None for what fp32 masters hold
    (yes); False takes half the time and leaves p off by some 1e-3 of its update."""
    params, grads, momenta, copies = list(params), list(grads), list(momenta), [] if copies is None else list(copies)
    if not (params or grads or momenta or copies):
        return
    lrs = [rate(lr, p.shape, adjust) if p.dim() == 2 else lr for p in params]
    _step(params, grads, momenta, copies, factor, lrs, [1.0 - lr * weight_decay] * len(params), float(momentum), bool(nesterov),
          int(steps), _coefficients(coefficients, steps), float(eps), precise is None or bool(precise))


class MuonShardOptimizer(shard_mod.Zero1ShardOptimizer):
    """A FlatShard's optimizer whose matrices take the orthogonalised update and whose other tensors take Adam, under the same
    norm, clip and gradient factor and with the same surface as Zero1ShardOptimizer.

    matrices: the shard's rows that are updated so (all of its two-dimensional ones with more than one row and column where
    None; embeddings and output layers are usually left to Adam).  Their momentum is kept in the shard's ``m``; their part of
    ``v`` is not used.  matrix_lr, matrix_weight_decay: lr and weight_decay where None; the other arguments are Adam's, or
    step_'s.  A step in pieces is refused: a step's matrices share launches."""

    def __init__(self, shard, matrices=None, matrix_lr=None, matrix_weight_decay=None, momentum=0.95, nesterov=True,
                 adjust='rms', steps=5, coefficients=COEFFICIENTS, matrix_eps=1e-7, precise=None, **adam):
        super().__init__(shard, **adam)
        if matrices is None:
            matrices = [i for i, s in enumerate(shard.shapes) if len(s) == 2 and min(s) > 1]
        self.matrices = sorted(int(i) for i in matrices)
        if len(set(self.matrices)) != len(self.matrices) or any(
                not 0 <= i < len(shard.shapes) or len(shard.shapes[i]) != 2 for i in self.matrices):
            raise RuntimeError('muon: matrices must be rows of the shard with two dimensions, each once')
        for i in self.matrices:
            if max(shard.shapes[i]) > MAX_SIDE:
                raise RuntimeError(f'muon: row {i} of {shard.shapes[i]}: sides of at most {MAX_SIDE}; name the other matrices')
        self.matrix_lr = None if matrix_lr is None else float(matrix_lr)
        self.matrix_weight_decay = None if matrix_weight_decay is None else float(matrix_weight_decay)
        self.how = dict(momentum=momentum, nesterov=nesterov, adjust=adjust, steps=steps, coefficients=coefficients,
                        eps=matrix_eps, precise=precise)
        pick = lambda buf: [shard.views(buf)[i] for i in self.matrices]  # noqa: E731
        self._p, self._g, self._m = pick('p'), pick('g'), pick('m')
        self._p16 = None if shard.p16 is None else pick('p16')
        rest = [i for i in range(len(shard.shapes)) if i not in set(self.matrices)]
        if len(rest) < len(shard.shapes):
            self._adam_table = ops.Table.flat([shard.offsets[i] for i in rest], [shard.numels[i] for i in rest], shard.g,
                                              shard.p, shard.m, shard.v, shard.p16) if rest else None

    def step(self, closure=None, groups=None, pieces=None, on_piece=None):
        """The matrices' update, then Adam over the other rows, with the gradient factor in both; then factor := 1."""
        if pieces is not None:
            raise RuntimeError('muon: a step in pieces is not available: its matrices share launches')
        if self.matrices:
            lr = self.lr if self.matrix_lr is None else self.matrix_lr
            decay = self.weight_decay if self.matrix_weight_decay is None else self.matrix_weight_decay
            step_(self._p, self._g, self._m, self._p16, lr=lr, weight_decay=decay, factor=self._step_factor(), **self.how)
        super().step()
