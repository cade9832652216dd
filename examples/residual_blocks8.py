"""Residual feed-forward blocks on 8-bit operands and checkpoints, their matrices under the orthogonalised update.

    python examples/residual_blocks8.py [--steps 40] [--tokens 2048] [--dim 512] [--hidden 1024] [--layers 4]

The stream h and a sublayer's output x go from block to block apart: a block adds x to h and takes the norm of the sum in one
pass (``norm.add_rms_norm``, with the products' 8-bit operand and the sum's 8-bit checkpoint), multiplies twice on 8-bit
weights, and hands on the new x and h.  In the backward pass the stream's gradient is added in the norm's own pass
(``norm.add_rms_norm_backward``).  The weights' gradients are BF16 and go through the shard's norm and clip; matrices then take
the orthogonalised update (``muon.MuonShardOptimizer``), the norms' weights Adam.
"""
import argparse
import os
import sys

import torch
from torch.autograd.function import once_differentiable

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from faster_yoco_amd import act8, linear8, muon, norm, shard  # noqa: E402

EPS = 1e-5


class Block8(torch.autograd.Function):
    """(x, h) -> (x, h) of one block.  up8, down8: the Weight8 of w_up and w_down."""

    @staticmethod
    def forward(ctx, x, h, w_norm, w_up, w_down, up8, down8):
        h, a, rstd, c = norm.add_rms_norm(x, h, w_norm, EPS, y8=True, checkpoint=True)
        u = linear8.matmul(a, up8)
        s, u = act8.pack(torch.nn.functional.silu(u)), act8.pack(u)
        ctx.save_for_backward(w_norm, rstd, up8.qt, up8.st, down8.qt, down8.st, *(p for t in (a, c, u, s) for p in (t.q, t.s)))
        ctx.dims, ctx.shapes = [t.dim for t in (a, c, u, s)], (up8.shape, down8.shape)
        return linear8.matmul(s, down8), h

    @staticmethod
    @once_differentiable
    def backward(ctx, dx, dh):
        w_norm, rstd, *kept = ctx.saved_tensors
        a, c, u8, s = (act8.Act8(*kept[4 + 2 * i:6 + 2 * i], d) for i, d in enumerate(ctx.dims))
        up8, down8 = (linear8.Weight8(None, None, *kept[2 * i:2 * i + 2], n) for i, n in enumerate(ctx.shapes))
        d_down = linear8.weight_grad(dx, s)
        ds = linear8.matmul(act8.pack(dx), down8, transposed=True)
        u = act8.unpack(u8).float()
        g = torch.sigmoid(u)
        du = (ds * (g * (1 + u * (1 - g)))).bfloat16()
        d_up = linear8.weight_grad(du, a)
        da = linear8.matmul(act8.pack(du), up8, transposed=True)
        d, d_norm = norm.add_rms_norm_backward(da, dh, c, rstd, w_norm)
        return d, d, d_norm, d_up, d_down, None, None


def plain(x, h, w_norm, w_up, w_down):
    """The same block in BF16 by torch alone."""
    h = x + h
    f = h.float()
    n = (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)).bfloat16() * w_norm
    return torch.nn.functional.silu(n @ w_up.t()) @ w_down.t(), h


class Model:
    """The blocks' parameters in one shard, and its optimizer."""

    def __init__(self, dim, hidden, layers, device, seed, lr=3e-3):
        shapes = [s for _ in range(layers) for s in ((dim,), (hidden, dim), (dim, hidden))]
        self.shard = shard.FlatShard(shapes, device, grad_dtype=torch.bfloat16)
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        for p in self.shard.views('p'):
            if p.dim() == 1:
                p.fill_(1.0)
            else:
                p.normal_(0.0, p.shape[1] ** -0.5, generator=gen)
        self.shard.p16.copy_(self.shard.p)
        self.optimizer = muon.MuonShardOptimizer(self.shard, lr=lr, weight_decay=0.0)
        self.leaves = [p.detach().requires_grad_() for p in self.shard.views('p16')]

    def forward(self, x):
        h = torch.zeros_like(x)
        for i in range(0, len(self.leaves), 3):
            w_norm, w_up, w_down = self.leaves[i:i + 3]
            x, h = Block8.apply(x, h, w_norm, w_up, w_down, linear8.pack_weight(w_up.detach()), linear8.pack_weight(w_down.detach()))
        return x + h

    def update(self):
        for g, p in zip(self.shard.views('g'), self.leaves):
            g.copy_(p.grad)
            p.grad = None
        self.optimizer.clip_grad_norm(1.0)
        self.optimizer.step()                          # the leaves are the BF16 copy it writes


def train(steps=40, tokens=2048, dim=512, hidden=1024, layers=4, seed=0, device='cuda', say=None):
    """The losses.  The task: a fixed random map of the input, mean squared error."""
    model = Model(dim, hidden, layers, device, seed)
    gen = torch.Generator(device=device)
    gen.manual_seed(seed + 1)
    teacher = torch.randn(dim, dim, device=device, generator=gen) * dim ** -0.5
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, dim, device=device, generator=gen)
        loss = (model.forward(x.bfloat16()).float() - torch.tanh(x @ teacher)).square().mean()
        loss.backward()
        model.update()
        losses.append(loss.detach())
        if say and (step % 10 == 0 or step == steps - 1):
            say(f'  step {step:4d}  loss {float(losses[-1]):.4f}')
    return [float(v) for v in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (('steps', 40), ('tokens', 2048), ('dim', 512), ('hidden', 1024), ('layers', 4)):
        ap.add_argument(f'--{name}', type=int, default=value)
    train(**vars(ap.parse_args()), say=print)


if __name__ == '__main__':
    main()
