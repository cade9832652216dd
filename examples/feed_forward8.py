"""A stack of pre-norm feed-forward blocks trained on 8-bit operands and checkpoints, with the shard's optimizer.

    python examples/feed_forward8.py [--steps 40] [--tokens 2048] [--dim 512] [--hidden 1024] [--layers 4]

Each block is x + silu(rms_norm(x) Wup^T) Wdown^T.  The norm writes its result as the 8-bit operand of the first product
and its input's 8-bit checkpoint in one pass; the products run on 8-bit weights, packed again after every update from the
BF16 copy that the optimizer writes; and all that a block keeps for its backward pass is 8-bit rows: of its input, of both
operands and of the activation's input.  The weights' gradients are BF16 and go through the shard's norm, clip and Adam.

The same blocks in BF16 by plain torch, from the same start and on the same data, stand beside it.
"""
import argparse
import os
import sys

import torch
from torch.autograd.function import once_differentiable

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from faster_yoco_amd import act8, linear8, norm, shard  # noqa: E402

EPS = 1e-5


class Block8(torch.autograd.Function):
    """One block.  up8, down8: the Weight8 of w_up and w_down; kept: a list that collects what is kept, in bytes."""

    @staticmethod
    def forward(ctx, x, w_norm, w_up, w_down, up8, down8, kept):
        a, rstd, c = norm.rms_norm(x, w_norm, EPS, y8=True, checkpoint=True)
        h = linear8.matmul(a, up8)
        u = act8.pack(torch.nn.functional.silu(h))
        h = act8.pack(h)
        ctx.save_for_backward(w_norm, rstd, up8.qt, up8.st, down8.qt, down8.st, *(p for t in (a, c, h, u) for p in (t.q, t.s)))
        ctx.dims, ctx.shapes = [t.dim for t in (a, c, h, u)], (up8.shape, down8.shape)
        kept.append(sum(t.nbytes() for t in (a, c, h, u)) + rstd.numel() * 4)
        return x + linear8.matmul(u, down8)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w_norm, rstd, *weights = ctx.saved_tensors
        a, c, h8, u = (act8.Act8(*weights[4 + 2 * i:6 + 2 * i], d) for i, d in enumerate(ctx.dims))
        up8, down8 = (linear8.Weight8(None, None, *weights[2 * i:2 * i + 2], s) for i, s in enumerate(ctx.shapes))
        d_down = linear8.weight_grad(dy, u)
        du = linear8.matmul(act8.pack(dy), down8, transposed=True)
        h = act8.unpack(h8).float()
        s = torch.sigmoid(h)
        dh = (du * (s * (1 + h * (1 - s)))).bfloat16()
        d_up = linear8.weight_grad(dh, a)
        da = linear8.matmul(act8.pack(dh), up8, transposed=True)
        dx, d_norm = norm.rms_norm_backward(da, c, rstd, w_norm)
        return dx + dy, d_norm, d_up, d_down, None, None, None


def plain(x, w_norm, w_up, w_down):
    """The same block in BF16 by torch alone."""
    f = x.float()
    n = (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)).bfloat16() * w_norm
    return x + torch.nn.functional.silu(n @ w_up.t()) @ w_down.t()


class Model:
    """The blocks' parameters in one shard, and its optimizer."""

    def __init__(self, dim, hidden, layers, device, seed):
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
        self.optimizer = shard.Zero1ShardOptimizer(self.shard, lr=2e-3, weight_decay=0.0)
        self.leaves = [p.detach().requires_grad_() for p in self.shard.views('p16')]

    def blocks(self):
        return [self.leaves[i:i + 3] for i in range(0, len(self.leaves), 3)]

    def update(self):
        for g, p in zip(self.shard.views('g'), self.leaves):
            g.copy_(p.grad)
            p.grad = None
        self.optimizer.clip_grad_norm(1.0)
        self.optimizer.step()                          # the leaves are the BF16 copy it writes


def train(steps=40, tokens=2048, dim=512, hidden=1024, layers=4, seed=0, eight=True, device='cuda', say=None):
    """(losses, bytes kept per token and block).  The task: a fixed random map of the input, mean squared error."""
    model = Model(dim, hidden, layers, device, seed)
    gen = torch.Generator(device=device)
    gen.manual_seed(seed + 1)
    teacher = torch.randn(dim, dim, device=device, generator=gen) * dim ** -0.5
    losses, kept = [], []
    for step in range(steps):
        x = torch.randn(tokens, dim, device=device, generator=gen)
        target = torch.tanh(x @ teacher)
        y = x.bfloat16()
        for w_norm, w_up, w_down in model.blocks():
            if eight:
                up8, down8 = linear8.pack_weight(w_up.detach()), linear8.pack_weight(w_down.detach())
                y = Block8.apply(y, w_norm, w_up, w_down, up8, down8, kept)
            else:
                y = plain(y, w_norm, w_up, w_down)
                kept.append((4 * dim + 4 * hidden) * tokens)       # x, the norm's result, h and u in BF16
        loss = (y.float() - target).square().mean()
        loss.backward()
        model.update()
        losses.append(loss.detach())
        if say and (step % 10 == 0 or step == steps - 1):
            say(f'  step {step:4d}  loss {float(losses[-1]):.4f}')
    return [float(v) for v in losses], sum(kept) / len(kept) / tokens


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (('steps', 40), ('tokens', 2048), ('dim', 512), ('hidden', 1024), ('layers', 4)):
        ap.add_argument(f'--{name}', type=int, default=value)
    a = vars(ap.parse_args())
    for eight in (True, False):
        print('8-bit operands and checkpoints' if eight else 'BF16 by torch')
        losses, kept = train(**a, eight=eight, say=print)
        print(f'  kept for the backward pass: {kept:.0f} bytes a token and block; loss {losses[0]:.4f} -> {losses[-1]:.4f}')


if __name__ == '__main__':
    main()
