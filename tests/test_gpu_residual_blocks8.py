"""The example's blocks and training steps: the stream's addition and norm, 8-bit products and checkpoints, and the shard's
optimizer with the orthogonalised update, together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def example(pkg):
    spec = importlib.util.spec_from_file_location('residual_blocks8', os.path.join(ROOT, 'examples', 'residual_blocks8.py'))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_block_gradients_against_plain_blocks(example):
    """Two blocks' gradients against the same in BF16: each of the up to six 8-bit factors in a row contributes some 2.5 %
    (e4m3's 2^-4 at most, 2^-4 / sqrt(6) root mean square): 2.5 % sqrt(6), and as much again for their being correlated."""
    from faster_yoco_amd import linear8
    g = torch.Generator(device='cuda').manual_seed(4)
    r = lambda *s: torch.randn(*s, device='cuda', generator=g)  # noqa: E731
    x, h, wn, wu, wd = (t.bfloat16() for t in (r(500, 384), r(500, 384), 1 + 0.1 * r(384), r(640, 384) * 0.05, r(384, 640) * 0.04))
    dx, dh = ((r(500, 384) * 1e-3).bfloat16() for _ in range(2))
    a = [t.clone().requires_grad_() for t in (x, h, wn, wu, wd)]
    b = [t.clone().requires_grad_() for t in (x, h, wn, wu, wd)]
    p = linear8.pack_weight(wu), linear8.pack_weight(wd)
    u, v = a[:2]
    for _ in range(2):
        u, v = example.Block8.apply(u, v, *a[2:], *p)
    torch.autograd.backward([u, v], [dx, dh])
    u, v = b[:2]
    for _ in range(2):
        u, v = example.plain(u, v, *b[2:])
    torch.autograd.backward([u, v], [dx, dh])
    for s, t in zip(a, b):
        assert float((s.grad.float() - t.grad.float()).norm() / t.grad.float().norm()) < 0.12
    assert torch.equal(a[0].grad, a[1].grad)


@pytest.mark.parametrize('dim,hidden,tokens', [(256, 512, 512), (200, 330, 300)])
def test_steps_follow_their_own_formulas(example, dim, hidden, tokens):
    """Three training steps: they run, are finite, and each step's matrices are what step_ makes of the clipped gradients."""
    from faster_yoco_amd import muon
    model = example.Model(dim, hidden, 2, torch.device('cuda'), 5)
    sh = model.shard
    for step in range(3):
        x = torch.randn(tokens, dim, device='cuda', generator=torch.Generator('cuda').manual_seed(step)).bfloat16()
        (model.forward(x).float() - x.float().tanh()).square().mean().backward()
        before = {k: [t.clone() for t in sh.views(k)] for k in ('p', 'm')}
        grads = [p.grad.clone() for p in model.leaves]
        total = float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt())
        model.update()
        assert all(g.isfinite().all() for g in grads)
        rows = model.optimizer.matrices
        assert rows == [1, 2, 4, 5]
        factor = torch.tensor([min(1.0, 1.0 / (total + 1e-6))], device='cuda')
        p, m = ([before[k][i] for i in rows] for k in ('p', 'm'))
        muon.step_(p, [grads[i] for i in rows], m, lr=3e-3, weight_decay=0.0, factor=factor)
        for a, i in zip(p, rows):
            # the factor's last bits (a 64-bit norm here) reach p only through the update's direction
            assert float((a - sh.views('p')[i]).norm()) <= 1e-5 * float(a.norm())
        assert all(torch.equal(c, t.bfloat16()) for c, t in zip(sh.views('p16'), sh.views('p')))


def test_the_example_runs(example, capsys):
    losses = example.train(steps=3, tokens=256, dim=128, hidden=192, layers=2, say=print)
    assert len(losses) == 3 and all(v == v and abs(v) < 1e4 for v in losses) and 'loss' in capsys.readouterr().out
