"""The example's training run: norms, 8-bit checkpoints, products, weight gradients and the shard's optimizer together."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def example(pkg):
    spec = importlib.util.spec_from_file_location('feed_forward8', os.path.join(ROOT, 'examples', 'feed_forward8.py'))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize('dim,hidden,tokens', [(256, 512, 1024), (200, 330, 777)])
def test_trains_as_bf16_does(example, dim, hidden, tokens):
    """The loss falls by a third at least, and its last ten values' mean is within a tenth of what the same blocks reach in
    BF16: products and gradients carry the 8-bit rounding's noise of a few per cent, which a loss averaged over 150,000
    values and ten steps hardly shows.
    Half of BF16's bytes are kept, and scales and row statistics beside them."""
    args = dict(steps=30, tokens=tokens, dim=dim, hidden=hidden, layers=2, seed=3)
    eight, kept8 = example.train(**args, eight=True)
    plain, kept16 = example.train(**args, eight=False)
    end8, end16 = (sum(v[-10:]) / 10 for v in (eight, plain))
    assert eight[-1] < 0.67 * eight[0] and abs(end8 - end16) < 0.1 * end16, (end8, end16)
    assert kept8 < (0.53 if dim % 128 == 0 and hidden % 128 == 0 else 0.7) * kept16


def test_block_gradients_against_plain_blocks(example):
    """One block's gradients against the same block in BF16: relative error below 8 %, where each of the up to three
    8-bit factors in a row contributes some 2.5 % (e4m3's 2^-4 at most, 2^-4 / sqrt(6) root mean square)."""
    from faster_yoco_amd import linear8
    g = torch.Generator(device='cuda').manual_seed(4)
    r = lambda *s: torch.randn(*s, device='cuda', generator=g)  # noqa: E731
    x, wn, wu, wd = (t.bfloat16() for t in (r(500, 384), 1 + 0.1 * r(384), r(640, 384) * 0.05, r(384, 640) * 0.04))
    dy = (r(500, 384) * 1e-3).bfloat16()
    a = [t.clone().requires_grad_() for t in (x, wn, wu, wd)]
    b = [t.clone().requires_grad_() for t in (x, wn, wu, wd)]
    example.Block8.apply(*a, linear8.pack_weight(wu), linear8.pack_weight(wd), []).backward(dy)
    example.plain(*b).backward(dy)
    for p, q in zip(a, b):
        assert float((p.grad.float() - q.grad.float()).norm() / q.grad.float().norm()) < 0.08


def test_a_block_keeps_what_autograd_sees(example):
    """Saved-tensor hooks see the 8-bit rows and both weights, and nothing of the block's input in its own type."""
    from faster_yoco_amd import linear8
    r = lambda *s: torch.randn(*s, device='cuda').bfloat16()  # noqa: E731
    x, wn, wu, wd = r(64, 256).requires_grad_(), r(256).requires_grad_(), r(384, 256), r(256, 384)
    p, kept, sizes = (linear8.pack_weight(wu), linear8.pack_weight(wd)), [], []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        example.Block8.apply(x, wn, wu, wd, *p, sizes)
    assert len(kept) == 14 and not any(t.shape == (64, 256) and t.dtype == torch.bfloat16 for t in kept)
    y = example.Block8.apply(x, wn, wu, wd, *p, sizes)            # without hooks, which pass the version check by
    p[1].qt.view(torch.uint8).zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
