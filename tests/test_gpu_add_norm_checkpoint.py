"""The residual stream's differentiable norms with checkpoints: autograd's gradients are the operator's own from the same 8-bit
rows, bit for bit, and the 64-bit gradient at the values of those rows within fp32's bound."""
import pytest
import torch

import blocks as ref
from blocks import U

pytestmark = pytest.mark.gpu


def inputs(n, dim, dtype):
    g = torch.Generator().manual_seed(n + dim)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [t.to(dtype) for t in (r(n, dim), r(n, dim) + 0.3, 1 + 0.2 * r(dim), 0.1 * r(dim), r(n, dim), r(n, dim))]


def bound_of(dx, dh, h, mean, rstd, xh, g, center):
    """As in test_gpu_add_norm.py: the norm's part within 128 u r (sizes), u of the sum with dh on the way."""
    size = g.abs() + g.abs().mean(1)[:, None] + xh.abs() * (g * xh).abs().mean(1)[:, None]
    m = rstd.double()[:, None] * (h.double().abs() + (mean.double().abs()[:, None] if center else 0))
    size = size + m * (g * xh).abs().mean(1)[:, None] + xh.abs() * (g.abs() * m).mean(1)[:, None]
    return 128 * U * rstd.double()[:, None] * size + U * (dx.abs() + dh.double().abs()) * 1.001


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('n,dim', [(40, 200), (7, 1537), (3000, 130), (5, 17000)])
def test_gradients_from_the_checkpoint(pkg, dev, n, dim, center, dtype):
    from faster_yoco_amd import act8, norm
    x, res, w, b, dy, dh = (t.to(dev) for t in inputs(n, dim, dtype))
    leaves = [t.clone().requires_grad_() for t in ((x, res, w, b) if center else (x, res, w))]
    h, y = (norm.add_layer_norm_train if center else norm.add_rms_norm_train)(*leaves, checkpoint=True)
    got = torch.autograd.grad([h, y], leaves, [dh, dy])
    if center:
        h2, y2, mean, rstd, c = norm.add_layer_norm(x, res, w, b, checkpoint=True)
        want = norm.add_layer_norm_backward(dy, dh, c, mean, rstd, w, bias=True)
    else:
        h2, y2, rstd, c = norm.add_rms_norm(x, res, w, checkpoint=True)
        mean, want = None, norm.add_rms_norm_backward(dy, dh, c, rstd, w)
    assert torch.equal(h, h2) and torch.equal(y, y2)
    assert all(torch.equal(p, q) for p, q in zip(got, (want[0], *want)))
    rows = act8.unpack(c, torch.float32).cpu()                    # exact in fp32
    cpu = lambda t: None if t is None else t.cpu()  # noqa: E731
    dx, _, _, xh, g = ref.norm_backward(cpu(dy), rows, cpu(mean), cpu(rstd), cpu(w), center)
    wanted = dx + cpu(dh).double()
    limit = bound_of(dx, cpu(dh), rows, cpu(mean), cpu(rstd), xh, g, center) + ref.rounded(wanted, dtype) * 1.001
    assert ((got[0].cpu().double() - wanted).abs() <= limit).all()
    # the limit tells the projections apart: a gradient without them lies outside it
    assert ((rstd.cpu().double()[:, None] * g + cpu(dh).double() - wanted).abs() > limit).any()


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_either_result_alone(pkg, dev, center):
    """y alone: the norm's gradient from the checkpoint, for x and the residual; h alone: dh, for both, and none for the weight."""
    from faster_yoco_amd import norm
    x, res, w, b, dy, dh = (t.to(dev) for t in inputs(40, 200, torch.float32))
    args = (x, res, w, b) if center else (x, res, w)
    f = norm.add_layer_norm_train if center else norm.add_rms_norm_train
    leaves = [t.clone().requires_grad_() for t in args]
    got = torch.autograd.grad(f(*leaves, checkpoint=True)[1], leaves, dy)
    if center:
        _, _, mean, rstd, c = norm.add_layer_norm(*args, checkpoint=True)
        want = norm.layer_norm_backward(dy, c, mean, rstd, w, bias=True)
    else:
        _, _, rstd, c = norm.add_rms_norm(*args, checkpoint=True)
        want = norm.rms_norm_backward(dy, c, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(got, (want[0], *want)))
    got = torch.autograd.grad(f(*leaves, checkpoint=True)[0], leaves, dh, allow_unused=True)
    assert torch.equal(got[0], dh) and torch.equal(got[1], dh) and all(t is None for t in got[2:])
