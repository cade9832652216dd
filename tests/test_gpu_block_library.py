"""The block-side operators as PyTorch operators: torch.library.opcheck passes for each, torch.compile traces them without a
graph break, and the differentiable forms refuse a second differentiation."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(dev, *shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def test_opcheck(pkg, dev):
    from faster_yoco_amd import act8, linear8, norm
    ops = torch.ops.yoco_z1
    x, w, dy = rows(dev, 37, 300), rows(dev, 200, 300, seed=1), rows(dev, 37, 200, seed=2)
    wn, bn = rows(dev, 300, seed=3), rows(dev, 300, seed=4)
    a, p = act8.pack(x), linear8.pack_weight(w)
    _, mean, rstd = norm.layer_norm(x, wn, bn)
    checks = [(ops.act8_pack, (x,)), (ops.act8_unpack, (a.q, a.s, 300, torch.float16)),
              (ops.weight8_pack, (w, True)), (ops.weight8_pack, (w, False)),
              (ops.product8, (a.q, a.s, p.q, p.s, 300, torch.float32)),
              (ops.weight_grad8, (dy, a.q, a.s, 300, torch.bfloat16)),
              (ops.norm_forward, (x, wn, bn, 1e-5, True, False, False)),
              (ops.norm_forward, (x, wn, None, 1e-5, False, True, True)),
              (ops.norm_backward, (x, x, None, None, mean, rstd, wn, True, True, True)),
              (ops.norm_backward, (x, None, a.q, a.s, None, rstd, None, False, False, False))]
    eight = (torch.float8_e4m3fn, torch.float8_e8m0fnu)
    for op, args in checks:
        out = op(*args)
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        tensors = [t for t in args if isinstance(t, torch.Tensor)]
        # the schema's test compares by products, which torch lacks for 8-bit types: no two tensors share memory
        own = [t.untyped_storage().data_ptr() for t in out]
        assert len(set(own)) == len(own) and not set(own) & {t.untyped_storage().data_ptr() for t in tensors}
        tests = () if any(t.dtype in eight for t in tensors + out) else ('test_schema',)
        res = torch.library.opcheck(op, args, test_utils=tests + ('test_faketensor', 'test_aot_dispatch_dynamic'))
        assert all(v == 'SUCCESS' for v in res.values()), (op, res)


def test_compiled_without_a_break(pkg, dev):
    from faster_yoco_amd import act8, linear8, norm

    def step(x, wn, w, dy):
        p = linear8.pack_weight(w)
        a, rstd, kept = norm.rms_norm(x, wn, y8=True, checkpoint=True)
        y = linear8.matmul(a, p)
        dw = linear8.weight_grad(dy, a)
        da = linear8.matmul(act8.pack(dy), p, transposed=True)
        dx, dwn = norm.rms_norm_backward(da, kept, rstd, wn)
        return y * 2, dw, dx, dwn, act8.unpack(kept)

    args = (rows(dev, 64, 384), rows(dev, 384, seed=1), rows(dev, 256, 384, seed=2), rows(dev, 64, 256, seed=3))
    want = step(*args)
    got = torch.compile(step, fullgraph=True, backend='aot_eager')(*args)
    for g, v in zip(got, want):
        assert torch.equal(g, v)


def test_second_derivatives_are_refused(pkg, dev):
    from faster_yoco_amd import linear8, norm
    x, w = rows(dev, 8, 256).requires_grad_(), rows(dev, 128, 256, seed=1).requires_grad_()
    for y in (norm.rms_norm_train(x), linear8.linear(x, w, linear8.pack_weight(w.detach()))):
        g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.float().square().sum().backward()
