"""Layer norm and RMS norm on the GPU against a plain 64-bit form, forward and backward, with 8-bit results and
checkpoints.

Bounds.  u = 2^-24.  A row's mean is a sum of at most 16 serial additions per lane and a tree of at most 10 more levels
(rows longer than 16384: dim / 8192 * 8 serial ones), so it is within 64 u of mean |x| for the sizes here, and so is every
other row sum; x - mean, the product with rstd (itself within 40 u) and the weight add a few roundings of values no larger
than m = max |x - mean| + max |x|.  A result is thus within 128 u m rstd |w| (and of |b|) before its last rounding."""
import pytest
import torch

import blocks as ref
from blocks import DTYPES, U

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 7), (5, 8), (17, 129), (4, 512), (33, 1000), (2, 1537), (9, 2048), (3, 2049), (6, 4099), (2, 8192),
         (2, 16384), (3, 16385), (2, 40001)]


def inputs(n, dim, dtype, seed=0, offset=0.3, w_dtype=None):
    g = torch.Generator().manual_seed(seed + n * 131 + dim)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (r(n, dim) * torch.exp(0.5 * r(1, dim)) + offset).to(dtype)
    w, b = (1 + 0.3 * r(dim)).to(w_dtype or dtype), (0.5 * r(dim)).to(w_dtype or dtype)
    dy = (r(n, dim) * torch.exp(0.7 * r(n, 1))).to(dtype)
    return x, w, b, dy


def forward_bound(x, w, b, y, mean, rstd):
    m = (x.double() - mean[:, None]).abs().amax(1) + x.double().abs().amax(1)
    k = (m * rstd)[:, None] * (w.double().abs() if w is not None else 1.0) + y.abs()
    return 128 * U * (k + (b.double().abs() if b is not None else 0.0))


def check_forward(pkg, dev, x, w, b, eps, center):
    from faster_yoco_amd import norm
    g = [None if t is None else t.to(dev) for t in (x, w, b)]
    out = norm.layer_norm(*g, eps) if center else norm.rms_norm(g[0], g[1], eps)
    y, mean, rstd = ref.norm(x, w, b, eps, center)
    assert out[0].dtype == x.dtype and out[0].shape == x.shape
    assert ((out[-1].cpu().double() - rstd).abs() <= 64 * U * rstd).all()
    if center:
        assert ((out[1].cpu().double() - mean).abs() <= 64 * U * x.double().abs().mean(1) + 1e-45).all()
    got = out[0].cpu().double()
    assert ((got - y).abs() <= forward_bound(x, w, b, y, mean, rstd) + ref.rounded(y, x.dtype) * 1.001).all()
    return out


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', SIZES)
def test_forward(pkg, dev, n, dim, dtype, center):
    x, w, b, _ = inputs(n, dim, dtype)
    check_forward(pkg, dev, x, w, b if center else None, 1e-5, center)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_forward_without_weights_and_with_fp32_ones(pkg, dev, center):
    for dim in (200, 3000):
        x, w, b, _ = inputs(7, dim, torch.bfloat16)
        check_forward(pkg, dev, x, None, None, 1e-6, center)
        x, w, b, _ = inputs(7, dim, torch.bfloat16, w_dtype=torch.float32)
        check_forward(pkg, dev, x, w, b if center else None, 0.0, center)
        check_forward(pkg, dev, x, w, None, 1e-2, center)
        if center:
            check_forward(pkg, dev, x, None, b, 1e-5, True)


def test_a_large_common_offset_keeps_its_digits(pkg, dev):
    """Mean 1000, deviation 1: the variance is taken about the mean."""
    x, w, b, _ = inputs(5, 1500, torch.float32, offset=1000.0)
    check_forward(pkg, dev, x, w, b, 1e-5, True)


@pytest.mark.parametrize('dim', [640, 20000])
def test_rows_that_are_constant_zero_or_not_finite(pkg, dev, dim):
    from faster_yoco_amd import norm
    x, w, b, dy = inputs(6, dim, torch.bfloat16)
    x[0], x[1] = 0.0, 2.0
    x[2, 3], x[3, 5] = float('inf'), float('nan')
    y, mean, rstd = norm.layer_norm(x.to(dev), w.to(dev), b.to(dev), 1e-5)
    assert torch.equal(y[0].cpu(), b) and torch.equal(y[1].cpu(), b)           # no deviation: the bias alone
    assert y[2].isnan().all() and y[3].isnan().all()
    assert y[4:].isfinite().all()
    z, r = norm.rms_norm(x.to(dev), w.to(dev), 1e-5)
    assert not z[0].any() and z[3].isnan().all() and z[4:].isfinite().all()
    a, r2, c = norm.rms_norm(x.to(dev), w.to(dev), 1e-5, y8=True, checkpoint=True)
    q, s = ref.pack(x)
    assert ref.same_codes(c.q, q) and torch.equal(ref.codes(c.s), s)
    assert torch.equal(r2[4:], r[4:]) and (ref.codes(a.q)[3, :dim] & 127 == 127).all()
    dx, dw, db = norm.layer_norm_backward(dy.to(dev), x.to(dev), mean, rstd, w.to(dev), bias=True)
    assert dx[[0, 1, 4, 5]].isfinite().all() and dx[3].isnan().all() and db.isfinite().all()


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', [(1, 1), (3, 130), (9, 512), (5, 1000), (3, 2049), (2, 4099), (2, 9000), (2, 20001)])
def test_eight_bit_results(pkg, dev, n, dim, dtype, center):
    """The checkpoint is x's 8-bit rows exactly.  y in 8 bits is within its bound of y, then half a step of its scale."""
    from faster_yoco_amd import norm
    x, w, b, _ = inputs(n, dim, dtype, 5)
    d = [t.to(dev) for t in (x, w, b)]
    out = norm.layer_norm(*d, y8=True, checkpoint=True) if center else norm.rms_norm(d[0], d[1], y8=True, checkpoint=True)
    a, c = out[0], out[-1]
    q, s = ref.pack(x)
    assert ref.same_codes(c.q, q) and torch.equal(ref.codes(c.s), s) and c.dim == a.dim == dim
    y, mean, rstd = ref.norm(x, w, b if center else None, 1e-5, center)
    qa, sa = ref.codes(a.q), ref.codes(a.s)
    got = ref.values(qa, sa, dim)
    near = forward_bound(x, w, b if center else None, y, mean, rstd)
    scale = 2.0 ** (sa.double().repeat_interleave(128, 1)[:, :dim] - 127)
    assert ((got - y).abs() <= near + torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10)).all()
    blocks = ref.exponents(torch.nn.functional.pad(y.abs(), (0, -dim % 128)).view(n, -1, 128).amax(2))
    assert (sa[:, :blocks.shape[1]].double() - 127 - blocks).abs().max() <= 1
    assert (sa[:, blocks.shape[1]:] == 127).all() and not qa[:, dim:].any()
    plain = norm.layer_norm(*d) if center else norm.rms_norm(d[0], d[1])
    assert all(torch.equal(p, o) for p, o in zip(plain[1:], out[1:]))         # the same statistics


def check_backward(pkg, dev, x, dy, w, center, packed):
    from faster_yoco_amd import act8, norm
    n, dim = x.shape
    _, mean, rstd = ref.norm(x, None, None, 1e-5, center)
    mean, rstd = mean.float(), rstd.float()
    if packed:
        q, s = ref.pack(x)
        given = act8.Act8(q.to(dev).view(ref.F8), s.to(dev).view(ref.E8), dim)
        x = ref.values(q, s, dim)
    else:
        given = x.to(dev)
    wd = None if w is None else w.to(dev)
    if center:
        out = norm.layer_norm_backward(dy.to(dev), given, mean.to(dev), rstd.to(dev), wd, bias=True)
    else:
        out = norm.rms_norm_backward(dy.to(dev), given, rstd.to(dev), wd)
    dx, dw, db, xh, g = ref.norm_backward(dy, x, mean, rstd, w, center)
    want = [dx] + ([dw] if w is not None else []) + ([db] if center else [])
    assert len(out) == len(want)
    # row sums within 64 u of their terms' sizes; what they are subtracted from and multiplied with rounds a few times
    size = g.abs() + (g.abs().mean(1) + 0)[:, None] + xh.abs() * (g * xh).abs().mean(1)[:, None]
    m = rstd.double()[:, None] * (x.double().abs() + (mean.double().abs()[:, None] if center else 0))      # xh's terms
    size = size + m * (g * xh).abs().mean(1)[:, None] + xh.abs() * (g.abs() * m).mean(1)[:, None]
    bound = 128 * U * rstd.double()[:, None] * size + ref.rounded(dx, dy.dtype) * 1.001
    assert ((out[0].cpu().double() - dx).abs() <= bound).all()
    gt = w.dtype if w is not None else dy.dtype
    sums = [(dy.double().abs() * m).sum(0)] * (w is not None) + [dy.double().abs().sum(0)] * center
    for got, v, a in zip(out[1:], want[1:], sums):
        assert got.dtype == gt and got.shape == (dim,)
        assert ((got.cpu().double() - v).abs() <= (n + 16) * U * a + ref.rounded(v, gt) * 1.001).all()


@pytest.mark.parametrize('packed', [False, True], ids=['x', 'checkpoint'])
@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', SIZES + [(700, 260), (3000, 64), (1100, 1100)])
def test_backward(pkg, dev, n, dim, dtype, center, packed):
    x, w, _, dy = inputs(n, dim, dtype, 9)
    check_backward(pkg, dev, x, dy, w, center, packed)


@pytest.mark.parametrize('packed', [False, True], ids=['x', 'checkpoint'])
@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', [(2561, 9), (2600, 513), (2570, 1537), (2900, 2560), (1030, 8200), (600, 14000)])
def test_backward_of_many_rows(pkg, dev, n, dim, dtype, center, packed):
    """Partial sums and a second launch."""
    from faster_yoco_amd import _lib
    assert _lib.lib().z1_norm_backward_workspace(n, dim) > 0
    x, w, _, dy = inputs(n, dim, dtype, 12)
    check_backward(pkg, dev, x, dy, w, center, packed)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('n,dim', [(511, 15), (512, 8), (513, 17), (1024, 129), (1537, 520), (2560, 31), (90, 16384)])
def test_backward_of_few_rows(pkg, dev, n, dim, center):
    """One launch: whole and partial turns of its rows, strips of columns that end inside."""
    from faster_yoco_amd import _lib, norm
    assert _lib.lib().z1_norm_backward_workspace(n, dim) == 0
    x, w, _, dy = inputs(n, dim, torch.bfloat16, 13)
    for packed in (False, True):
        check_backward(pkg, dev, x, dy, w, center, packed)
    if center:                                         # dw and db each without the other
        g = [t.to(dev) for t in (dy, x, w)]
        _, mean, rstd = norm.layer_norm(g[1], g[2])
        both = norm.layer_norm_backward(g[0], g[1], mean, rstd, g[2], bias=True)
        assert torch.equal(norm.layer_norm_backward(g[0], g[1], mean, rstd, g[2])[1], both[1])
        op = torch.ops.yoco_z1.norm_backward
        assert torch.equal(op(g[0], g[1], None, None, mean, rstd, g[2], True, False, True)[1], both[2])
        assert torch.equal(op(g[0], g[1], None, None, mean, rstd, g[2], True, False, False)[0], both[0])


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_backward_without_weight_and_with_fp32_one(pkg, dev, center):
    for dim in (300, 17000):
        x, w, _, dy = inputs(20, dim, torch.bfloat16, 10, w_dtype=torch.float32)
        check_backward(pkg, dev, x, dy, None, center, False)
        check_backward(pkg, dev, x, dy, w, center, False)
        check_backward(pkg, dev, x, dy, w, center, True)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_gradients_match_differences(pkg, dev, center):
    """Central differences of sum(dy * y) in 64 bits, step 1e-5: their own error is far below the bound of 1e-5 relative
    to the gradient's size that fp32 kernels are held to here."""
    from faster_yoco_amd import norm
    n, dim = 3, 37
    x, w, b, dy = inputs(n, dim, torch.float32, 11)
    f = lambda x, w, b: (dy.double() * ref.norm(x, w, b, 1e-5, center)[0]).sum()  # noqa: E731
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    y = norm.layer_norm_train(*leaves) if center else norm.rms_norm_train(*leaves[:2])
    y.backward(dy.to(dev))
    for i, t in enumerate((x, w, b) if center else (x, w)):
        t = t.double()
        want = torch.zeros_like(t).view(-1)
        for k in range(t.numel()):
            hi, lo = t.clone(), t.clone()
            hi.view(-1)[k] += 1e-5
            lo.view(-1)[k] -= 1e-5
            args = [x.double(), w.double(), b.double() if center else None]
            up, down = list(args), list(args)
            up[i], down[i] = hi, lo
            want[k] = (f(*up) - f(*down)) / 2e-5
        got = leaves[i].grad.cpu().double().view(-1)
        assert (got - want).abs().max() <= 1e-5 * want.abs().max()


def test_strides_and_leading_dimensions(pkg, dev):
    from faster_yoco_amd import norm
    base, w, b, dyb = inputs(30, 901, torch.bfloat16, 12)
    w, b = w[:700].contiguous(), b[:700].contiguous()
    for sl in (lambda t: t[:, 5:705], lambda t: t[::2, 1:701]):
        x, dy = sl(base), sl(dyb)
        got = norm.layer_norm(sl(base.to(dev)), w.to(dev), b.to(dev))
        want = norm.layer_norm(x.contiguous().to(dev), w.to(dev), b.to(dev))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        got = norm.layer_norm_backward(sl(dyb.to(dev)), sl(base.to(dev)), *want[1:], w.to(dev), bias=True)
        back = norm.layer_norm_backward(dy.contiguous().to(dev), x.contiguous().to(dev), *want[1:], w.to(dev), bias=True)
        assert all(torch.equal(p, q) for p, q in zip(got, back))
    x = base.to(dev)[:, :700]
    y3 = norm.rms_norm(x.reshape(5, 6, 700), w.to(dev))[0]
    assert y3.shape == (5, 6, 700) and torch.equal(y3.view(30, 700), norm.rms_norm(x, w.to(dev))[0])
    xt = base.to(dev).t()[:700]                                                # elements apart: copied
    assert torch.equal(norm.rms_norm(xt)[0], norm.rms_norm(xt.contiguous())[0])
    y1, r1 = norm.rms_norm(x[0], w.to(dev))
    assert y1.shape == (700,) and torch.equal(y1, y3[0, 0])
    leaf = x.clone().requires_grad_()
    norm.rms_norm_train(leaf, w.to(dev)).sum().backward()                      # a broadcast gradient
    one = torch.ones_like(x)
    assert torch.equal(leaf.grad, norm.rms_norm_backward(one, x, norm.rms_norm(x, w.to(dev))[1], w.to(dev))[0])


def test_same_bits_every_time_and_on_another_stream(pkg, dev):
    from faster_yoco_amd import norm
    x, w, b, dy = (t.to(dev) for t in inputs(1500, 777, torch.bfloat16, 13))
    y, mean, rstd = norm.layer_norm(x, w, b)
    first = norm.layer_norm_backward(dy, x, mean, rstd, w, bias=True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = norm.layer_norm_backward(dy, x, mean, rstd, w, bias=True)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = norm.layer_norm(x, w, b)
        r = norm.layer_norm_backward(dy, x, o[1], o[2], w, bias=True)
    for seed in (14, 15, 16):
        x2, _, _, dy2 = inputs(1500, 777, torch.bfloat16, seed)
        x.copy_(x2.to(dev))
        dy.copy_(dy2.to(dev))
        want = norm.layer_norm(x, w, b)
        back = norm.layer_norm_backward(dy, x, want[1], want[2], w, bias=True)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip((*o, *r), (*want, *back)))


def test_training_form_keeps_the_checkpoint(pkg, dev):
    from faster_yoco_amd import act8, norm
    x, w, b, dy = (t.to(dev) for t in inputs(64, 640, torch.bfloat16, 17))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    norm.layer_norm_train(*leaves, checkpoint=True).backward(dy)
    y, mean, rstd, a = norm.layer_norm(x, w, b, checkpoint=True)
    assert isinstance(a, act8.Act8) and a.nbytes() < x.numel() * 1.02
    for got, want in zip(leaves, norm.layer_norm_backward(dy, a, mean, rstd, w, bias=True)):
        assert torch.equal(got.grad, want)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_no_rows(pkg, dev, center):
    from faster_yoco_amd import norm
    x = torch.empty(0, 300, dtype=torch.bfloat16, device=dev)
    w = torch.ones(300, dtype=torch.bfloat16, device=dev)
    if center:
        y, mean, rstd = norm.layer_norm(x, w, w)
        out = norm.layer_norm_backward(x, x, mean, rstd, w, bias=True)
    else:
        y, rstd = norm.rms_norm(x, w)
        out = norm.rms_norm_backward(x, x, rstd, w)
    assert y.shape == (0, 300) and out[0].shape == (0, 300)
    assert all(not t.any() and t.shape == (300,) for t in out[1:])             # sums of nothing


def test_refusals(pkg, dev):
    from faster_yoco_amd import act8, norm
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    w, r = torch.ones(256, dtype=torch.bfloat16, device=dev), torch.ones(4, device=dev)
    with pytest.raises(RuntimeError, match='no CPU path'):
        norm.layer_norm(x.cpu())
    with pytest.raises(RuntimeError, match='no CPU path'):
        norm.layer_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match='at least one column'):
        norm.rms_norm(x[:, :0])
    with pytest.raises(RuntimeError, match='expected fp32, bf16 or fp16'):
        norm.rms_norm(x.double())
    with pytest.raises(RuntimeError, match='weight: expected'):
        norm.layer_norm(x, w[:255])
    with pytest.raises(RuntimeError, match="the rows' type"):
        norm.layer_norm(x, w.half())
    with pytest.raises(RuntimeError, match='one type'):
        norm.layer_norm(x, w, w.float())
    with pytest.raises(RuntimeError, match='eps'):
        norm.layer_norm(x, w, eps=-1.0)
    with pytest.raises(RuntimeError, match='one shape and type'):
        norm.rms_norm_backward(x, x.float(), r, w)
    with pytest.raises(RuntimeError, match='one shape and type'):
        norm.rms_norm_backward(x, x[:3], r, w)
    with pytest.raises(RuntimeError, match='rstd'):
        norm.rms_norm_backward(x, x, r[:3], w)
    with pytest.raises(RuntimeError, match='mean'):
        norm.layer_norm_backward(x, x, r.double(), r, w)
    with pytest.raises(RuntimeError, match='checkpoint of 200 columns'):
        norm.rms_norm_backward(x, act8.pack(x[:, :200]), r, w)
    with pytest.raises(RuntimeError, match='values'):
        norm.rms_norm_backward(x, act8.pack(x[:3]), r, w)


@pytest.mark.parametrize('packed', [False, True], ids=['x', 'checkpoint'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize('n,dim', [(3, 130), (5, 1537), (3, 4099), (2600, 137), (2600, 1030), (2, 20001)])
def test_backward_of_rows_of_one_large_value(pkg, dev, n, dim, dtype, packed):
    """x = mean = 2^120 and rstd = 316: (x - mean) rstd is 0 in the row, and mean * rstd, which the columns past its end would
    bring in, beyond fp32."""
    x, w, _, dy = inputs(n, dim, dtype, 21)
    x[0], x[-1] = 2.0 ** 120, 2.0 ** 120
    check_backward(pkg, dev, x, dy, w, True, packed)


@pytest.mark.parametrize('n,dim', [(300, 200), (3000, 520), (40, 20001)])
def test_gradient_of_an_fp32_bias_without_a_weight(pkg, dev, n, dim):
    """db has the bias's type: the fp32 sum itself, not one rounded to the rows' type."""
    from faster_yoco_amd import norm
    x, _, b, dy = inputs(n, dim, torch.bfloat16, 23, w_dtype=torch.float32)
    xd, dyd, bd = x.to(dev), dy.to(dev), b.to(dev).requires_grad_()
    norm.layer_norm_train(xd, None, bd).backward(dyd)
    want, size = dy.double().sum(0), dy.double().abs().sum(0)
    assert bd.grad.dtype == torch.float32
    assert ((bd.grad.cpu().double() - want).abs() <= (n + 16) * U * size + ref.rounded(want, torch.float32) * 1.001).all()
    _, mean, rstd = norm.layer_norm(xd, None, bd.detach())
    _, db = norm.layer_norm_backward(dyd, xd, mean, rstd, bias=True, grad_dtype=torch.float32)
    assert db.dtype == torch.float32 and torch.equal(db, bd.grad)
    assert torch.equal(norm.layer_norm_backward(dyd, xd, mean, rstd, bias=True)[1], db.bfloat16())
    with pytest.raises(RuntimeError, match='expected fp32, bf16 or fp16'):
        norm.layer_norm_backward(dyd, xd, mean, rstd, bias=True, grad_dtype=torch.float64)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('dim', [1300, 3000, 5300, 9001, 10240, 12288, 12289])
def test_forward_of_every_width_that_registers_hold(pkg, dev, dim, dtype, center):
    """Three to six groups of 8 columns to a lane, one to four waves to a row, and the first width beyond."""
    x, w, b, _ = inputs(5, dim, dtype, 27)
    check_forward(pkg, dev, x, w, b if center else None, 1e-5, center)
