"""The residual stream's addition and norm in one pass, and its gradients, on the GPU.

h is one addition of two values of its type, rounded to that type: exact against the same in 64 bits (a sum of two fp32, bf16
or fp16 values rounded once; for 16-bit types by way of fp32, whose own rounding can only decide a tie of the second one, so
those are compared with torch's fp32 sum rounded).  The rest is the norm of that h: the same bits as ``norm``'s own operators
give for it, and within their bounds of the 64-bit form.

Bounds of dx.  The norm's part is within 128 u r (sizes) of its 64-bit value, as in the plain norm's gradient (its derivation:
tests/test_gpu_norm.py); adding dh rounds once more in fp32, u (|part| + |dh|), and then to the type."""
import pytest
import torch

import blocks as ref
from blocks import DTYPES, U

pytestmark = pytest.mark.gpu

# one element to a few, a wave's access and its neighbours, rows of 1, 2, 4 waves, rows that are read again
SIZES = [(1, 1), (3, 7), (5, 8), (17, 129), (4, 512), (33, 1000), (2, 1537), (9, 2048), (6, 4099), (2, 8192), (2, 12288),
         (2, 12289), (3, 16385), (2, 40001)]


def inputs(n, dim, dtype, seed=0, w_dtype=None):
    g = torch.Generator().manual_seed(seed + n * 131 + dim)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (0.3 * r(n, dim)).to(dtype)
    res = (r(n, dim) * torch.exp(0.5 * r(1, dim)) + 0.3).to(dtype)
    w, b = (1 + 0.3 * r(dim)).to(w_dtype or dtype), (0.5 * r(dim)).to(w_dtype or dtype)
    dy, dh = ((r(n, dim) * torch.exp(0.7 * r(n, 1))).to(dtype) for _ in range(2))
    return x, res, w, b, dy, dh


def summed(x, res):
    return (x.float() + res.float()).to(x.dtype)


def same(a, b):
    return torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


def check_forward(dev, x, res, w, b, center, eps=1e-5):
    from faster_yoco_amd import norm
    d = [None if t is None else t.to(dev) for t in (x, res, w, b)]
    h = summed(x, res)
    for y8 in (False, True):
        for checkpoint in (False, True):
            kw = dict(y8=y8, checkpoint=checkpoint)
            if center:
                got, want = norm.add_layer_norm(*d, eps, **kw), norm.layer_norm(h.to(dev), *d[2:], eps, **kw)
            else:
                got, want = norm.add_rms_norm(*d[:3], eps, **kw), norm.rms_norm(h.to(dev), d[2], eps, **kw)
            assert got[0].dtype == x.dtype and torch.equal(got[0].cpu(), h)
            assert len(got) == len(want) + 1
            for g, v in zip(got[1:], want):
                if isinstance(v, torch.Tensor):
                    assert g.dtype == v.dtype and g.shape == v.shape and torch.equal(g, v)
                else:
                    assert same(g.q, v.q) and same(g.s, v.s) and g.dim == v.dim
    y, mean, rstd = ref.norm(h, w, b if center else None, eps, center)
    out = norm.add_layer_norm(*d, eps) if center else norm.add_rms_norm(*d[:3], eps)
    m = (h.double() - mean[:, None]).abs().amax(1) + h.double().abs().amax(1)
    k = (m * rstd)[:, None] * (w.double().abs() if w is not None else 1.0) + y.abs()
    bound = 128 * U * (k + (b.double().abs() if b is not None and center else 0.0)) + ref.rounded(y, x.dtype) * 1.001
    assert ((out[1].cpu().double() - y).abs() <= bound).all()


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', SIZES)
def test_forward(pkg, dev, n, dim, dtype, center):
    x, res, w, b, _, _ = inputs(n, dim, dtype)
    check_forward(dev, x, res, w, b, center)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_forward_without_weights_and_with_fp32_ones(pkg, dev, center):
    for dim in (200, 3000, 13000):
        x, res, w, b, _, _ = inputs(7, dim, torch.bfloat16, w_dtype=torch.float32)
        check_forward(dev, x, res, None, None, center, 1e-6)
        check_forward(dev, x, res, w, b, center, 0.0)


def test_a_sum_that_cancels_or_leaves_the_type(pkg, dev):
    """h = 0, infinite sums, NaN: the row's results are those of the norm of that h, and no other row changes."""
    from faster_yoco_amd import norm
    for dim in (640, 20000):
        x, res, w, b, _, _ = inputs(6, dim, torch.float16, 3)
        res[0] = -x[0]
        x[1, 3], res[1, 3] = 60000.0, 60000.0                     # past fp16's largest
        x[2, 5], res[2, 5] = float('inf'), float('-inf')
        d = [t.to(dev) for t in (x, res, w)]
        h, y, rstd = norm.add_rms_norm(*d)
        y2, r2 = norm.rms_norm(h, d[2])
        assert not h[0].any() and not y[0].any() and h[1, 3] == float('inf') and h[2, 5].isnan()
        assert torch.equal(y.nan_to_num(7.0), y2.nan_to_num(7.0)) and torch.equal(rstd.nan_to_num(7.0), r2.nan_to_num(7.0))
        assert y[3:].isfinite().all()


def check_backward(dev, x, res, w, dy, dh, center, packed):
    from faster_yoco_amd import act8, norm
    h = summed(x, res)
    n, dim = h.shape
    _, mean, rstd = ref.norm(h, None, None, 1e-5, center)
    mean, rstd = mean.float(), rstd.float()
    if packed:
        q, s = ref.pack(h)
        given, h = act8.Act8(q.to(dev).view(ref.F8), s.to(dev).view(ref.E8), dim), ref.values(q, s, dim)
    else:
        given = h.to(dev)
    d = [None if t is None else t.to(dev) for t in (dy, dh, mean, rstd, w)]
    if center:
        out = norm.add_layer_norm_backward(d[0], d[1], given, *d[2:], bias=True)
        plain = norm.layer_norm_backward(d[0], given, *d[2:], bias=True)
    else:
        out = norm.add_rms_norm_backward(d[0], d[1], given, *d[3:])
        plain = norm.rms_norm_backward(d[0], given, *d[3:])
    assert len(out) == len(plain) == 1 + (w is not None) + center
    for g, v in zip(out[1:], plain[1:]):
        assert g.dtype == v.dtype and torch.equal(g, v)           # dw and db do not see dh
    dx, _, _, xh, g = ref.norm_backward(dy, h, mean, rstd, w, center)
    size = g.abs() + g.abs().mean(1)[:, None] + xh.abs() * (g * xh).abs().mean(1)[:, None]
    m = rstd.double()[:, None] * (h.double().abs() + (mean.double().abs()[:, None] if center else 0))
    size = size + m * (g * xh).abs().mean(1)[:, None] + xh.abs() * (g.abs() * m).mean(1)[:, None]
    want = dx + dh.double()
    bound = 128 * U * rstd.double()[:, None] * size + U * (dx.abs() + dh.double().abs()) * 1.001
    assert out[0].dtype == dy.dtype and out[0].shape == dy.shape
    got, limit = out[0].cpu().double(), bound + ref.rounded(want, dy.dtype) * 1.001
    # what lies past the type's largest value by more than its bound is infinite there (one column's checkpoint is off its mean by
    # up to 2^-4, times rstd = 316: fp16 ends at 65504)
    past = want.abs() - limit > ref.LARGEST[dy.dtype]
    assert torch.equal(got[past], torch.copysign(torch.full_like(want, float('inf')), want)[past])
    assert ((got - want).abs() <= limit)[~past].all()


@pytest.mark.parametrize('packed', [False, True], ids=['h', 'checkpoint'])
@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', SIZES + [(700, 260), (3000, 64), (2570, 1537), (1030, 8200), (600, 14000)])
def test_backward(pkg, dev, n, dim, dtype, center, packed):
    """Few rows (one launch), many (two), long rows (read twice)."""
    x, res, w, _, dy, dh = inputs(n, dim, dtype, 9)
    check_backward(dev, x, res, w, dy, dh, center, packed)


@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_backward_without_weight_and_with_fp32_one(pkg, dev, center):
    for n, dim in ((20, 300), (20, 17000), (2600, 130)):
        x, res, w, _, dy, dh = inputs(n, dim, torch.bfloat16, 10, w_dtype=torch.float32)
        check_backward(dev, x, res, None, dy, dh, center, False)
        check_backward(dev, x, res, w, dy, dh, center, True)


@pytest.mark.parametrize('n,dim', [(11, 515), (2600, 515), (5, 16500)])
def test_strided_rows(pkg, dev, n, dim):
    """Rows that start at any element, each tensor with a stride of its own, one row for all (stride 0), leading dimensions,
    and columns that are not neighbours (copied)."""
    from faster_yoco_amd import norm
    x, res, w, b, dy, dh = inputs(n, dim, torch.bfloat16, 4)

    def inside(t, before, after):
        big = torch.full((n, before + dim + after), float('nan'), dtype=t.dtype, device=dev)
        big[:, before:before + dim] = t.to(dev)
        return big[:, before:before + dim]
    d = [t.to(dev) for t in (x, res, w, b, dy, dh)]
    v = [inside(x, 1, 2), inside(res, 3, 0), d[2], d[3], inside(dy, 5, 1), inside(dh, 0, 7)]
    want, got = norm.add_layer_norm(*d[:4]), norm.add_layer_norm(*v[:4])
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    h, _, mean, rstd = want
    grads = norm.add_layer_norm_backward(d[4], d[5], h, mean, rstd, d[2], bias=True)
    hv = inside(h.cpu(), 2, 1)
    assert all(torch.equal(a, c) for a, c in
               zip(grads, norm.add_layer_norm_backward(v[4], v[5], hv, mean, rstd, d[2], bias=True)))
    one = d[1][:1].expand(n, dim)                                 # one residual row for all
    assert torch.equal(norm.add_rms_norm(d[0], one, d[2])[1], norm.add_rms_norm(d[0], one.contiguous(), d[2])[1])
    t = d[0].t().contiguous().t()                                 # columns apart
    assert torch.equal(norm.add_layer_norm(t, *d[1:4])[1], want[1])
    three = norm.add_layer_norm(d[0][None], d[1][None], d[2], d[3], y8=True, checkpoint=True)
    assert three[0].shape == (1, n, dim) and torch.equal(three[0][0], h) and three[1].rows == n


def test_rows_past_32_bits_apart(pkg, dev):
    from faster_yoco_amd import norm
    x, res, w, b, dy, dh = (t.to(dev) for t in inputs(3, 515, torch.bfloat16, 9))
    flat = torch.empty((1 << 31) + 4000, dtype=torch.bfloat16, device=dev)
    far = [flat[i * 600:].as_strided((3, 515), ((1 << 30) + 3, 1)) for i in range(4)]
    for t, v in zip((x, res, dy, dh), far):
        v.copy_(t)
    want, got = norm.add_layer_norm(x, res, w, b), norm.add_layer_norm(far[0], far[1], w, b)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    h, _, mean, rstd = want
    assert all(torch.equal(p, q) for p, q in zip(norm.add_layer_norm_backward(dy, dh, h, mean, rstd, w, bias=True),
                                                 norm.add_layer_norm_backward(far[2], far[3], h, mean, rstd, w, bias=True)))


def test_one_tensor_as_both(pkg, dev):
    """h = 2 x, exactly; x's gradient is twice dx."""
    from faster_yoco_amd import norm
    x, _, w, _, dy, dh = (None if t is None else t.to(dev) for t in inputs(7, 300, torch.float32, 10))
    a, r = x.clone().requires_grad_(), [t.clone().requires_grad_() for t in (x, x)]
    for args in ((a, a), r):
        h, y = norm.add_rms_norm_train(*args, w)
        assert torch.equal(h, 2 * x)
        torch.autograd.backward([h, y], [dh, dy])
    assert torch.equal(r[0].grad, r[1].grad) and torch.equal(a.grad, 2 * r[0].grad)


def test_no_rows(pkg, dev):
    from faster_yoco_amd import norm
    x, w = torch.empty(0, 300, device=dev, dtype=torch.bfloat16), torch.ones(300, device=dev, dtype=torch.bfloat16)
    h, y, rstd = norm.add_rms_norm(x, x, w)
    assert h.shape == y.shape == (0, 300) and rstd.shape == (0,)
    dx, dw = norm.add_rms_norm_backward(x, x, h, rstd, w)
    assert dx.shape == (0, 300) and not dw.any()


@pytest.mark.parametrize('checkpoint', [False, True])
@pytest.mark.parametrize('center', [True, False], ids=['layer', 'rms'])
def test_train_against_autograd(pkg, dev, center, checkpoint):
    """Both results used, one of them, and x the residual itself: torch's gradients of the plain form in 64 bits.  fp32, 40
    rows of 200: every result is a sum of at most 240 terms, so within 2^9 u of their sizes, which are below 2^6; the 8-bit
    checkpoint's rows are off by 2^-4 of themselves, which enters the gradients once."""
    from faster_yoco_amd import norm
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x0, res0, w0, b0, uh, uy = r(40, 200), r(40, 200), 1 + 0.2 * r(200), 0.1 * r(200), r(40, 200), r(40, 200)
    limit = 2.0 ** 15 * U if not checkpoint else 2.0

    def leaves(device, dtype):
        return [t.to(device, dtype).requires_grad_() for t in ((x0, res0, w0, b0) if center else (x0, res0, w0))]

    def ours(v):
        f = norm.add_layer_norm_train if center else norm.add_rms_norm_train
        return f(*v, checkpoint=checkpoint)

    def plain(v):
        h = v[0] + v[1]
        c = h - h.mean(1, keepdim=True) if center else h
        y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * v[2]
        return h, y + v[3] if center else y
    for use_h, use_y in ((True, True), (True, False), (False, True)):
        got, want = leaves(dev, torch.float32), leaves('cpu', torch.float64)
        for v, f, device, dtype in ((got, ours, dev, torch.float32), (want, plain, 'cpu', torch.float64)):
            h, y = f(v)
            loss = (h * uh.to(device, dtype)).sum() * use_h + (y * uy.to(device, dtype)).sum() * use_y if use_h and use_y else \
                (h * uh.to(device, dtype)).sum() if use_h else (y * uy.to(device, dtype)).sum()
            loss.backward()
        for a, c in zip(got, want):
            if c.grad is None:
                assert a.grad is None
            else:
                assert ((a.grad.cpu().double() - c.grad).abs() <= limit).all()
        if got[0].grad is not None:
            assert torch.equal(got[0].grad, got[1].grad) and got[0].grad.data_ptr() != got[1].grad.data_ptr()
    x = x0.to(dev).requires_grad_()                               # x is the residual: twice the gradient
    h, y = (norm.add_layer_norm_train if center else norm.add_rms_norm_train)(x, x, checkpoint=checkpoint)
    (gx,) = torch.autograd.grad((h * uh.to(dev)).sum() + (y * uy.to(dev)).sum(), x)
    a, c = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    h, y = (norm.add_layer_norm_train if center else norm.add_rms_norm_train)(a, c, checkpoint=checkpoint)
    (ga,) = torch.autograd.grad((h * uh.to(dev)).sum() + (y * uy.to(dev)).sum(), a)
    assert torch.equal(gx, ga + ga)


def test_gradient_against_differences(pkg, dev):
    """Central differences of the 64-bit form along random directions against the kernel's gradient (fp32): a step of 2^-12
    leaves third-order terms of 2^-24 times third derivatives, and the fp32 gradient 2^-15 of the sizes: 1e-3 of the sum's."""
    from faster_yoco_amd import norm
    g = torch.Generator().manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, res, w, uh, uy = r(6, 50), r(6, 50), 1 + 0.2 * r(50), r(6, 50), r(6, 50)

    def loss(x, res, w):
        h = x + res
        return (h * uh).sum() + (h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5) * w * uy).sum()
    leaves = [t.float().to(dev).requires_grad_() for t in (x, res, w)]
    h, y = norm.add_rms_norm_train(*leaves)
    ((h * uh.float().to(dev)).sum() + (y * uy.float().to(dev)).sum()).backward()
    base = [t.detach().cpu().double() for t in leaves]
    for i, leaf in enumerate(leaves):
        d = r(*leaf.shape)
        step = [t + (d * 2.0 ** -12 if j == i else 0) for j, t in enumerate(base)]
        back = [t - (d * 2.0 ** -12 if j == i else 0) for j, t in enumerate(base)]
        want = float(loss(*step) - loss(*back)) * 2.0 ** 11
        terms = leaf.grad.cpu().double() * d
        assert abs(float(terms.sum()) - want) <= 1e-3 * float(terms.abs().sum())


def test_refusals(pkg, dev):
    from faster_yoco_amd import act8, norm
    x = torch.randn(6, 256, device=dev, dtype=torch.bfloat16)
    w, st = torch.ones(256, device=dev, dtype=torch.bfloat16), torch.ones(6, device=dev)
    a = act8.pack(x)
    for call, text in ((lambda: norm.add_rms_norm(x, x[:5]), 'a residual of'), (lambda: norm.add_rms_norm(x, x.float()), 'one shape'),
                       (lambda: norm.add_rms_norm(x, x[:, :128]), 'a residual of'), (lambda: norm.add_rms_norm(x, x.cpu()), 'GPU tensor'),
                       (lambda: norm.add_rms_norm(x.double(), x.double()), 'fp32, bf16 or fp16'),
                       (lambda: norm.add_rms_norm(x, x, w[:5]), 'contiguous'), (lambda: norm.add_rms_norm(x, x, eps=-1.0), 'eps'),
                       (lambda: norm.add_rms_norm_backward(x, x[:5], x, st, w), 'dh of'),
                       (lambda: norm.add_rms_norm_backward(x, x.float(), x, st, w), 'one shape'),
                       (lambda: norm.add_rms_norm_backward(x, x, x[:5], st, w), 'one shape'),
                       (lambda: norm.add_rms_norm_backward(x, x, act8.pack(x[:5]), st, w), 'contiguous values'),
                       (lambda: norm.add_rms_norm_backward(x, x, act8.pack(x[:, :128]), st, w), 'checkpoint of'),
                       (lambda: norm.add_rms_norm_backward(x, x.cpu(), a, st, w), 'GPU tensor'),
                       (lambda: norm.add_layer_norm_backward(x, x, a, None, st, w), 'means')):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_captured_on_another_stream(pkg, dev):
    """Forward and backward in a graph, on a stream of its own; each replay, with new inputs written in between, gives the
    eager results."""
    from faster_yoco_amd import norm
    x, res, w, b, dy, dh = (t.to(dev) for t in inputs(2600, 520, torch.bfloat16, 6))

    def both():
        h, y, mean, rstd, c = norm.add_layer_norm(x, res, w, b, checkpoint=True)
        return [h, y, mean, rstd, c.q.view(torch.uint8), *norm.add_layer_norm_backward(dy, dh, c, mean, rstd, w, bias=True),
                *norm.add_layer_norm_backward(dy[:9], dh[:9], h[:9], mean[:9], rstd[:9], w, bias=True)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = both()
    torch.cuda.synchronize()
    for k in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)))
        dh.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_as_operators(pkg, dev):
    ops = torch.ops.yoco_z1
    x, res, w, b, dy, dh = (t.to(dev) for t in inputs(37, 300, torch.bfloat16, 7))
    h, y, mean, rstd = ops.add_norm_forward(x, res, w, b, 1e-5, True, False, False)
    for op, args in ((ops.add_norm_forward, (x, res, w, b, 1e-5, True, False, False)),
                     (ops.add_norm_forward, (x, res, w, None, 1e-5, False, False, False)),
                     (ops.add_norm_backward, (dy, dh, h, None, None, mean, rstd, w, True, True, True))):
        res_ = torch.library.opcheck(op, args, test_utils=('test_schema', 'test_faketensor', 'test_aot_dispatch_dynamic'))
        assert all(v == 'SUCCESS' for v in res_.values()), res_
    args = (x, res, w, None, 1e-5, False, True, True)             # 8-bit results: torch's schema test has no products of them
    res_ = torch.library.opcheck(ops.add_norm_forward, args, test_utils=('test_faketensor', 'test_aot_dispatch_dynamic'))
    assert all(v == 'SUCCESS' for v in res_.values()), res_
