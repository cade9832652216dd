"""Orthogonalised matrices and the matrices' step on the GPU against plain 64-bit forms (bounds: matrices.py)."""
import math

import pytest
import torch

import matrices as ref
import ways_muon
from matrices import HALF

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# one row or column, less than a block and a tile, their neighbours, tall and wide, every tile's size and its ends
SHAPES = [(1, 1), (1, 9), (7, 1), (2, 2), (3, 5), (16, 16), (17, 100), (63, 64), (65, 64), (64, 65), (128, 130), (100, 37),
          (31, 33), (32, 2048), (2048, 20), (64, 1000), (96, 300),
          (129, 131), (200, 333), (257, 256), (300, 1000), (511, 129), (128, 512), (127, 600), (512, 120), (130, 4000)]
KINDS = ['noise', 'strong', 'falling', 'flat']


def gen(*key):
    return torch.Generator().manual_seed(hash(key) % (1 << 31) if not all(isinstance(k, int) for k in key) else
                                         sum(k * 1009 ** i for i, k in enumerate(key)) % (1 << 31))


def matrix(m, n, kind='noise', dtype=torch.float32, scale=1e-3):
    return (ref.spectrum(m, n, kind, gen(m, n, KINDS.index(kind))) * scale).to(dtype)


def far(got, want):
    return float((got.double().cpu() - want).norm())


def limit(x, out, precise, **kw):
    """Four times the distance that the stored roundings leave, and the result's own rounding of every element."""
    want = ref.exact(x, **kw)
    near = float((ref.stored(x, precise=precise, **kw) - want).norm())
    floor = 2.0 ** -20 if precise else 2.0 ** -13       # of the norm: what a draw of few roundings may hide
    return want, 4 * near + floor * float(want.norm()) + HALF[out] * float(want.norm())


def check(dev, x, out, precise, **kw):
    from faster_yoco_amd import muon
    got = muon.orthogonalize(x.to(dev), dtype=out, precise=precise, **kw)
    assert got.dtype == out and got.shape == x.shape and got.is_contiguous()
    want, most = limit(x, out, precise, **kw)
    assert far(got, want) <= most, (far(got, want) / float(want.norm()), most / float(want.norm()))
    return got


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('m,n', SHAPES)
def test_five_steps(pkg, dev, m, n, kind):
    x = matrix(m, n, kind)
    check(dev, x, torch.bfloat16, False)
    check(dev, x, torch.float32, True)


@pytest.mark.parametrize('kind', ['noise', 'strong'])
@pytest.mark.parametrize('m,n', [(7, 1), (3, 5), (40, 60), (130, 70), (200, 333), (600, 300)])
def test_one_step_element_by_element(pkg, dev, m, n, kind):
    from faster_yoco_amd import muon
    x = matrix(m, n, kind)
    got = muon.orthogonalize(x.to(dev), steps=1, precise=False)
    want, bound = ref.exact(x, 1), ref.one_step_bound(x)
    assert ((got.cpu().double() - want).abs() <= bound * 1.01 + HALF[torch.float32] * want.abs()).all()


@pytest.mark.parametrize('out', DTYPES, ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_types(pkg, dev, dtype, out):
    for m, n in ((70, 150), (150, 70)):
        check(dev, matrix(m, n, 'falling', dtype, 1.0), out, out != torch.bfloat16)


def test_the_type_decides_the_exactness(pkg, dev):
    from faster_yoco_amd import muon
    for dtype in DTYPES:
        x = matrix(90, 130, 'falling', dtype, 1.0).to(dev)
        assert torch.equal(muon.orthogonalize(x), muon.orthogonalize(x, dtype=dtype, precise=dtype != torch.bfloat16))
    x = matrix(90, 130).to(dev)
    assert not torch.equal(muon.orthogonalize(x), muon.orthogonalize(x, precise=False))


@pytest.mark.parametrize('m,n', [(1024, 1300), (2300, 700), (1537, 1537)])
@pytest.mark.parametrize('precise', [False, True])
def test_larger_ones(pkg, dev, m, n, precise):
    x = matrix(m, n, 'strong')
    check(dev, x, torch.float32 if precise else torch.bfloat16, precise)


def test_every_tile(pkg, dev):
    """Counts at which the products run in tiles of 64, 128 and 256: equal matrices give equal results, and those of one."""
    from faster_yoco_amd import muon
    x = matrix(300, 520, 'falling')
    one = check(dev, x, torch.bfloat16, False)
    for count in (2, 20, 64, 160):
        many = muon.orthogonalize(x.to(dev).expand(count, 300, 520), dtype=torch.bfloat16)
        assert all(torch.equal(many[i], many[0]) for i in range(count))
        want, most = limit(x, torch.bfloat16, False)
        assert far(many[0], want) <= most
    assert torch.equal(muon.orthogonalize(x.to(dev), dtype=torch.bfloat16), one)


@pytest.mark.parametrize('precise,size', [(0, t) for t in ways_muon.FAST] + [(1, t) for t in ways_muon.PRECISE], ids=str)
def test_every_form(pkg, dev, precise, size):
    """Sizes that take every form of the kernels: two matrices by turns, every copy within its bound of the 64-bit form (computed on
    the GPU, where the largest take seconds less), and the same bits for each -- but for pairs, whose products hi lo and lo hi are
    added in the other order above the diagonal of a tile of 256 than where its quarters are tiles, which have no such half."""
    from faster_yoco_amd import muon
    count, m, n = size
    g = torch.Generator(device=dev).manual_seed(m * 31 + n)
    x = torch.randn(2, m, n, generator=g, device=dev) * 1e-3
    k = min(3, m, n)
    x[1] = x[1] * 0.05 + torch.randn(m, k, generator=g, device=dev) @ torch.randn(k, n, generator=g, device=dev) * 1e-3
    out = torch.float32 if precise else torch.bfloat16
    got = muon.orthogonalize(x[torch.arange(count, device=dev) % 2], dtype=out, precise=bool(precise))
    for i in range(min(count, 2)):
        assert precise or all(torch.equal(got[j], got[i]) for j in range(i, count, 2))
        want = ref.exact(x[i])
        # fp16 operands: as the stored roundings leave it.  Pairs: what N = 3 K / 16 additions in fp32 leave, N^(1/2) U32 of a
        # sum where their roundings add up at random: of X_0 (norm 1) into the small directions, 3.4^5 = 484 times by the end,
        # twice that with the later steps', and of each step's large ones, through slopes up to 1.6, 17 times; four times both
        if precise:
            many = math.sqrt(3 * max(m, n) / 16 + 8) * ref.U32
            most = 4 * (2 * 484 * many + 17 * many * float(want.norm()))
        else:
            most = 4 * float((ref.stored(x[i]) - want).norm()) + 2.0 ** -13 * float(want.norm())
        for j in range(i, count, 2):
            assert float((got[j].double() - want).norm()) <= most + HALF[out] * float(want.norm())


def test_scales_of_the_input(pkg, dev):
    """From the smallest norms to ones whose squares leave fp32: only the direction counts, above eps."""
    from faster_yoco_amd import muon
    x = matrix(40, 60)
    want = ref.exact(x)
    for scale in (2.0 ** -10, 1.0, 2.0 ** 60, 2.0 ** 130):
        got = muon.orthogonalize((x.double() * scale).float().to(dev), precise=True)      # 2^130 itself is no fp32
        assert far(got, want) <= 2.0 ** -18 * float(want.norm())
    tiny = x.double() / x.double().norm() * 1e-9                  # a hundredth of eps
    assert far(muon.orthogonalize(tiny.float().to(dev), precise=True), ref.exact(tiny.float())) <= 2.0 ** -15 * float(
        ref.exact(tiny.float()).norm())


def test_zeros_infinities_and_nan(pkg, dev):
    from faster_yoco_amd import muon
    x = torch.stack([matrix(70, 90) for _ in range(4)])
    x[0] = 0
    x[1, 3, 5], x[2, 60, 80] = float('nan'), float('inf')
    got = muon.orthogonalize(x.to(dev))
    assert not got[0].any() and got[1].isnan().all() and got[2].isnan().all()
    assert torch.equal(got[3], muon.orthogonalize(x[3].to(dev)))
    y = matrix(70, 90)
    y[5] = 0
    y[:, 7] = 0                                                   # an empty row and column stay so
    q = muon.orthogonalize(y.to(dev))
    assert not q[5].any() and not q[:, 7].any() and q.isfinite().all()


def test_strides_and_leading_dimensions(pkg, dev):
    from faster_yoco_amd import muon
    x = torch.stack([matrix(50, 33, k) for k in KINDS] * 2).view(2, 4, 50, 33).to(dev)
    want = muon.orthogonalize(x)
    assert want.shape == x.shape
    big = torch.full((2, 4, 53, 40), float('nan'), device=dev)
    big[:, :, 1:51, 3:36] = x
    assert torch.equal(muon.orthogonalize(big[:, :, 1:51, 3:36]), want)
    assert torch.equal(muon.orthogonalize(x.mT.contiguous().mT), want)            # columns apart: copied
    assert torch.equal(muon.orthogonalize(x[0, 1]), want[0, 1])
    assert torch.equal(muon.orthogonalize(x[:1].expand(3, 4, 50, 33))[2], want[0])
    odd = torch.empty(50 * 33 + 1, device=dev, dtype=torch.bfloat16)[1:].view(50, 33)             # an address of 2 mod 4
    odd.copy_(x[0, 0])
    assert torch.equal(muon.orthogonalize(odd), muon.orthogonalize(x[0, 0].bfloat16()))
    # transposed: the same matrix on its other side (its norm is summed in another order)
    assert far(muon.orthogonalize(x[0, 0].t().contiguous()).t(), want[0, 0].cpu().double()) <= 2.0 ** -15 * float(want[0, 0].norm())


def test_no_matrices(pkg, dev):
    from faster_yoco_amd import muon
    for shape in ((0, 4, 5), (3, 0, 5), (3, 4, 0)):
        assert muon.orthogonalize(torch.empty(shape, device=dev)).shape == shape
    muon.step_([], [], [], lr=1.0)
    e = torch.empty(0, 5, device=dev)
    muon.step_([e], [e], [e.clone()], lr=1.0)


def test_coefficients_of_each_step(pkg, dev):
    cs = [(3.4445, -4.7750, 2.0315), (3.0, -3.2, 1.2), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)]
    for m, n in ((60, 90), (300, 200)):
        check(dev, matrix(m, n), torch.float32, True, steps=4, coefficients=cs)
        check(dev, matrix(m, n), torch.bfloat16, False, steps=4, coefficients=cs)
        check(dev, matrix(m, n, 'flat'), torch.float32, True, steps=12, coefficients=(1.5, -0.5, 0.0))


def test_the_result_is_near_orthogonal(pkg, dev):
    from faster_yoco_amd import muon
    q = muon.orthogonalize(matrix(200, 800).to(dev), precise=False).double().cpu()
    s = torch.linalg.svdvals(q)
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


def state(shapes, g_dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = [[], [], [], []]
    for m, n in shapes:
        r = lambda: torch.randn(m, n, generator=g)  # noqa: E731
        p = 0.02 * r()
        for o, t in zip(out, (p, (1e-3 * r()).to(g_dtype), 1e-3 * r(), p.bfloat16())):
            o.append(t)
    return [[t.to(dev) for t in o] for o in out]


@pytest.mark.parametrize('precise', [False, True])
@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_step(pkg, dev, dtype, nesterov, precise):
    """momentum: three fp32 roundings.  p: two roundings, and the update's distance times its rate.  The copy: bf16 of p."""
    from faster_yoco_amd import muon
    shapes = [(70, 130), (130, 70), (70, 130), (5, 3), (64, 64)]
    p, g, m, p16 = state(shapes, dtype, dev)
    p0, m0 = [t.cpu().clone() for t in p], [t.cpu().clone() for t in m]
    factor = torch.tensor([0.37], device=dev)
    kw = dict(lr=0.01, momentum=0.9, nesterov=nesterov, weight_decay=0.3)
    muon.step_(p, g, m, p16, factor=factor, adjust='shape', precise=precise, **kw)
    f = float(factor)
    for i, s in enumerate(shapes):
        rate = 0.01 * math.sqrt(max(1.0, s[0] / s[1]))
        assert muon.rate(0.01, s, 'shape') == rate
        want, mom, q, u = ref.step(p0[i], g[i].cpu(), m0[i], lr=0.01, mu=float(torch.tensor(0.9)), nesterov=nesterov,
                                   weight_decay=0.3, rate=rate, factor=f)
        size = 0.9 * m0[i].double().abs() + 0.1 * f * g[i].cpu().double().abs()
        assert ((m[i].cpu().double() - mom).abs() <= 4 * 2.0 ** -24 * size).all()
        near = float((ref.stored(u, precise=precise) - q).norm())
        off = rate * (4 * near + (2.0 ** -18 if precise else 2.0 ** -13) * float(q.norm()))
        off += 2.0 ** -24 * float((3 * p0[i].double().abs() + 2 * rate * q.abs()).norm())
        assert far(p[i], want) <= off
        assert torch.equal(p16[i], p[i].bfloat16())


def test_step_without_copies_or_factor_and_with_strided_gradients(pkg, dev):
    from faster_yoco_amd import muon
    shapes = [(33, 50)] * 3
    a, b = state(shapes, torch.bfloat16, dev), state(shapes, torch.bfloat16, dev)
    muon.step_(a[0], a[1], a[2], a[3], lr=1e-3)
    wide = torch.zeros(33, 3 * 57, device=dev, dtype=torch.bfloat16)
    views = [wide[:, 57 * i + 1:57 * i + 51] for i in range(3)]
    for v, g in zip(views, b[1]):
        v.copy_(g)
    muon.step_(b[0], views, b[2], lr=1e-3, factor=torch.ones(1, device=dev))
    assert all(torch.equal(x, y) for x, y in zip(a[0] + a[2], b[0] + b[2]))


def test_many_matrices_of_a_shape(pkg, dev):
    """More than a launch names: the same as one by one."""
    from faster_yoco_amd import muon
    shapes = [(20, 24)] * 71
    a, b = state(shapes, torch.float32, dev, 3), state(shapes, torch.float32, dev, 3)
    muon.step_(*a, lr=1e-2)
    for t in zip(*b):
        muon.step_(*([v] for v in t), lr=1e-2)
    assert all(torch.equal(x, y) for u, v in zip(a, b) for x, y in zip(u, v))


def test_a_matrix_with_a_nan_leaves_the_others(pkg, dev):
    from faster_yoco_amd import muon
    a, b = state([(40, 30)] * 3, torch.float32, dev, 4), state([(40, 30)] * 3, torch.float32, dev, 4)
    a[1][1][3, 3] = float('nan')
    muon.step_(*a, lr=1e-2)
    muon.step_(*b, lr=1e-2)
    assert a[0][1].isnan().all()
    assert all(torch.equal(a[k][i], b[k][i]) for k in range(4) for i in (0, 2))


def test_neighbours_in_memory_are_left_alone(pkg, dev):
    """Odd matrices inside a flat buffer: what lies between them keeps its bits."""
    from faster_yoco_amd import muon
    shapes, at = [(33, 17), (17, 33), (1, 5), (65, 66)], 3
    flat = [torch.full((6000,), 7.0, device=dev, dtype=t) for t in (torch.float32, torch.float32, torch.bfloat16)]
    views, spots = [[], [], []], torch.ones(6000, dtype=torch.bool, device=dev)
    for m, n in shapes:
        for v, f in zip(views, flat):
            v.append(f[at:at + m * n].view(m, n))
        spots[at:at + m * n] = False
        at += m * n + 5
    g = [torch.randn(s, device=dev) for s in shapes]
    muon.step_(views[0], g, views[1], views[2], lr=0.1)
    assert all((f[spots] == 7).all() for f in flat) and all((v != 7).any() for v in views[0])


def test_on_another_stream_and_captured(pkg, dev):
    """A graph of a step and of orthogonalize, on a stream of its own; replays, with other gradients in between, give the eager
    results; two graphs captured one after the other do not share scratch that either still needs."""
    from faster_yoco_amd import muon
    shapes = [(130, 70), (70, 130), (130, 70)]
    a, b = state(shapes, torch.bfloat16, dev, 5), state(shapes, torch.bfloat16, dev, 5)
    x = matrix(90, 140).to(dev)
    factor = torch.tensor([0.5], device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        muon.step_([t.clone() for t in a[0]], a[1], [t.clone() for t in a[2]], lr=1e-2)
        muon.orthogonalize(x)
        s.synchronize()
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        with torch.cuda.graph(graphs[0], stream=s):
            muon.step_(*a, lr=1e-2, factor=factor)
            q = muon.orthogonalize(x)
        with torch.cuda.graph(graphs[1], stream=s):
            q2 = muon.orthogonalize(x * 2, precise=False)
    torch.cuda.synchronize()
    for k in range(3):
        for t, u in zip(a[1], b[1]):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(k)))
            u.copy_(t)
        x.mul_(-1.5)
        factor.mul_(0.7)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        muon.step_(*b, lr=1e-2, factor=factor)
        assert all(torch.equal(u, v) for c, d in zip(a, b) for u, v in zip(c, d))
        assert torch.equal(q, muon.orthogonalize(x)) and torch.equal(q2, muon.orthogonalize(x * 2, precise=False))


def test_two_streams_at_once(pkg, dev):
    from faster_yoco_amd import muon
    xs = [matrix(200, 150, k).to(dev) for k in ('noise', 'strong')]
    want = [muon.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                got[i].append(muon.orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for v, w in zip(got, want) for g in v)


def test_results_do_not_depend_on_the_run(pkg, dev):
    from faster_yoco_amd import muon
    x = torch.stack([matrix(260, 300, k) for k in KINDS]).to(dev)
    first = muon.orthogonalize(x)
    assert all(torch.equal(muon.orthogonalize(x), first) for _ in range(3))


def test_refusals(pkg, dev):
    from faster_yoco_amd import muon
    x = matrix(8, 6).to(dev)
    p, m, p16 = x.clone(), x.clone(), x.bfloat16()
    step = lambda **k: muon.step_(**({'params': [p], 'grads': [x], 'momenta': [m], 'copies': [p16], 'lr': 1e-3} | k))  # noqa: E731
    for call, text in ((lambda: muon.orthogonalize(x[0]), 'matrices'), (lambda: muon.orthogonalize(x.double()), 'fp32, bf16 or fp16'),
                       (lambda: muon.orthogonalize(x, dtype=torch.float64), 'fp32, bf16 or fp16'),
                       (lambda: muon.orthogonalize(x, steps=0), 'steps'), (lambda: muon.orthogonalize(x, steps=65), 'steps'),
                       (lambda: muon.orthogonalize(x, coefficients=(1.0, 2.0)), 'coefficients'),
                       (lambda: muon.orthogonalize(x, coefficients=[(1.0, 0.0, 0.0)] * 4), 'coefficients'),
                       (lambda: muon.orthogonalize(x, coefficients=(5.0, 0.0, 0.0)), 'range'),
                       (lambda: muon.orthogonalize(x, coefficients=(2.0, 0.0, 0.0)), 'range'),       # 2^5 after five
                       (lambda: muon.orthogonalize(x, coefficients=(float('nan'), 0.0, 0.0)), 'range'),
                       (lambda: muon.orthogonalize(x, eps=0.0), 'eps'),
                       (lambda: step(params=[p[:, :4]]), 'contiguous'), (lambda: step(params=[p.bfloat16()]), 'contiguous'),
                       (lambda: step(params=[p[0]]), 'a matrix'), (lambda: step(momenta=[m.half()]), 'contiguous'),
                       (lambda: step(momenta=[m[:5]]), "p's shape"), (lambda: step(copies=[p]), 'contiguous'),
                       (lambda: step(grads=[x[:5]]), "p's shape"), (lambda: step(grads=[x.t().contiguous().t()]), 'neighbouring'),
                       (lambda: step(grads=[x.double()]), 'fp32, bf16 or fp16'), (lambda: step(grads=[]), 'as many'),
                       (lambda: step(grads=[x.cpu()]), 'GPU tensor'), (lambda: step(momentum=1.0), 'momentum'),
                       (lambda: step(factor=torch.ones(2, device=dev)), 'factor'), (lambda: step(adjust='other'), 'adjust'),
                       (lambda: step(momenta=[p]), 'named twice'),
                       (lambda: step(params=[p, p], grads=[x, x], momenta=[m, m.clone()], copies=None), 'named twice')):
        with pytest.raises(RuntimeError, match=text):
            call()
    assert torch.equal(p, x) and torch.equal(m, x)                # nothing was written


def test_small_matrices_of_a_call_side_by_side(pkg, dev):
    """Small matrices run by themselves whatever else a call holds: in any mixture each comes out as alone, bit for bit.  Those
    of up to four parts of 32 x 32 come out as exactly as pairs do."""
    from faster_yoco_amd import muon
    sizes = [(20, 31), (20, 200), (60, 61), (200, 20), (40, 100), (1, 1), (33, 90), (64, 64), (128, 32), (100, 90), (16, 16), (1, 400)]
    u = [matrix(m, n, KINDS[i % len(KINDS)]).to(dev) for i, (m, n) in enumerate(sizes)]
    for precise in (False, True):
        p = [torch.zeros_like(t) for t in u]
        muon.step_(p, u, [torch.zeros_like(t) for t in u], lr=1.0, adjust=1.0, weight_decay=0.0, momentum=0.0, precise=precise)
        for t, q in zip(u, p):
            assert torch.equal(-q, muon.orthogonalize(t, precise=precise)), t.shape
            if -(-t.shape[0] // 32) * -(-t.shape[1] // 32) <= 4:
                want, most = limit(t.cpu(), torch.float32, True)
                assert far(-q, want) <= most, t.shape


def test_offsets_past_32_bits(pkg, dev):
    """Matrices and rows that lie 2^31 elements and more apart, read by the small matrices' kernel and by the others."""
    from faster_yoco_amd import muon
    flat = torch.empty((1 << 31) + 300000, dtype=torch.bfloat16, device=dev)
    for m, n in ((40, 50), (150, 140)):
        x = flat.as_strided((2, m, n), ((1 << 31) + 77, n + 3, 1))
        x.copy_(torch.stack([matrix(m, n), matrix(m, n, 'strong')]))
        assert torch.equal(muon.orthogonalize(x), muon.orthogonalize(x.clone(memory_format=torch.contiguous_format)))
    for n in (60, 2000):
        x = flat.as_strided((3, n), ((1 << 30) + 5, 1))
        x.copy_(matrix(3, n))
        assert torch.equal(muon.orthogonalize(x), muon.orthogonalize(x.clone(memory_format=torch.contiguous_format)))
        p, q = (torch.zeros(3, n, device=dev) for _ in range(2))
        muon.step_([p], [x], [torch.zeros_like(p)], lr=0.1)
        muon.step_([q], [x.clone(memory_format=torch.contiguous_format)], [torch.zeros_like(q)], lr=0.1)
        assert torch.equal(p, q) and (p != 0).any()


def test_overlapping_tensors_are_refused(pkg, dev):
    """Views that share some bytes with what is written; gradients may share theirs with each other, and lie next to it."""
    from faster_yoco_amd import muon
    flat, g = torch.ones(200, device=dev), torch.ones(10, 20, device=dev)
    at = lambda i, m=4, n=6: flat[i:i + m * n].view(m, n)  # noqa: E731
    z = lambda m=4, n=6: torch.zeros(m, n, device=dev)  # noqa: E731
    for args, text in ((([at(0), at(23)], [g[:4, :6]] * 2, [z(), z()]), 'overlap'), (([at(0)], [g[:4, :6]], [at(20)]), 'overlap'),
                       (([at(0), at(100)], [g[:4, :6]] * 2, [z(), at(90)]), 'overlap'),
                       (([at(24)], [at(0, 5)[1:]], [z()]), 'overlaps what is written'),
                       (([at(24)], [at(47)], [z()]), 'overlaps what is written'),
                       (([at(24)], [at(10, 2, 48)[:, :24].reshape(2, 24)[:, :6].expand(2, 6)], [z()]), "p's shape"),
                       (([at(30, 2, 5)], [flat.as_strided((2, 5), (100, 1), 20)], [z(2, 5)]), 'overlaps what is written')):
        with pytest.raises(RuntimeError, match=text):
            muon.step_(*args, lr=0.1)
    assert (flat == 1).all()
    muon.step_([at(24), at(48)], [at(0), at(0)], [at(72), at(96)], lr=0.1)
    assert (flat[:24] == 1).all() and (flat[120:] == 1).all() and (flat[24:72] < 1).all()
    assert ((flat[72:120] - 1).abs() < 1e-6).all()                # 0.95 + 0.05 of ones


def test_parameters_and_their_gradients(pkg, dev):
    """A model's parameters as they are, outside no_grad too: the update records nothing."""
    from faster_yoco_amd import muon
    w = [torch.nn.Parameter(matrix(30, 20).to(dev)), torch.nn.Parameter(matrix(150, 140).to(dev))]
    sum((p * p).sum() for p in w).backward()
    old = [p.detach().clone() for p in w]
    momenta = [torch.zeros_like(p, requires_grad=False) for p in w]
    muon.step_(w, [p.grad for p in w], momenta, lr=0.01, weight_decay=0.0, nesterov=False, momentum=0.0)
    for p, o, m in zip(w, old, momenta):
        assert p.is_leaf and p.grad_fn is None and torch.equal(m, p.grad)
        # the same call's launches hold other matrices: last bits, 1e-3 of the result
        want = o - muon.rate(0.01, o.shape, 'rms') * muon.orthogonalize(2 * o, precise=False)
        assert float((p.detach() - want).norm()) < 4e-3 * float((want - o).norm())


def test_as_operators(pkg, dev):
    ops = torch.ops.yoco_z1
    c = [3.4445, -4.775, 2.0315] * 2
    x = matrix(3 * 20, 30).view(3, 20, 30).to(dev)
    p, m, p16 = x[0].clone(), x[1].clone(), x[0].bfloat16()
    checks = [(ops.orthogonalize, (x, 2, c, 1e-7, torch.bfloat16, False)),
              (ops.muon_step_, ([p], [x[2]], [m], [p16], None, [1e-3], [0.99], 0.9, True, 2, c, 1e-7, False))]
    for op, args in checks:
        res = torch.library.opcheck(op, args, test_utils=('test_schema', 'test_faketensor', 'test_aot_dispatch_dynamic'))
        assert all(v == 'SUCCESS' for v in res.values()), (op, res)
