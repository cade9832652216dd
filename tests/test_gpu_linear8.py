"""8-bit products and the weight's gradient on the GPU against the same sums in 64 bits over what the 8-bit operands stand
for.

Bound.  Each product of two operands is exact in fp32 (e4m3: 4 significant bits; the gradient: 8 by 4), so a sum of n of
them in fp32, in whatever order, is within n u of the sum of their sizes, u = 2^-24; the matrix instructions may cut
rather than round, which doubles it.  Then one rounding to the result's type."""
import pytest
import torch

import blocks as ref
from blocks import DTYPES, U

pytestmark = pytest.mark.gpu


def rows(n, dim, seed, spread=0.5):
    g = torch.Generator().manual_seed(seed + 7 * n + dim)
    return (torch.randn(n, dim, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))).bfloat16()


def near(got, want, sizes, n, dtype):
    assert got.dtype == dtype and tuple(got.shape) == tuple(want.shape)
    assert ((got.cpu().double() - want).abs() <= 2 * (n + 8) * U * sizes + ref.rounded(want, dtype) * 1.001).all()


def operands(M, N, K, seed=0):
    x, w = rows(M, K, seed), rows(N, K, seed + 1, 0.1) * 0.05
    return x, w, ref.values(*ref.pack(x), K), ref.weight_values(*ref.pack_weight(w)[:2], (N, K))


SHAPES = [(1, 1, 1), (1, 300, 1000), (2, 64, 128), (7, 1501, 130), (31, 100, 700), (32, 129, 256), (33, 31, 640),
          (64, 256, 512), (65, 257, 100), (127, 128, 384), (129, 129, 1153), (200, 700, 2048), (333, 1501, 1000),
          (513, 300, 129), (1000, 1, 77)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_product(pkg, dev, M, N, K, dtype):
    from faster_yoco_amd import act8, linear8
    x, w, xv, wv = operands(M, N, K)
    y = linear8.matmul(act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev)), dtype)
    near(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), K, dtype)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('M,N,K', [(100, 256, 8192), (40, 70, 2300), (33, 1, 1030), (257, 300, 4100), (130, 129, 1025)])
def test_product_in_parts_of_k(pkg, dev, M, N, K, dtype):
    """Few tiles and a long K: partial results, joined."""
    from faster_yoco_amd import _lib, act8, linear8
    parts = _lib.lib().z1_product8_workspace(M, N, K, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]) > 0
    assert parts or K < 2000                           # nine blocks of K are done before a second launch would begin
    x, w, xv, wv = operands(M, N, K, 30)
    p = linear8.pack_weight(w.to(dev))
    y = linear8.matmul(act8.pack(x.to(dev)), p, dtype)
    near(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), K, dtype)
    assert torch.equal(y, linear8.matmul(act8.pack(x.to(dev)), p, dtype))


@pytest.mark.parametrize('M,N,K', [(300, 2500, 600), (2100, 4000, 520)])
def test_product_in_large_tiles(pkg, dev, M, N, K):
    from faster_yoco_amd import act8, linear8
    x, w, xv, wv = operands(M, N, K, 31)
    y = linear8.matmul(act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev)))
    near(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), K, torch.bfloat16)


@pytest.mark.parametrize('M,N,K', [(1900, 2900, 1300), (2048, 3072, 520), (4000, 1500, 600)])
def test_product_in_tiles_of_128_by_192(pkg, dev, M, N, K):
    from faster_yoco_amd import act8, linear8
    x, w, xv, wv = operands(M, N, K, 36)
    y = linear8.matmul(act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev)))
    near(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), K, torch.bfloat16)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('M,N,K', [(1, 12300, 300), (5, 6200, 1111), (16, 9000, 700), (33, 2100, 700), (64, 4096, 384),
                                   (50, 2049, 1500), (65, 8190, 2000), (100, 8185, 2304), (128, 8192, 1900)])
def test_few_rows_of_many_outputs(pkg, dev, M, N, K, dtype):
    from faster_yoco_amd import act8, linear8
    x, w, xv, wv = operands(M, N, K, 35)
    a, p = act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev), transposed=False)
    y = linear8.matmul(a, p, dtype)
    near(y, xv @ wv.t(), xv.abs() @ wv.abs().t(), K, dtype)
    assert torch.equal(y, linear8.matmul(a, p, dtype))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize('T,N,K', [(8192, 256, 256), (1100, 130, 70), (3001, 2, 3), (1024, 600, 300), (200, 4000, 2100)])
def test_weight_gradient_in_parts_and_large_tiles(pkg, dev, T, N, K, dtype):
    from faster_yoco_amd import _lib, act8, linear8
    parts = _lib.lib().z1_weight_grad8_workspace(T, N, K) > 0
    assert parts if T > 1024 else not parts or T > 1000           # 1024 tokens: as the costs have it
    x, dy = rows(T, K, 32), rows(T, N, 33) * 1e-3
    xv, d = ref.values(*ref.pack(x), K), dy.double()
    a = act8.pack(x.to(dev))
    dw = linear8.weight_grad(dy.to(dev), a, dtype)
    near(dw, d.t() @ xv, d.abs().t() @ xv.abs(), T, dtype)
    assert torch.equal(dw, linear8.weight_grad(dy.to(dev), a, dtype))


@pytest.mark.parametrize('M,N,K', SHAPES)
def test_product_with_the_other_order(pkg, dev, M, N, K):
    """dy @ w: the input's gradient."""
    from faster_yoco_amd import act8, linear8
    _, w, _, wv = operands(1, N, K, 2)
    dy = rows(M, N, 3) * 1e-3
    dv = ref.values(*ref.pack(dy), N)
    dx = linear8.matmul(act8.pack(dy.to(dev)), linear8.pack_weight(w.to(dev)), torch.bfloat16, transposed=True)
    near(dx, dv @ wv, dv.abs() @ wv.abs(), N, torch.bfloat16)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize('T,N,K', [(1, 1, 1), (1, 130, 200), (2, 64, 128), (15, 33, 700), (16, 128, 128), (31, 129, 127),
                                   (32, 300, 256), (33, 256, 300), (100, 1000, 513), (333, 1501, 1000), (2000, 70, 90),
                                   (5000, 128, 129), (4097, 7, 1)])
def test_weight_gradient(pkg, dev, T, N, K, dtype):
    from faster_yoco_amd import act8, linear8
    x, dy = rows(T, K, 4), rows(T, N, 5) * 1e-3
    xv = ref.values(*ref.pack(x), K)
    dw = linear8.weight_grad(dy.to(dev), act8.pack(x.to(dev)), dtype)
    d = dy.double()
    near(dw, d.t() @ xv, d.abs().t() @ xv.abs(), T, dtype)


@pytest.mark.parametrize('M,N,K', [(5, 70, 300), (150, 260, 640), (300, 513, 257)])
def test_whole_numbers_are_exact(pkg, dev, M, N, K):
    """Whole numbers of at most 8, scaled by powers of two of every block's own: every sum is exact in fp32, so each
    result is too, whichever lane holds which element."""
    from faster_yoco_amd import act8, linear8
    g = torch.Generator().manual_seed(6)
    x = torch.randint(-8, 9, (M, K), generator=g).double()
    w = torch.randint(-8, 9, (N, K), generator=g).double()
    col = torch.arange(K) // 128
    x = x * 2.0 ** (torch.arange(M) % 3)[:, None] * 2.0 ** (col % 2)
    w = w * 2.0 ** (torch.arange(N) // 128 % 2)[:, None] * 2.0 ** (col % 3)
    a, p = act8.pack(x.float().to(dev)), linear8.pack_weight(w.float().to(dev))
    assert torch.equal(linear8.matmul(a, p, torch.float32).cpu().double(), x @ w.t())
    dy = torch.randint(-8, 9, (M, N), generator=g).double()
    d8 = act8.pack(dy.float().to(dev))
    assert torch.equal(linear8.matmul(d8, p, torch.float32, transposed=True).cpu().double(), dy @ w)
    assert torch.equal(linear8.weight_grad(dy.bfloat16().to(dev), a, torch.float32).cpu().double(), dy.t() @ x)


def test_scales_of_every_size(pkg, dev):
    """Rows of 2^-110 and of 2^100, weights of 2^60 and 2^-50: the products' scales add up beyond a byte's own range."""
    from faster_yoco_amd import act8, linear8
    x, w = rows(40, 256, 7).double(), rows(300, 256, 8, 0.1).double()
    for ex, ew in ((-110, 60), (100, -50), (-60, -60), (40, 40)):
        xs, ws = (x * 2.0 ** ex).float(), (w * 2.0 ** ew).float()
        xv, wv = ref.values(*ref.pack(xs), 256), ref.weight_values(*ref.pack_weight(ws)[:2], (300, 256))
        y = linear8.matmul(act8.pack(xs.to(dev)), linear8.pack_weight(ws.to(dev)), torch.float32)
        want, sizes = xv @ wv.t(), xv.abs() @ wv.abs().t()
        assert ((y.cpu().double() - want).abs() <= 2 * 264 * U * sizes + 2.0 ** -126).all()


@pytest.mark.parametrize('M', [3, 200])
def test_values_that_are_not_finite_stay_in_their_rows(pkg, dev, M):
    from faster_yoco_amd import act8, linear8
    x, w, _, _ = operands(M, 300, 700, 9)
    dy = rows(M, 300, 10)
    clean = x.clone()
    x[1, 400], x[2, 3] = float('nan'), float('inf')
    p = linear8.pack_weight(w.to(dev))
    y = linear8.matmul(act8.pack(x.to(dev)), p)
    assert y[1].isnan().all() and y[2].isnan().all() and not torch.cat([y[:1], y[3:]]).isnan().any()
    dw = linear8.weight_grad(dy.to(dev), act8.pack(x.to(dev)), torch.float32)
    bad = torch.zeros(700, dtype=torch.bool)
    bad[[400, 3]] = True
    assert dw[:, bad].isnan().all() and not dw[:, ~bad].isnan().any()
    dy[1, 7] = float('nan')
    dw = linear8.weight_grad(dy.to(dev), act8.pack(clean.to(dev)), torch.float32)
    assert dw[7].isnan().all() and dw[torch.arange(300) != 7].isfinite().all()


def test_gradient_rows_of_any_stride(pkg, dev):
    from faster_yoco_amd import act8, linear8
    x, base = rows(90, 300, 11).to(dev), rows(90, 801, 12).to(dev)
    a = act8.pack(x)
    for dy in (base[:, 3:700], base[:, 1:130], base.t().contiguous().t()[:, :640], base[:1, :640].expand(90, 640)):
        assert torch.equal(linear8.weight_grad(dy, a), linear8.weight_grad(dy.contiguous(), a))
    assert torch.equal(linear8.weight_grad(base[:, :640].reshape(9, 10, 640), a), linear8.weight_grad(base[:, :640].contiguous(), a))


@pytest.mark.parametrize('T,N,K', [(3001, 65, 300), (2050, 7, 260), (5000, 1, 40), (1000, 1001, 130), (64, 9, 9)])
def test_gradient_of_odd_rows_in_parts(pkg, dev, T, N, K):
    from faster_yoco_amd import act8, linear8
    x, dy = rows(T, K, 37), rows(T, N, 38) * 1e-3
    xv, d = ref.values(*ref.pack(x), K), dy.double()
    for dtype in DTYPES:
        dw = linear8.weight_grad(dy.to(dev), act8.pack(x.to(dev)), dtype)
        near(dw, d.t() @ xv, d.abs().t() @ xv.abs(), T, dtype)


@pytest.mark.parametrize('T', [1, 63, 130])
def test_gradient_rows_of_whole_dwords_and_odd_width(pkg, dev, T):
    """The last row's last element shares its dword with what lies behind the tensor."""
    from faster_yoco_amd import act8, linear8
    a, base = act8.pack(rows(T, 200, 41).to(dev)), rows(T, 800, 42).to(dev)
    for n in (1, 7, 129, 333, 799):
        dy = base[:, :n]
        assert torch.equal(linear8.weight_grad(dy, a), linear8.weight_grad(dy.contiguous(), a))
        assert linear8.weight_grad(dy, a)[-1].any()


def test_gradient_of_one_row_for_all_tokens(pkg, dev):
    """Rows a stride of zero apart, not finite in places: only what they enter is."""
    from faster_yoco_amd import act8, linear8
    x = rows(70, 200, 43).abs().to(dev) + 1
    row = rows(1, 300, 44).to(dev)
    row[0, 5] = float('inf')
    dw = linear8.weight_grad(row.expand(70, 300), act8.pack(x), torch.float32)
    assert torch.equal(dw, linear8.weight_grad(row.repeat(70, 1), act8.pack(x), torch.float32))
    assert (dw[5] == float('inf')).all() and dw[:5].isfinite().all() and dw[6:].isfinite().all()


def test_gradient_of_no_tokens(pkg, dev):
    from faster_yoco_amd import act8, linear8
    a = act8.pack(rows(4, 200, 45).to(dev))
    none = act8.Act8(a.q[:0], a.s[:0], 200)
    for dy in (torch.empty(0, 300), torch.empty(0, 301), torch.empty(1, 300).expand(1, 300)[:0]):
        assert torch.equal(linear8.weight_grad(dy.bfloat16().to(dev), none), torch.zeros(dy.shape[1], 200, dtype=torch.bfloat16, device=dev))


def test_linear_is_its_three_products(pkg, dev):
    from faster_yoco_amd import act8, linear8
    x = rows(96, 384, 13).to(dev).view(4, 24, 384).requires_grad_()
    w = (rows(260, 384, 14, 0.1) * 0.05).to(dev).requires_grad_()
    dy = rows(96, 260, 15).to(dev).view(4, 24, 260)
    p = linear8.pack_weight(w.detach())
    y = linear8.linear(x, w, p)
    y.backward(dy)
    a = act8.pack(x.detach())
    assert y.shape == (4, 24, 260) and torch.equal(y.detach().view(96, 260), linear8.matmul(a, p))
    assert torch.equal(x.grad.view(96, 384), linear8.matmul(act8.pack(dy), p, transposed=True))
    assert torch.equal(w.grad, linear8.weight_grad(dy, a))


def test_gradients_match_differences(pkg, dev):
    """The function is linear in x and in w where its operands are what 8 bits hold: differences of whole steps are exact
    in 64 bits, and the kernels' fp32 sums are exact for these whole numbers."""
    from faster_yoco_amd import act8, linear8
    g = torch.Generator().manual_seed(16)
    x = torch.randint(-4, 5, (5, 130), generator=g).double()
    w = torch.randint(-4, 5, (140, 130), generator=g).double()
    dy = torch.randint(-4, 5, (5, 140), generator=g).double()
    f = lambda x, w: (dy * (x @ w.t())).sum()  # noqa: E731
    p = linear8.pack_weight(w.float().to(dev))
    dx = linear8.matmul(act8.pack(dy.float().to(dev)), p, torch.float32, transposed=True).cpu().double()
    dw = linear8.weight_grad(dy.bfloat16().to(dev), act8.pack(x.float().to(dev)), torch.float32).cpu().double()
    for i, j in ((0, 0), (4, 129), (2, 64)):
        e = torch.zeros_like(x)
        e[i, j] = 1
        assert (f(x + e, w) - f(x - e, w)) / 2 == dx[i, j]
    for i, j in ((0, 0), (139, 129), (128, 127)):
        e = torch.zeros_like(w)
        e[i, j] = 1
        assert (f(x, w + e) - f(x, w - e)) / 2 == dw[i, j]


def test_nothing_to_multiply(pkg, dev):
    from faster_yoco_amd import act8, linear8
    p = linear8.pack_weight(torch.ones(200, 300, dtype=torch.bfloat16, device=dev))
    none = act8.pack(torch.empty(0, 300, dtype=torch.bfloat16, device=dev))
    assert linear8.matmul(none, p).shape == (0, 200)
    dw = linear8.weight_grad(torch.empty(0, 200, dtype=torch.bfloat16, device=dev), none)
    assert dw.shape == (200, 300) and not dw.any()


def test_offsets_past_32_bits(pkg, dev):
    """2.2e9 operand bytes in 70000 rows: the last rows' products are those of the same rows alone, and their part of the
    weight's gradient is there."""
    from faster_yoco_amd import act8, linear8
    n, K = 70000, 31000
    assert n * K > 2 ** 31
    x = torch.zeros(n, K, dtype=torch.bfloat16, device=dev)
    last = rows(300, K, 17).to(dev)
    x[-300:] = last
    a, b = act8.pack(x), act8.pack(last)
    del x
    p = linear8.pack_weight((rows(40, K, 18, 0.1) * 0.05).to(dev), transposed=False)
    y = linear8.matmul(a, p, torch.float32)
    want = linear8.matmul(b, p, torch.float32)
    assert (y[-300:] - want).abs().max() <= 2 * (K + 8) * U * want.abs().max() * 40 and not y[:-300].any()
    dy = torch.zeros(n, 40, dtype=torch.bfloat16, device=dev)
    dy[-300:] = rows(300, 40, 19).to(dev)
    dw = linear8.weight_grad(dy, a, torch.float32)
    alone = linear8.weight_grad(dy[-300:], b, torch.float32)
    assert (dw - alone).abs().max() <= 2 * 308 * U * 300 * alone.abs().max() and alone.any()


def test_other_stream_and_graph(pkg, dev):
    from faster_yoco_amd import act8, linear8
    x, dy = rows(200, 700, 20).to(dev), rows(200, 300, 21).to(dev)
    p = linear8.pack_weight((rows(300, 700, 22, 0.1)).to(dev))

    def step():
        a, d = act8.pack(x), act8.pack(dy)
        return (linear8.matmul(a, p), linear8.matmul(d, p, transposed=True), linear8.weight_grad(dy, a),
                linear8.matmul(act8.Act8(a.q[:1], a.s[:1], 700), p))
    want = step()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = step()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (23, 24, 25):
        x.copy_(rows(200, 700, seed).to(dev))
        dy.copy_(rows(200, 300, seed + 1).to(dev))
        want = step()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals(pkg, dev):
    from faster_yoco_amd import act8, linear8
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    a, p = act8.pack(x), linear8.pack_weight(torch.zeros(300, 256, dtype=torch.bfloat16, device=dev))
    with pytest.raises(RuntimeError, match='do not fit a weight 300 x 256'):
        linear8.matmul(act8.pack(x[:, :200]), p)
    with pytest.raises(RuntimeError, match='from the left'):
        linear8.matmul(a, p, transposed=True)
    with pytest.raises(RuntimeError, match='without its other order'):
        linear8.matmul(act8.pack(torch.zeros(4, 300, device=dev)),
                       linear8.pack_weight(torch.zeros(300, 256, device=dev), transposed=False), transposed=True)
    with pytest.raises(RuntimeError, match='expected fp32, bf16 or fp16'):
        linear8.matmul(a, p, torch.float64)
    with pytest.raises(RuntimeError, match='bf16 gradient rows'):
        linear8.weight_grad(x.float(), a)
    with pytest.raises(RuntimeError, match='linear8.weight_grad'):
        linear8.weight_grad(x[:3], a)
    with pytest.raises(RuntimeError, match='GPU tensor|no CPU path'):
        linear8.weight_grad(x, act8.Act8(a.q.cpu(), a.s.cpu(), 256))
    with pytest.raises(RuntimeError, match='expected bf16 rows'):
        linear8.linear(x.float(), x, p)
    with pytest.raises(RuntimeError, match='8-bit blocks of'):
        linear8.linear(x, x, p)


def test_what_linear_keeps_is_saved_for_autograd(pkg, dev):
    """Saved-tensor hooks see all that is kept, only what a gradient needs is, and a weight written before the backward pass
    is an error, not another weight's gradient; one replaced is not used."""
    from faster_yoco_amd import linear8
    x, w = rows(96, 384, 13).to(dev), (rows(260, 384, 14, 0.1) * 0.05).to(dev)
    dy = rows(96, 260, 15).to(dev)
    p, other = linear8.pack_weight(w), linear8.pack_weight(w * 2)

    def run(need_x, need_w, p):
        kept, xs, ws = [], x.clone().requires_grad_(need_x), w.clone().requires_grad_(need_w)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
            y = linear8.linear(xs, ws, p)
        return y, xs, ws, sorted(tuple(t.shape) for t in kept)
    order, packed = [(3, 4), (384, 384)], [(96, 4), (96, 384)]
    assert run(True, False, p)[3] == order and run(False, True, p)[3] == packed
    y, xs, ws, kept = run(True, True, p)
    assert kept == sorted(order + packed)
    qt, p.qt = p.qt, other.qt                          # replaced: the kept one counts
    y.backward(dy)
    p.qt = qt
    y2, xs2, ws2, _ = run(True, True, p)
    y2.backward(dy)
    assert torch.equal(xs.grad, xs2.grad) and torch.equal(ws.grad, ws2.grad)
    y = linear8.linear(x.clone().requires_grad_(), w, p)           # without hooks, which pass the version check by
    p.qt.view(torch.uint8).copy_(other.qt.view(torch.uint8))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward(dy)


def test_linear_without_the_other_order(pkg, dev):
    from faster_yoco_amd import linear8
    x, w = rows(8, 256, 46).to(dev), rows(128, 256, 47).to(dev)
    p = linear8.pack_weight(w, transposed=False)
    with pytest.raises(RuntimeError, match='without its other order'):
        linear8.linear(x.clone().requires_grad_(), w, p)
    ws = w.clone().requires_grad_()                    # the weight's gradient does not need it
    linear8.linear(x, ws, p).sum().backward()
    assert ws.grad.shape == w.shape
