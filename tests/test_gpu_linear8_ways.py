"""Every form of the product and weight gradient kernels, in every result type, against the sums in 64 bits over what the
operands stand for (bounds: test_gpu_linear8).  Rows differ in size, and a few channels are a hundred times the rest."""
import pytest
import torch

import blocks as ref
import ways
from blocks import DTYPES
from test_gpu_linear8 import near

pytestmark = pytest.mark.gpu


def rows(n, dim, seed, large=1.0):
    g = torch.Generator().manual_seed(seed + 7 * n + dim)
    x = torch.randn(n, dim, generator=g) * torch.exp(0.5 * torch.randn(n, 1, generator=g))
    x[:, 3::200] *= large
    return x.bfloat16()


@pytest.mark.parametrize('form', ways.PRODUCTS, ids=str)
def test_product(pkg, dev, form):
    from faster_yoco_amd import _lib, act8, linear8
    M, N, K = ways.PRODUCTS[form]
    assert ways.product(_lib.lib(), M, N, K) == form
    x, w = rows(M, K, 1, 100.0) * 0.01, rows(N, K, 2) * 0.05
    xv, wv = ref.values(*ref.pack(x), K).to(dev), ref.weight_values(*ref.pack_weight(w)[:2], (N, K)).t().contiguous().to(dev)
    want, sizes = (xv @ wv).cpu(), (xv.abs() @ wv.abs()).cpu()
    a, p = act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev), transposed=False)
    for dtype in DTYPES:
        y = linear8.matmul(a, p, dtype)
        near(y, want, sizes, K, dtype)
        assert torch.equal(y, linear8.matmul(a, p, dtype))


@pytest.mark.parametrize('form', ways.GRADIENTS, ids=str)
def test_weight_gradient(pkg, dev, form):
    from faster_yoco_amd import _lib, act8, linear8
    T, N, K = ways.GRADIENTS[form]
    assert ways.gradient(_lib.lib(), T, N, K, N % 2 == 0) == form
    x, dy = rows(T, K, 3, 100.0) * 0.01, rows(T, N, 4) * 0.01
    xv, d = ref.values(*ref.pack(x), K).to(dev), dy.double().t().contiguous().to(dev)
    want, sizes = (d @ xv).cpu(), (d.abs() @ xv.abs()).cpu()
    a = act8.pack(x.to(dev))
    for dtype in DTYPES:
        dw = linear8.weight_grad(dy.to(dev), a, dtype)
        near(dw, want, sizes, T, dtype)
        assert torch.equal(dw, linear8.weight_grad(dy.to(dev), a, dtype))


def test_whole_numbers_past_32_bits_of_offsets(pkg, dev):
    """2.2e9 operand bytes in 70000 rows, whole numbers of at most 8: every sum is exact in fp32, so the last rows' products
    and their part of the weight's gradient are too, and a block of K left out or taken twice shows."""
    from faster_yoco_amd import act8, linear8
    n, last, N, K = 70000, 300, 40, 31000
    assert n * K > 2 ** 31 and 8 * 8 * K < 2 ** 24
    g = torch.Generator().manual_seed(18)
    whole = lambda *s: torch.randint(-8, 9, s, generator=g).bfloat16()  # noqa: E731
    rest, w, dy_rest = whole(last, K), whole(N, K), whole(last, N)
    x = torch.zeros(n, K, dtype=torch.bfloat16, device=dev)
    x[-last:] = rest.to(dev)
    a = act8.pack(x)
    del x
    y = linear8.matmul(a, linear8.pack_weight(w.to(dev), transposed=False), torch.float32)
    assert torch.equal(y[-last:].cpu().double(), rest.double() @ w.double().t()) and not y[:-last].any()
    dy = torch.zeros(n, N, dtype=torch.bfloat16, device=dev)
    dy[-last:] = dy_rest.to(dev)
    dw = linear8.weight_grad(dy, a, torch.float32)
    assert torch.equal(dw.cpu().double(), dy_rest.double().t() @ rest.double())
