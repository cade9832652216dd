"""Products of operands whose terms differ much in size: sums are fp32 whatever the result's type, so the bound of an fp32 sum
holds (n u of the terms' sizes, doubled for cutting, then the rounding to the result's type) where large terms cancel and
where a few channels are a thousand times the rest."""
import pytest
import torch

import blocks as ref
from blocks import DTYPES
from test_gpu_linear8 import near

pytestmark = pytest.mark.gpu

# one row, few rows, more rows than those, tiles of each size, and K in parts
SHAPES = [(1, 70, 512), (20, 300, 1000), (40, 3000, 512), (100, 256, 8192), (300, 400, 640), (250, 8190, 640), (1000, 3000, 512),
          (2040, 4090, 520), (1900, 2900, 1000), (2100, 4000, 520)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_large_terms_that_cancel(pkg, dev, M, N, K, dtype):
    """Of each eight columns two give 256 and -256 and six 2^-6: the sum is that of the six, 0.094 for every eight columns.
    (All sums of them are multiples of 2^-6 below 2^18, exact in fp32, so the result is the exact one, rounded once.)"""
    from faster_yoco_amd import act8, linear8
    k = torch.arange(K)
    x = torch.where(k % 8 < 2, 16.0, 0.125).repeat(M, 1)
    w = torch.where(k % 8 == 0, 16.0, torch.where(k % 8 == 1, -16.0, 0.125)).repeat(N, 1)
    y = linear8.matmul(act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev), transposed=False), dtype)
    want = (x[:1].double() @ w[:1].double().t()).to(dtype)
    assert want.item() > 0.011 * K and (y.cpu() == want.item()).all()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('size', [12.0, 100.0, 1000.0])
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_channels_much_larger_than_the_rest(pkg, dev, M, N, K, size, dtype):
    from faster_yoco_amd import act8, linear8
    g = torch.Generator().manual_seed(K + N)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) * 0.05
    x[:, 5::256] *= size
    if dtype == torch.float16:
        x /= size                                      # stays within the type
    rows, outputs = slice(None, None, max(1, M // 64)), slice(None, None, max(1, N // 128))
    y = linear8.matmul(act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev), transposed=False), dtype)
    xv = ref.values(*ref.pack(x), K)[rows]
    wv = ref.weight_values(*ref.pack_weight(w)[:2], (N, K))[outputs]
    near(y[rows][:, outputs], xv @ wv.t(), xv.abs() @ wv.abs().t(), K, dtype)
