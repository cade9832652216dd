"""What lies behind the operands of the 8-bit products and weight gradients, in the same allocation, does not reach a result:
rows, outputs and tokens past the end are NaN here, in every tile and part that an end can fall into."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BEHIND = 600                                          # rows of NaN: more than any tile has


def rows(n, dim, seed):
    g = torch.Generator().manual_seed(seed + 7 * n + dim)
    return torch.randn(n, dim, generator=g).bfloat16()


def before_nan(x, dev):
    return torch.cat([x, torch.full((BEHIND, x.shape[1]), float('nan'), dtype=x.dtype)]).to(dev)


@pytest.mark.parametrize('M,N,K', [(1, 70, 300), (33, 70, 700), (33, 4100, 640), (64, 130, 2300), (65, 257, 1000), (100, 256, 8192),
                                   (130, 129, 513), (257, 300, 4100), (333, 1501, 1000), (1900, 2900, 1300), (2100, 4001, 520)])
def test_rows_behind_a_product(pkg, dev, M, N, K):
    from faster_yoco_amd import act8, linear8
    x, w = rows(M, K, 1), rows(N, K, 2)
    a, p = act8.pack(before_nan(x, dev)), linear8.pack_weight(before_nan(w, dev), transposed=False)
    assert a.q[M:].float().isnan().sum() == BEHIND * K
    a = act8.Act8(a.q[:M], a.s[:M], K)
    p = linear8.Weight8(p.q[:N], p.s[:-(-N // 128)], None, None, (N, K))
    for dtype in (torch.bfloat16, torch.float32):
        y = linear8.matmul(a, p, dtype)
        want = linear8.matmul(act8.pack(x.to(dev)), linear8.pack_weight(w.to(dev)), dtype)
        assert y.isfinite().all() and torch.equal(y, want)


@pytest.mark.parametrize('T,N,K', [(1, 130, 200), (1, 131, 200), (33, 256, 300), (63, 65, 300), (64, 128, 128), (65, 300, 129),
                                   (100, 1000, 513), (333, 1502, 1000), (500, 2100, 4000), (3001, 64, 300), (3001, 65, 300),
                                   (70, 6, 40), (70, 7, 40)])
def test_tokens_behind_a_gradient(pkg, dev, T, N, K):
    from faster_yoco_amd import act8, linear8
    x, dy = rows(T, K, 3), rows(T, N, 4)
    a = act8.pack(before_nan(x, dev))
    a = act8.Act8(a.q[:T], a.s[:T], K)
    for dtype in (torch.bfloat16, torch.float32):
        dw = linear8.weight_grad(before_nan(dy, dev)[:T], a, dtype)
        want = linear8.weight_grad(dy.to(dev), act8.pack(x.to(dev)), dtype)
        assert dw.isfinite().all() and torch.equal(dw, want)
