"""8-bit rows and weights on the GPU against a plain 64-bit form: every byte and every scale, for all types, odd sizes and
strides, blocks of zeros, subnormals, the types' largest values, infinities and NaN."""
import pytest
import torch

import blocks as ref
from blocks import DTYPES, E8, F8

pytestmark = pytest.mark.gpu


def rows(n, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, dim, generator=g, dtype=torch.float64) * torch.exp(2 * torch.randn(1, dim, generator=g, dtype=torch.float64))
    return x.to(dtype)


def check(a, x):
    q, s = ref.pack(x)
    assert a.q.dtype == F8 and a.s.dtype == E8 and a.dim == x.shape[1]
    assert tuple(a.q.shape) == tuple(q.shape) and tuple(a.s.shape) == tuple(s.shape)
    assert torch.equal(ref.codes(a.s), s)
    assert ref.same_codes(a.q, q)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('n,dim', [(1, 1), (1, 7), (3, 8), (2, 127), (5, 128), (70, 129), (3, 511), (2, 512), (2, 513),
                                   (333, 1000), (9, 4099), (1, 20000)])
def test_pack_and_unpack(pkg, dev, n, dim, dtype):
    from faster_yoco_amd import act8
    x = rows(n, dim, dtype)
    a = act8.pack(x.to(dev))
    check(a, x)
    want = ref.values(*ref.pack(x), dim)
    for t in DTYPES:
        got = act8.unpack(a, t).cpu().double()
        assert got.shape == (n, dim)
        v = want.clamp(-ref.LARGEST[t], ref.LARGEST[t])
        assert (got - v).abs().le(ref.rounded(v, t) * (t == torch.float16)).all()         # exact but for fp16's range


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_strides_and_leading_dimensions(pkg, dev, dtype):
    from faster_yoco_amd import act8
    base = rows(40, 1031, dtype, 1)
    d = base.to(dev)
    check(act8.pack(d[:, 3:703]), base[:, 3:703])                 # rows at odd elements
    check(act8.pack(d[::3, 1:130]), base[::3, 1:130])
    check(act8.pack(d.t()), base.t().contiguous())                # elements apart: copied
    check(act8.pack(d[:, :640].reshape(4, 10, 640)), base[:, :640])
    check(act8.pack(d[7]), base[7:8])
    check(act8.pack(d[5:6].expand(6, 1031)), base[5:6].expand(6, 1031))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_special_values(pkg, dev, dtype):
    """Blocks that are all zeros, all NaN, hold an infinity, subnormals, the type's largest and smallest values, and
    maxima on either side of where the scale steps."""
    from faster_yoco_amd import act8
    info = torch.finfo(dtype)
    x = rows(24, 384, dtype, 2)
    x[0, :128] = 0
    x[1, 128:256] = float('nan')
    x[2, 5] = float('inf')
    x[3, 300] = -float('inf')
    x[3, 301] = float('nan')
    x[4] = float('inf')
    x[5, :128] = info.max
    x[6, :128] = -info.max
    x[7, :128] = info.smallest_normal
    x[8, :128] = info.smallest_normal * info.eps                  # the smallest subnormal
    x[9, :128] = 0
    x[9, 3] = info.smallest_normal * info.eps
    for i, m in enumerate((448.0, 450.0, 1.75, 1.7578125, 3.5, 3.515625, 0.4375, 0.439453125)):
        x[10 + i, 128:256] = torch.linspace(-1, 1, 128).to(dtype) * m
        x[10 + i, 200] = m
    x[20] = -0.0
    a = act8.pack(x.to(dev))
    check(a, x)
    q, s = ref.pack(x)
    for t in DTYPES:
        got, want = act8.unpack(a, t).cpu().double(), ref.values(q, s, 384)
        assert torch.equal(got.isnan(), want.isnan()) and not got.isinf().any()
        v = want.nan_to_num(0.0).clamp(-ref.LARGEST[t], ref.LARGEST[t])
        assert (got.nan_to_num(0.0) - v).abs().le(ref.rounded(v, t)).all()


def test_every_code_comes_back(pkg, dev):
    """Packing what 8-bit rows stand for gives them again (largest code in each block, so that the scale stays)."""
    from faster_yoco_amd import act8
    v = torch.arange(256, dtype=torch.uint8).view(F8).double()
    x = torch.cat([v[:127], v[126:127], v[128:255], v[254:255]])[None].repeat(5, 1)
    x *= torch.tensor([1.0, 2.0 ** -100, 2.0 ** 100, 2.0 ** 7, 2.0 ** -13], dtype=torch.float64)[:, None]
    a = act8.pack(x.float().to(dev))
    assert torch.equal(ref.values(ref.codes(a.q), ref.codes(a.s), 256), x)
    assert torch.equal(act8.unpack(a, torch.float32).cpu().double(), x)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('N,K', [(1, 1), (1, 300), (127, 129), (128, 128), (200, 1), (513, 257), (1501, 1000)])
def test_weights(pkg, dev, N, K, dtype):
    from faster_yoco_amd import linear8
    w = rows(N, K, dtype, 3)
    want = ref.pack_weight(w)
    got = linear8.pack_weight(w.to(dev))
    assert tuple(got.shape) == (N, K)
    for g, v in zip((got.q, got.s, got.qt, got.st), want):
        assert tuple(g.shape) == tuple(v.shape)
    assert torch.equal(ref.codes(got.s), want[1]) and torch.equal(ref.codes(got.st), want[3])
    assert ref.same_codes(got.q, want[0]) and ref.same_codes(got.qt, want[2])
    one = linear8.pack_weight(w.to(dev), transposed=False)
    assert one.qt is None and torch.equal(ref.codes(one.q), ref.codes(got.q))


def test_weight_special_values(pkg, dev):
    from faster_yoco_amd import linear8
    w = rows(300, 300, torch.bfloat16, 4)
    w[:128, :128] = 0
    w[130, 5] = float('inf')
    w[140, 140] = float('nan')
    w[:128, 256:] = float('nan')
    w[256:, 256:] = torch.finfo(torch.bfloat16).max
    want = ref.pack_weight(w)
    big = torch.zeros(300, 700, dtype=torch.bfloat16)
    big[:, 31:331] = w
    got = linear8.pack_weight(big.to(dev)[:, 31:331])             # rows at odd elements
    assert torch.equal(ref.codes(got.s), want[1]) and torch.equal(ref.codes(got.st), want[3])
    assert ref.same_codes(got.q, want[0]) and ref.same_codes(got.qt, want[2])


def test_no_rows(pkg, dev):
    from faster_yoco_amd import act8
    a = act8.pack(torch.empty(0, 200, dtype=torch.bfloat16, device=dev))
    assert tuple(a.q.shape) == (0, 256) and tuple(a.s.shape) == (0, 4)
    assert tuple(act8.unpack(a).shape) == (0, 200)


def test_offsets_past_32_bits(pkg, dev):
    """2.2e9 elements: the last rows are packed and unpacked like the same rows alone."""
    from faster_yoco_amd import act8
    n, dim = 65793, 33001
    assert n * dim > 2 ** 31
    x = torch.zeros(n, dim, dtype=torch.bfloat16, device=dev)
    last = rows(5, dim, torch.bfloat16, 5).to(dev)
    x[-5:] = last
    a, b = act8.pack(x), act8.pack(last)
    assert torch.equal(a.q[-5:].view(torch.uint8), b.q.view(torch.uint8))
    assert torch.equal(a.s[-5:].view(torch.uint8), b.s.view(torch.uint8))
    assert not a.q[:-5].view(torch.uint8).any()
    del x
    y = act8.unpack(a)
    assert torch.equal(y[-5:], act8.unpack(b)) and not y[:-5].any()


def test_other_stream_and_graph(pkg, dev):
    """On a stream of its own, and replayed from a graph with eager work between the replays."""
    from faster_yoco_amd import act8
    x = rows(37, 700, torch.bfloat16, 6).to(dev)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = act8.pack(x)
        y = act8.unpack(a)
    torch.cuda.current_stream().wait_stream(st)
    check(a, x.cpu())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = act8.pack(x)
        z = act8.unpack(a)
    for seed in (7, 8, 9):
        x.copy_(rows(37, 700, torch.bfloat16, seed).to(dev))
        want = act8.unpack(act8.pack(x))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want)
    assert y.shape == z.shape


def test_refusals(pkg, dev):
    from faster_yoco_amd import act8, linear8
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    a = act8.pack(x)
    with pytest.raises(RuntimeError, match='no CPU path'):
        act8.pack(x.cpu())
    with pytest.raises(RuntimeError, match='expected fp32, bf16 or fp16'):
        act8.pack(x.double())
    with pytest.raises(RuntimeError, match='at least one column'):
        act8.pack(x[:, :0])
    with pytest.raises(RuntimeError, match='at least one dimension'):
        act8.pack(x[0, 0])
    with pytest.raises(RuntimeError, match='expected fp32, bf16 or fp16'):
        act8.unpack(a, torch.float64)
    for bad in (act8.Act8(a.q, a.s, 129), act8.Act8(a.q, a.s, 300), act8.Act8(a.q[:3], a.s, 256),
                act8.Act8(a.q, a.s[:, :3], 256), act8.Act8(a.q.view(torch.uint8), a.s, 256),
                act8.Act8(a.q, a.s.view(torch.uint8), 256), act8.Act8(a.q, a.s.cpu(), 256),
                act8.Act8(torch.empty(4 * 256 + 8, dtype=torch.uint8, device=dev)[8:].view(4, 256).view(F8), a.s, 256)):
        if bad.dim == 129:
            assert act8.unpack(bad).shape == (4, 129)             # the same blocks, fewer columns of the last
            continue
        with pytest.raises(RuntimeError, match='act8.unpack'):
            act8.unpack(bad)
    with pytest.raises(RuntimeError, match=r'a weight \[N, K\]'):
        linear8.pack_weight(x[0])
    with pytest.raises(RuntimeError, match='at least one row'):
        linear8.pack_weight(x[:0])
    with pytest.raises(RuntimeError, match='at least one column'):
        linear8.pack_weight(x[:, :0])
