"""CPU-side checks of the block-side operators (no kernel launches): argument errors of the C ABI come back as codes, the
operators are registered, write none of their arguments, trace on fake tensors with the shapes they return, and refuse CPU
tensors."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

P = ctypes.c_void_p


def test_operators_are_registered_and_write_nothing(pkg):
    from faster_yoco_amd import library
    for name in library.BLOCK_OPS:
        schema = getattr(torch.ops.yoco_z1, name).default._schema
        assert schema.returns and not any(a.alias_info is not None for a in schema.arguments)


def test_argument_errors_without_device_work(pkg):
    from faster_yoco_amd import _lib
    L = _lib.lib()
    NULL, SIZE, DTYPE, MODE, WS = -1, -2, -3, -5, -6
    a = P(64)                                                     # never read: every call below stops before a launch
    fwd = lambda **k: L.z1_norm_forward(*({'x': a, 'rows': 4, 'dim': 8, 'stride': 8, 'dtype': 1, 'w': None, 'b': None,  # noqa: E731
                                           'wd': 0, 'eps': 1e-5, 'center': 1, 'y': a, 'yq': None, 'ys': None, 'cq': None,
                                           'cs': None, 'mean': a, 'rstd': a, 'stream': None} | k).values())
    for bad, rc in (({'rows': -1}, SIZE), ({'dim': 0}, SIZE), ({'dim': 1 << 25}, SIZE), ({'stride': -8}, SIZE),
                    ({'dtype': 3}, DTYPE), ({'wd': 2}, DTYPE), ({'center': 2}, MODE), ({'x': None}, NULL),
                    ({'mean': None}, NULL), ({'rstd': None}, NULL), ({'y': None}, NULL), ({'yq': a, 'ys': a}, NULL),
                    ({'y': None, 'yq': a}, NULL), ({'cq': a}, NULL), ({'center': 0, 'b': a}, NULL)):
        assert fwd(**bad) == rc, bad
    assert fwd(rows=0, x=None, y=None, rstd=None) == 0
    bwd = lambda **k: L.z1_norm_backward(*({'dy': a, 'ds': 8, 'x': a, 'xs': 8, 'q': None, 's': None, 'rows': 4000, 'dim': 8,  # noqa: E731
                                            'dtype': 1, 'mean': a, 'rstd': a, 'w': None, 'wd': 0, 'center': 1, 'dx': a,
                                            'dw': a, 'db': a, 'gd': 0, 'ws': a, 'n': 1 << 20, 'stream': None} | k).values())
    for bad, rc in (({'rows': -1}, SIZE), ({'dim': 0}, SIZE), ({'ds': -1}, SIZE), ({'xs': -1}, SIZE), ({'dtype': 7}, DTYPE),
                    ({'gd': 7}, DTYPE), ({'wd': 2}, DTYPE), ({'center': 3}, MODE), ({'center': 0}, NULL), ({'dy': None}, NULL),
                    ({'x': None}, NULL), ({'q': a, 's': a}, NULL), ({'x': None, 'q': a}, NULL), ({'mean': None}, NULL),
                    ({'rstd': None}, NULL), ({'dx': None}, NULL), ({'ws': None}, NULL), ({'n': 3}, WS)):
        assert bwd(**bad) == rc, bad
    assert bwd(rows=0, dy=None, x=None, dw=None, db=None) == 0
    assert L.z1_norm_backward_workspace(-1, 8) == SIZE and L.z1_norm_backward_workspace(4, 0) == SIZE
    # few rows go in one launch and need none
    assert L.z1_norm_backward_workspace(0, 8) == L.z1_norm_backward_workspace(5, 8) == 0
    assert L.z1_norm_backward_workspace(5000, 8) >= 16
    assert [L.z1_act8_columns(d) for d in (1, 128, 129, 0, -3)] == [128, 128, 256, SIZE, SIZE]
    assert [L.z1_act8_scales(d) for d in (1, 512, 513, 0)] == [4, 4, 8, SIZE]
    assert L.z1_act8_pack(a, -1, 8, 8, 0, a, a, None) == SIZE and L.z1_act8_pack(a, 4, 0, 8, 0, a, a, None) == SIZE
    assert L.z1_act8_pack(a, 1 << 40, 1 << 20, 8, 0, a, a, None) == SIZE
    assert L.z1_act8_pack(a, 4, 8, 8, 9, a, a, None) == DTYPE and L.z1_act8_pack(a, 4, 8, 8, 0, None, a, None) == NULL
    assert L.z1_act8_pack(None, 0, 8, 8, 0, None, None, None) == 0
    assert L.z1_act8_unpack(a, a, 4, 8, a, 9, None) == DTYPE and L.z1_act8_unpack(a, None, 4, 8, a, 0, None) == NULL
    assert L.z1_act8_unpack(a, a, 4, -8, a, 0, None) == SIZE and L.z1_act8_unpack(None, None, 0, 8, None, 0, None) == 0
    assert L.z1_weight8_pack(a, -1, 8, 8, 0, a, a, a, a, None) == SIZE
    assert L.z1_weight8_pack(a, 8, 8, 8, 5, a, a, a, a, None) == DTYPE
    assert L.z1_weight8_pack(a, 8, 8, 8, 0, a, a, a, None, None) == NULL
    mul = lambda M, N, K, dtype, ws=None, n=0, p=a: L.z1_product8(p, p, M, a, a, N, K, a, dtype, ws, n, None)  # noqa: E731
    assert mul(-1, 8, 8, 0) == SIZE and mul(4, 8, 0, 0) == SIZE and mul(4, 8, 8, 4) == DTYPE and mul(4, 8, 8, 0, p=None) == NULL
    assert L.z1_product8(None, None, 0, None, None, 8, 8, None, 0, None, 0, None) == 0
    need = L.z1_product8_workspace(100, 256, 8192, 1)              # few tiles, a long K: partial results
    assert need >= 2 * 100 * 256 and need % (100 * 256) == 0
    assert mul(100, 256, 8192, 1) == NULL and mul(100, 256, 8192, 1, a, need - 1) == WS
    assert L.z1_product8_workspace(8, 8192, 8192, 1) == 0 and L.z1_product8_workspace(0, 8, 8, 1) == 0
    assert L.z1_product8_workspace(4, 8, -1, 1) == SIZE and L.z1_product8_workspace(4, 8, 8, 9) == DTYPE
    grad = lambda T, N, K, stride, dtype, ws=None, n=0, p=a: L.z1_weight_grad8(p, stride, a, a, T, N, K, a, dtype, ws, n, None)  # noqa: E731
    assert grad(4, 8, 8, -1, 0) == SIZE and grad(4, 8, 8, (1 << 24) + 1, 0) == SIZE and grad(4, 8, 8, 8, 4) == DTYPE
    assert grad(4, 8, 8, 8, 0, p=None) == NULL
    need = L.z1_weight_grad8_workspace(8192, 256, 256)
    assert need >= 2 * 256 * 256 and need % (256 * 256) == 0
    assert grad(8192, 256, 256, 256, 1) == NULL and grad(8192, 256, 256, 256, 1, a, need - 1) == WS
    assert L.z1_weight_grad8_workspace(8, 8, 0) == SIZE and L.z1_weight_grad8_workspace(0, 8, 8) == 0


def test_python_surfaces_refuse_cpu_tensors(pkg):
    from faster_yoco_amd import act8, linear8, norm
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    a = act8.Act8(torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn),
                  torch.zeros(4, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu), 128)
    w = linear8.Weight8(a.q, a.s[:1], a.q, a.s, (4, 128))
    r = torch.ones(4)
    for call in (lambda: act8.pack(x), lambda: act8.unpack(a), lambda: linear8.pack_weight(x), lambda: linear8.matmul(a, w),
                 lambda: linear8.weight_grad(x, a), lambda: norm.layer_norm(x), lambda: norm.rms_norm(x),
                 lambda: norm.layer_norm_backward(x, x, r, r), lambda: norm.rms_norm_backward(x, a, r)):
        with pytest.raises(RuntimeError, match='no CPU path'):
            call()


def test_rows_of_views_where_strides_allow(pkg):
    from faster_yoco_amd import act8
    x = torch.arange(240.0).view(4, 6, 10)
    assert act8.rows_of(x).data_ptr() == x.data_ptr() and act8.rows_of(x).shape == (24, 10)
    assert act8.rows_of(x[0, 0]).shape == (1, 10)
    assert act8.rows_of(x[:, :, 2:5]).stride() == (10, 1)         # still a view
    t = act8.rows_of(x[0].t())
    assert t.is_contiguous() and torch.equal(t, x[0].t())
    e = torch.ones(()).expand(5, 7)
    assert act8.rows_of(e).is_contiguous()
    assert act8.rows_of(torch.empty(3, 0, 10)).shape == (0, 10)
    assert act8.rows_of(torch.empty(0, 5, 0)).shape == (0, 0)


def test_a_block_traces_on_fake_tensors(pkg):
    """Norm -> product -> gradients traced with fake tensors: every launch is an operator node, and the shapes agree."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from faster_yoco_amd import act8, linear8, norm

    def block(x, w, b, weight, dy):
        a, mean, rstd, c = norm.layer_norm(x, w, b, y8=True, checkpoint=True)
        p = linear8.pack_weight(weight)
        y = linear8.matmul(a, p)
        d = linear8.matmul(act8.pack(dy), p, transposed=True)
        dw = linear8.weight_grad(dy, a)
        return (y, dw, act8.unpack(a), *norm.layer_norm_backward(d, c, mean, rstd, w, bias=True))

    with FakeTensorMode():
        t = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device='cuda')  # noqa: E731
        args = (t(40, 300), t(300), t(300), t(500, 300), t(40, 500))
        gm = make_fx(block, tracing_mode='fake')(*args)
        out = block(*args)
    assert [tuple(o.shape) for o in out] == [(40, 500), (500, 300), (40, 300), (40, 300), (300,), (300,)]
    called = [str(n.target) for n in gm.graph.nodes if n.op == 'call_function' and 'yoco_z1' in str(n.target)]
    assert called == [f'yoco_z1.{n}.default' for n in ('norm_forward', 'weight8_pack', 'product8', 'act8_pack', 'product8',
                                                       'weight_grad8', 'act8_unpack', 'norm_backward')]


def test_a_given_gradient_type_on_fake_tensors(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    op = torch.ops.yoco_z1.norm_backward
    with FakeTensorMode():
        x, r = torch.empty(40, 300, dtype=torch.bfloat16, device='cuda'), torch.empty(40, device='cuda')
        types = lambda *a: [t.dtype for t in op(x, x, None, None, r, r, None, True, False, True, *a)]  # noqa: E731
        assert types() == [torch.bfloat16] * 2 and types(torch.float32) == [torch.bfloat16, torch.float32]


def test_a_build_without_the_block_side_functions_is_accepted(pkg, tmp_path):
    """A library of the update's functions alone binds; one that lacks any of those is refused by name."""
    from faster_yoco_amd import _lib
    names = [n for n in _lib.SIGNATURES if n not in _lib.BLOCK_SIGNATURES]
    assert len(names) > 20 and len(_lib.BLOCK_SIGNATURES) >= 12

    def imported(names, code):
        src, lib = tmp_path / 'stub.c', tmp_path / f'stub{len(names)}.so'
        src.write_text(''.join(f'int {n}(void) {{ return 0; }}\n' for n in names))
        subprocess.run(['gcc', '-shared', '-fPIC', '-o', str(lib), str(src)], check=True)
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        return subprocess.run([sys.executable, '-c', code], cwd=root, env=dict(os.environ, YOCO_Z1_LIB=str(lib)),
                              capture_output=True, text=True)
    res = imported(names, 'import faster_yoco_amd as f\nL = f._lib.lib()\nassert L.z1_owner_sum_waves(5) == 0\n'
                          "assert not hasattr(L, 'z1_norm_forward')\nprint('bound')")
    assert res.returncode == 0 and res.stdout.strip() == 'bound', res.stderr
    res = imported(names[1:], 'import faster_yoco_amd')
    assert res.returncode != 0 and f'RuntimeError: yoco_z1: {tmp_path}' in res.stderr and f'has no {names[0]}' in res.stderr


def test_every_form_of_the_products_has_a_tested_shape(pkg):
    """The shapes that the GPU tests run are in the forms they are listed under, and no shape takes a form that is not listed."""
    import math
    import random

    import ways
    from faster_yoco_amd import _lib
    L = _lib.lib()
    for form, shape in ways.PRODUCTS.items():
        assert ways.product(L, *shape) == form, shape
    for form, (T, N, K) in ways.GRADIENTS.items():
        assert ways.gradient(L, T, N, K, N % 2 == 0) == form, (T, N, K)
    rng = random.Random(5)
    size = lambda hi: int(math.exp(rng.uniform(0, math.log(hi))))  # noqa: E731
    products, gradients = set(), set()
    for _ in range(60000):
        M, N, K = size(20000), size(20000), size(20000)
        products.add(ways.product(L, M, N, K))
        gradients.add(ways.gradient(L, M, N, K, rng.random() < 0.5))
    assert products == set(ways.PRODUCTS) and gradients == set(ways.GRADIENTS)
    way = (ctypes.c_int * 4)()
    assert L.z1_product8_way(0, 8, 8, way) == L.z1_weight_grad8_way(8, 8, 0, 1, way) == -2
    assert L.z1_product8_way(8, 8, 8, None) == L.z1_weight_grad8_way(8, 8, 8, 1, None) == -1
