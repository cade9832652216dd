"""CPU-side checks of the residual stream's addition and norm: argument errors of the C ABI, refusals, fake tensors."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p


def test_argument_errors_without_device_work(pkg):
    from faster_yoco_amd import _lib
    L = _lib.lib()
    NULL, SIZE, DTYPE, MODE, WS = -1, -2, -3, -5, -6
    a = P(64)                                                     # never read: every call below stops before a launch
    fwd = lambda **k: L.z1_add_norm_forward(*({'x': a, 'stride': 8, 'r': a, 'rstride': 8, 'rows': 4, 'dim': 8, 'dtype': 1,  # noqa: E731
                                               'w': None, 'b': None, 'wd': 0, 'eps': 1e-5, 'center': 1, 'h': a, 'y': a,
                                               'yq': None, 'ys': None, 'cq': None, 'cs': None, 'mean': a, 'rstd': a,
                                               'stream': None} | k).values())
    for bad, rc in (({'rows': -1}, SIZE), ({'dim': 0}, SIZE), ({'stride': -8}, SIZE), ({'rstride': -8}, SIZE),
                    ({'dtype': 3}, DTYPE), ({'wd': 2}, DTYPE), ({'center': 2}, MODE), ({'x': None}, NULL), ({'r': None}, NULL),
                    ({'h': None}, NULL), ({'mean': None}, NULL), ({'rstd': None}, NULL), ({'y': None}, NULL),
                    ({'yq': a, 'ys': a}, NULL), ({'cq': a}, NULL), ({'center': 0, 'b': a}, NULL)):
        assert fwd(**bad) == rc, bad
    assert fwd(rows=0, x=None, r=None, h=None, y=None, rstd=None) == 0
    bwd = lambda **k: L.z1_add_norm_backward(*({'dy': a, 'ds': 8, 'dh': a, 'hs': 8, 'h': a, 'xs': 8, 'q': None, 's': None,  # noqa: E731
                                                'rows': 4000, 'dim': 8, 'dtype': 1, 'mean': a, 'rstd': a, 'w': None, 'wd': 0,
                                                'center': 1, 'dx': a, 'dw': a, 'db': a, 'gd': 0, 'ws': a, 'n': 1 << 20,
                                                'stream': None} | k).values())
    for bad, rc in (({'rows': -1}, SIZE), ({'ds': -1}, SIZE), ({'hs': -1}, SIZE), ({'xs': -1}, SIZE), ({'dtype': 7}, DTYPE),
                    ({'gd': 7}, DTYPE), ({'center': 3}, MODE), ({'center': 0}, NULL), ({'dy': None}, NULL), ({'dh': None}, NULL),
                    ({'h': None}, NULL), ({'q': a, 's': a}, NULL), ({'mean': None}, NULL), ({'rstd': None}, NULL),
                    ({'dx': None}, NULL), ({'ws': None}, NULL), ({'n': 3}, WS)):
        assert bwd(**bad) == rc, bad
    assert bwd(rows=0, dy=None, dh=None, h=None, dw=None, db=None) == 0


def test_cpu_tensors_are_refused(pkg):
    from faster_yoco_amd import norm
    x, r = torch.zeros(4, 128, dtype=torch.bfloat16), torch.ones(4)
    for call in (lambda: norm.add_layer_norm(x, x), lambda: norm.add_rms_norm(x, x), lambda: norm.add_rms_norm_train(x, x),
                 lambda: norm.add_layer_norm_backward(x, x, x, r, r), lambda: norm.add_rms_norm_backward(x, x, x, r)):
        with pytest.raises(RuntimeError, match='no CPU path'):
            call()
    with pytest.raises(RuntimeError, match='a residual of'):
        norm.add_rms_norm(x, x[:3])
    with pytest.raises(RuntimeError, match='dh of'):
        norm.add_rms_norm_backward(x, x[:3], x, r)


def test_shapes_on_fake_tensors(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from faster_yoco_amd import norm
    with FakeTensorMode():
        t = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device='cuda')  # noqa: E731
        x, w = t(2, 20, 300), t(300)
        h, y, mean, rstd, c = norm.add_layer_norm(x, x, w, w, y8=True, checkpoint=True)
        assert h.shape == x.shape and y.q.shape == c.q.shape == (40, 384) and y.s.shape == (40, 4)
        assert mean.shape == rstd.shape == (40,) and mean.dtype == torch.float32
        dx, dw, db = norm.add_layer_norm_backward(x, x, c, mean, rstd, w, bias=True)
        assert dx.shape == x.shape and dw.shape == db.shape == (300,) and dw.dtype == torch.bfloat16
        h, y = norm.add_rms_norm_train(x.requires_grad_(), x, w)
        assert h.shape == y.shape == x.shape
