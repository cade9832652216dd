"""CPU-side checks of the matrices' update: argument errors of the C ABI come back as codes, coefficients that let the iterates
leave their range are refused, the operators trace on fake tensors, CPU tensors are refused."""
import ctypes
import random

import pytest
import torch

P = ctypes.c_void_p
GOOD = [3.4445, -4.775, 2.0315]


def floats(v):
    return (ctypes.c_float * len(v))(*v)


def test_argument_errors_without_device_work(pkg):
    from faster_yoco_amd import _lib
    L = _lib.lib()
    NULL, SIZE, DTYPE, MODE, WS = -1, -2, -3, -5, -6
    a = P(64)                                                     # never read: every call below stops before a launch
    need = L.z1_orthogonalize_workspace(2, 300, 700, 0)
    assert need > 0 and need % 16 == 0 and L.z1_orthogonalize_workspace(2, 300, 700, 1) > need
    assert L.z1_orthogonalize_workspace(2, 700, 300, 0) == need and L.z1_orthogonalize_workspace(0, 300, 700, 0) == 0
    for bad in ((-1, 30, 70), (2, 0, 70), (2, 30, 0), (2, 30, (1 << 20) + 1), (1 << 20, 30, 70)):
        assert L.z1_orthogonalize_workspace(*bad, 0) == SIZE
    call = lambda **k: L.z1_orthogonalize(*({'x': a, 'step': 2100, 'stride': 700, 'count': 2, 'm': 300, 'n': 700, 'dtype': 1,  # noqa: E731
                                             'out': a, 'od': 1, 'steps': 1, 'c': floats(GOOD), 'eps': 1e-7, 'precise': 0,
                                             'ws': a, 'bytes': need, 'stream': None} | k).values())
    for bad, rc in (({'count': -1}, SIZE), ({'m': 0}, SIZE), ({'n': 1 << 21}, SIZE), ({'stride': -1}, SIZE), ({'step': -1}, SIZE),
                    ({'dtype': 5}, DTYPE), ({'od': 5}, DTYPE), ({'steps': 0}, SIZE), ({'steps': 65}, SIZE), ({'c': None}, NULL),
                    ({'x': None}, NULL), ({'out': None}, NULL), ({'eps': 0.0}, MODE), ({'eps': -1.0}, MODE),
                    ({'eps': float('nan')}, MODE), ({'c': floats([4.5, 0, 0])}, MODE), ({'ws': None}, NULL),
                    ({'bytes': need - 1}, WS), ({'precise': 1}, WS)):
        assert call(**bad) == rc, bad
    assert call(count=0, x=None, out=None, ws=None) == 0
    matrix = lambda **k: _lib.Z1Matrix(*({'g': a, 'stride': 700, 'momentum': a, 'p': a, 'p16': None, 'm': 300, 'n': 700,  # noqa: E731
                                          'lr': 1e-3, 'keep': 1.0} | k).values())
    two = lambda **k: (_lib.Z1Matrix * 2)(matrix(), matrix(**k))  # noqa: E731
    need = L.z1_muon_workspace(two(), 2, 0)
    assert need == L.z1_orthogonalize_workspace(2, 300, 700, 0) and L.z1_muon_workspace(two(), 2, 1) > need
    assert L.z1_muon_workspace(None, 0, 0) == 0 and L.z1_muon_workspace(None, 1, 0) == NULL
    assert L.z1_muon_workspace(two(), 33, 0) == L.z1_muon_workspace(two(), -1, 0) == SIZE
    assert L.z1_muon_workspace(two(m=0), 2, 0) == L.z1_muon_workspace(two(n=1 << 21), 2, 0) == SIZE
    good = _lib.Z1Muon(None, 0.9, 1, 1, floats(GOOD), 1e-7, 0)
    how = lambda **k: ctypes.byref(_lib.Z1Muon(*({'f': None, 'mu': 0.9, 'n': 1, 'steps': 1, 'c': floats(GOOD), 'eps': 1e-7,  # noqa: E731
                                                  'precise': 0} | k).values()))
    step = lambda **k: L.z1_muon_step(*({'list': two(), 'count': 2, 'dtype': 1, 'how': ctypes.byref(good), 'ws': a,  # noqa: E731
                                         'bytes': need, 'stream': None} | k).values())
    for bad, rc in (({'count': -1}, SIZE), ({'count': 33}, SIZE), ({'list': two(m=0)}, SIZE), ({'dtype': 9}, DTYPE),
                    ({'how': None}, NULL), ({'list': None}, NULL), ({'list': two(g=None)}, NULL), ({'list': two(p=None)}, NULL),
                    ({'list': two(momentum=None)}, NULL), ({'list': two(stride=-1)}, SIZE), ({'how': how(steps=0)}, SIZE),
                    ({'how': how(c=None)}, NULL), ({'how': how(eps=0.0)}, MODE), ({'how': how(c=floats([9, 0, 0]))}, MODE),
                    ({'ws': None}, NULL), ({'bytes': need - 1}, WS), ({'how': how(precise=1)}, WS)):
        assert step(**bad) == rc, bad
    assert step(count=0, list=None, ws=None) == 0


def test_coefficients_are_admitted_as_the_polynomial_says(pkg):
    """Against the polynomial sampled densely: what is admitted stays below 4 (and B below 32), what is refused comes within a
    part in a hundred of leaving it."""
    from faster_yoco_amd import _lib
    L = _lib.lib()
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    for k in range(400):
        steps = rng.choice((1, 2, 5))
        c = [[rng.uniform(0, 4.2), rng.uniform(-6, 1), rng.choice((0.0, rng.uniform(-1, 4)))] for _ in range(steps)]
        if k == 0:
            c = [GOOD] * 5
        rc = L.z1_orthogonalize(P(64), 0, 700, 1, 300, 700, 0, P(64), 0, len(c), floats([v for t in c for v in t]), 1e-7, 0, None, 0, None)
        admitted = rc == -1                                       # the missing workspace is what it stops at
        assert admitted or rc == -5
        seen[admitted] += 1
        top, large = 1.0, 0.0
        for t in c:
            a, b, d = (ctypes.c_float(v).value for v in t)
            s = torch.linspace(0, 1, 20001, dtype=torch.float64) * top
            large = max(large, float((b * s ** 2 + d * s ** 4).abs().max()))
            top = float((a * s + b * s ** 3 + d * s ** 5).abs().max())
            if top > 1e6:
                break
            if admitted:
                assert top < 4.0 and large < 32.0
        most = []
        if not admitted:
            top = 1.0
            for t in c:
                s = torch.linspace(0, 1, 20001, dtype=torch.float64) * top * 1.002
                most.append(float((t[1] * s ** 2 + t[2] * s ** 4).abs().max()) / 32)
                top = float((t[0] * s + t[1] * s ** 3 + t[2] * s ** 5).abs().max())
                most.append(top / 4)
                if top > 4:
                    break
            assert max(most) > 0.95
    assert min(seen.values()) > 20


def test_operators_and_their_writes(pkg):
    from faster_yoco_amd import library
    assert set(library.MATRIX_OPS) == {'orthogonalize', 'muon_step_'}
    written = lambda n: [a.name for a in getattr(torch.ops.yoco_z1, n).default._schema.arguments  # noqa: E731
                         if a.alias_info is not None and a.alias_info.is_write]
    assert written('orthogonalize') == [] and written('muon_step_') == ['p', 'momentum', 'p16']


def test_cpu_tensors_and_wrong_arguments_are_refused(pkg):
    from faster_yoco_amd import muon
    x = torch.zeros(4, 6)
    for call in (lambda: muon.orthogonalize(x), lambda: muon.step_([x], [x], [x.clone()], lr=1.0)):
        with pytest.raises(RuntimeError, match='no CPU path'):
            call()
    for call, text in ((lambda: muon.orthogonalize(x[0]), 'matrices'),
                       (lambda: muon.orthogonalize(x, coefficients=[1.0, 2.0, 3.0, 4.0, 5.0]), 'triple'),
                       (lambda: muon.orthogonalize(x, coefficients=[(1.0, 2.0)] * 5), 'triple'),
                       (lambda: muon.orthogonalize(x, steps=1 << 60), '1 to 64 steps'),
                       (lambda: muon.orthogonalize(x, steps=-1), '1 to 64 steps'),
                       (lambda: muon.step_([x], [x], [x], lr=1.0, adjust='none'), 'adjust')):
        with pytest.raises(RuntimeError, match=text):
            call()
    assert muon.step_([], [], [], lr=1.0) is None
    assert muon.rate(1.0, (4, 9), 'rms') == pytest.approx(0.6) and muon.rate(1.0, (9, 4), 'shape') == 1.5
    assert muon.rate(2.0, (9, 4), 0.25) == 0.5


def test_shapes_on_fake_tensors(pkg):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from faster_yoco_amd import muon
    with FakeTensorMode():
        x = torch.empty(2, 3, 30, 70, dtype=torch.float16, device='cuda')
        assert muon.orthogonalize(x).shape == x.shape and muon.orthogonalize(x).dtype == torch.float16
        assert muon.orthogonalize(x, dtype=torch.bfloat16).dtype == torch.bfloat16
        p, m = torch.empty(30, 70, device='cuda'), torch.empty(30, 70, device='cuda')
        muon.step_([p], [x[0, 0]], [m], [p.bfloat16()], lr=1e-3)


def test_every_form_has_a_tested_size(pkg):
    """The sizes that the GPU tests run take every form that any size takes."""
    import math

    import ways_muon
    from faster_yoco_amd import _lib
    L = _lib.lib()
    rng = random.Random(7)
    size = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi))))  # noqa: E731
    for precise, tested in ((0, ways_muon.FAST), (1, ways_muon.PRECISE)):
        covered = set().union(*(ways_muon.forms(L, *t, precise) for t in tested))
        seen = set()
        for _ in range(20000):
            seen |= ways_muon.forms(L, size(1, 300), size(1, 9000), size(1, 9000), precise)
        assert seen <= covered, seen - covered
    way = (ctypes.c_int * 12)()
    assert L.z1_orthogonalize_way(0, 8, 8, 0, way) == L.z1_orthogonalize_way(1, 0, 8, 0, way) == -2
    assert L.z1_orthogonalize_way(1, 8, 8, 0, None) == -1
