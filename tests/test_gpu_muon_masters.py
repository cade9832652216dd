"""The fp32 masters that a step writes by itself are as exact as their type: no caller has to ask for it."""
import math

import pytest
import torch

import matrices as ref

pytestmark = pytest.mark.gpu

SHAPES = [(64, 128), (128, 64), (150, 300), (512, 1024), (1024, 512)]


def off_and_limit(p0, g, m0, p, lr):
    """|p - its 64-bit value|, and what fp32 leaves: of p three roundings, of the update's term two, and the orthogonalised matrix
    within 3e-5 (pairs, several directions: test_gpu_muon_spectra.py), u's own rounding included: 2^-24 of u, 485 times as large
    by the end, is 2.9e-5 of a result of norm 1, and these have norms of 8 and more."""
    rate = lr * 0.2 * math.sqrt(max(p.shape))
    want, _, q, _ = ref.step(p0, g, m0, lr=lr, mu=float(torch.tensor(0.95)), nesterov=True, weight_decay=0.1, rate=rate)
    limit = 2.0 ** -24 * float((3 * p0.double().abs() + 2 * rate * q.abs()).norm()) + rate * 3e-5 * float(q.norm())
    return float((p.cpu().double() - want).norm()), limit


def state(dev):
    g = torch.Generator().manual_seed(11)
    r = lambda m, n: torch.randn(m, n, generator=g)  # noqa: E731
    return [[0.02 * r(*s) for s in SHAPES], [1e-3 * r(*s) for s in SHAPES], [1e-3 * r(*s) for s in SHAPES]]


def test_step(pkg, dev):
    from faster_yoco_amd import muon
    p0, g, m0 = state(dev)
    p, m = [t.to(dev) for t in p0], [t.to(dev) for t in m0]
    p16 = [t.bfloat16() for t in p]
    muon.step_(p, [t.to(dev) for t in g], m, p16, lr=0.01)
    for i in range(len(SHAPES)):
        off, limit = off_and_limit(p0[i], g[i], m0[i], p[i], 0.01)
        assert off <= limit, (SHAPES[i], off, limit)
        assert torch.equal(p16[i], p[i].bfloat16())


def test_shard(pkg, dev):
    from faster_yoco_amd import muon, shard
    p0, g, m0 = state(dev)
    sh = shard.FlatShard(SHAPES + [(40,)], dev)
    for name, values in (('p', p0), ('g', g), ('m', m0)):
        for t, v in zip(sh.views(name), values):
            t.copy_(v)
    muon.MuonShardOptimizer(sh, lr=0.01, weight_decay=0.1).step()
    for i in range(len(SHAPES)):
        off, limit = off_and_limit(p0[i], g[i], m0[i], sh.views('p')[i], 0.01)
        assert off <= limit, (SHAPES[i], off, limit)


def test_the_choice_is_the_callers(pkg, dev):
    """precise=True is what nothing is; precise=False is another result."""
    from faster_yoco_amd import muon
    p0, g, m0 = state(dev)
    out = []
    for kw in ({}, {'precise': True}, {'precise': False}):
        p = [t.to(dev) for t in p0]
        muon.step_(p, [t.to(dev) for t in g], [t.to(dev) for t in m0], lr=0.01, **kw)
        out.append(p)
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1]))
    assert all(not torch.equal(a, b) for a, b, s in zip(out[0], out[2], SHAPES) if min(s) > 64)
