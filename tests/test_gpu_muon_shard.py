"""MuonShardOptimizer: a shard's matrices by the orthogonalised update and its other rows by Adam, bit for bit what each does
alone, under one norm, clip and factor."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(96, 40), (40,), (40, 96), (7, 5, 3), (130, 70), (1, 50), (33, 1), (129,)]
HP = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def shard_of(dev, grad_dtype=torch.bfloat16, seed=0, shapes=SHAPES, **kw):
    from faster_yoco_amd import shard
    sh = shard.FlatShard(shapes, dev, grad_dtype=grad_dtype, **kw)
    g = torch.Generator().manual_seed(seed)
    for name, scale in (('p', 0.02), ('m', 1e-3), ('g', 3e-2)):
        getattr(sh, name).copy_(torch.randn(sh.total, generator=g) * scale)
    sh.v.copy_(torch.rand(sh.total, generator=g) * 1e-6)
    if sh.p16 is not None:
        sh.p16.copy_(sh.p)
    return sh


def state(sh):
    return [getattr(sh, k).clone() for k in ('p', 'm', 'v', 'p16') if getattr(sh, k) is not None]


@pytest.mark.parametrize('matrices', [None, [2, 4], [], [0, 2, 4, 5, 6]], ids=str)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=str)
def test_each_row_as_alone(pkg, dev, dtype, matrices):
    from faster_yoco_amd import muon, shard
    one, two = shard_of(dev, dtype), shard_of(dev, dtype)
    opt = muon.MuonShardOptimizer(one, matrices, momentum=0.9, **HP)
    adam = shard.Zero1ShardOptimizer(two, **HP)
    rows = [0, 2, 4] if matrices is None else matrices
    assert opt.matrices == rows
    own = {k: [t.clone() for t in one.views(k)] for k in ('p', 'm', 'v', 'p16')}
    for step in range(2):
        opt.multiply_grads(0.5)
        adam.multiply_grads(0.5)
        assert torch.equal(opt.clip_grad_norm(0.25), adam.clip_grad_norm(0.25))
        factor = opt._multiply_factor.clone()
        assert torch.equal(factor, adam._multiply_factor)
        opt.step()
        adam.step()
        assert opt.step_count == step + 1 and opt._multiply_factor == 1.0
        p, m, p16 = ([own[k][i] for i in rows] for k in ('p', 'm', 'p16'))
        muon.step_(p, [one.views('g')[i] for i in rows], m, p16, lr=HP['lr'], weight_decay=0.1, momentum=0.9, factor=factor)
    for i in range(len(SHAPES)):
        for k in ('p', 'm', 'v', 'p16'):
            want = own[k][i] if i in rows else two.views(k)[i]
            assert torch.equal(one.views(k)[i], want), (i, k)


def test_rates_of_its_own_and_without_a_copy(pkg, dev):
    from faster_yoco_amd import muon
    sh = shard_of(dev, bf16_copy=False)
    opt = muon.MuonShardOptimizer(sh, matrix_lr=0.1, matrix_weight_decay=0.0, adjust=1.0, nesterov=False, steps=3,
                                  coefficients=(1.5, -0.5, 0.0), matrix_eps=1e-6, precise=True, **HP)
    own = {k: [sh.views(k)[i].clone() for i in opt.matrices] for k in ('p', 'm')}
    opt.step()                                                    # a factor of 1, no clip
    muon.step_(own['p'], [sh.views('g')[i] for i in opt.matrices], own['m'], lr=0.1, weight_decay=0.0, adjust=1.0, nesterov=False,
               steps=3, coefficients=(1.5, -0.5, 0.0), eps=1e-6, precise=True)
    for k in own:
        assert all(torch.equal(sh.views(k)[i], t) for i, t in zip(opt.matrices, own[k]))


def test_matrices_alone(pkg, dev):
    """A shard of nothing else: Adam has no rows and launches nothing."""
    from faster_yoco_amd import muon
    sh = shard_of(dev, shapes=[(20, 30), (30, 20)])
    opt, v = muon.MuonShardOptimizer(sh, device_step=True, **HP), sh.v.clone()
    assert opt._adam_table is None
    opt.update()
    assert torch.equal(sh.v, v) and torch.equal(sh.p16, sh.p.bfloat16()) and int(opt._step_dev) == 1


@pytest.mark.parametrize('device_step', [False, True])
def test_captured(pkg, dev, device_step):
    """An update in a graph, its gradients rewritten between replays, against eager updates."""
    from faster_yoco_amd import muon
    one, two = shard_of(dev, seed=2), shard_of(dev, seed=2)
    a, b = (muon.MuonShardOptimizer(s, device_step=device_step, **HP) for s in (one, two))
    a.update(0.5)
    b.update(0.5)
    before = state(one)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        gn = a.update(0.5)
    if device_step:
        a._step_dev.fill_(1)
    assert all(torch.equal(x, y) for x, y in zip(before, state(one)))         # capturing ran nothing
    for k in range(3):
        g = torch.randn(one.total, generator=torch.Generator().manual_seed(k)) * 0.05
        one.g.copy_(g)
        two.g.copy_(g)
        if not device_step:
            b.step_count = 1                                      # the graph holds one step's corrections
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gn, b.update(0.5))
        assert all(torch.equal(x, y) for x, y in zip(state(one), state(two)))


def test_the_reduced_forms_and_refusals(pkg, dev):
    from faster_yoco_amd import exchange, muon
    one, two = shard_of(dev, seed=3), shard_of(dev, seed=3)
    a, b = (muon.MuonShardOptimizer(s, **HP) for s in (one, two))
    parts = [(torch.randn(one.total, device=dev) * 0.01).bfloat16() for _ in range(4)]
    a.reduce_grads(parts)
    a.clip_grad_norm(0.1)
    a.step()
    b.reduce_clip(parts, 0.1)
    b.step()
    assert all(torch.equal(x, y) for x, y in zip(state(one), state(two)))
    for bad in ([1], [3], [0, 0], [8], [-1]):
        with pytest.raises(RuntimeError, match='matrices must be rows'):
            muon.MuonShardOptimizer(one, bad)
    held = state(one)
    with pytest.raises(RuntimeError, match='pieces'):
        a.step(pieces=[0, len(SHAPES)])
    with pytest.raises(RuntimeError, match='pieces'):
        exchange.PipelinedExchange(one, [0, len(SHAPES)], lambda f, l: None).step(a)
    assert a.step_count == 1 and all(torch.equal(x, y) for x, y in zip(state(one), held))
