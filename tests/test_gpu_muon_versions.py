"""What a step writes in place is known to autograd as written: a backward pass over values from before it is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('size', [(6, 4), (150, 140)], ids=['small', 'large'])
def test_versions_advance(pkg, dev, size):
    from faster_yoco_amd import muon
    p, g, m = (torch.full(size, v, device=dev) for v in (1.0, 0.5, 0.25))
    c = p.bfloat16()
    before = [t._version for t in (p, m, c)]
    muon.step_([p], [g], [m], [c], lr=0.1)
    assert [t._version for t in (p, m, c)] == [v + 1 for v in before] and g._version == 0
    ops = torch.ops.yoco_z1.muon_step_
    ops([p], [g], [m], [c], None, [0.1], [1.0], 0.9, True, 1, [3.0, -3.2, 1.2], 1e-7, True)
    assert [t._version for t in (p, m, c)] == [v + 2 for v in before] and g._version == 0


def test_a_backward_pass_over_what_was_written_is_refused(pkg, dev):
    from faster_yoco_amd import muon
    w = torch.nn.Parameter(torch.randn(30, 20, device=dev))
    x = torch.randn(5, 20, device=dev, requires_grad=True)
    y = (x @ w.t()).square().sum()
    muon.step_([w], [torch.ones_like(w)], [torch.zeros_like(w)], lr=0.1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    (x @ w.t()).sum().backward()                                  # a forward pass from after it is not
    assert torch.equal(x.grad, w.detach().sum(0).expand(5, 20)) or (x.grad - w.detach().sum(0)).abs().max() < 1e-4


def test_a_shards_views_and_inference(pkg, dev):
    """A view's version is its buffer's; tensors made in inference mode have none."""
    from faster_yoco_amd import muon, shard
    sh = shard.FlatShard([(20, 30), (30, 20)], dev)
    sh.g.fill_(1.0)
    leaf = sh.views('p16')[0].detach().requires_grad_()
    x = torch.ones(4, 30, device=dev, dtype=torch.bfloat16, requires_grad=True)
    y = (x @ leaf.t()).sum()
    muon.MuonShardOptimizer(sh).step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    with torch.inference_mode():
        p = [torch.ones(20, 30, device=dev)]
        muon.step_(p, [torch.ones(20, 30, device=dev)], [torch.zeros(20, 30, device=dev)], lr=0.1)
        assert p[0].isfinite().all() and (p[0] != 1).any()


def test_captured_and_compiled(pkg, dev):
    """A captured step bumps when it is captured, as torch's own in-place operators do, and runs when it is replayed; a compiled
    one gives the eager bits."""
    from faster_yoco_amd import muon
    a, b, c = ([torch.full((70, 90), v, device=dev) for v in (1.0, 0.5, 0.25)] for _ in range(3))
    step = lambda t: muon.step_([t[0]], [t[1]], [t[2]], lr=0.1)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(a)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        step(b)
        torch.compile(step, fullgraph=True, backend='aot_eager')(c)
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
