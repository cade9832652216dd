"""A step that cannot run as a whole changes nothing: sizes are checked before the first launch."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LONG = (1 << 20) + 1


def lists(dev, shapes, dtypes):
    p = [torch.full(s, 0.5, device=dev) for s in shapes]
    return p, [torch.ones(s, device=dev, dtype=t) for s, t in zip(shapes, dtypes)], [torch.full(s, 0.25, device=dev) for s in shapes]


@pytest.mark.parametrize('shapes,dtypes', [
    ([(4, 6), (70, 80), (1, LONG)], [torch.float32, torch.float32, torch.float16]),          # a launch for each gradient type
    ([(4, 6)] * 32 + [(LONG, 2)], [torch.bfloat16] * 33),                                      # more than a launch names
    ([(2, LONG)], [torch.float32])], ids=['types', 'many', 'one'])
def test_a_side_past_the_limit_is_refused_first(pkg, dev, shapes, dtypes):
    from faster_yoco_amd import muon
    p, g, m = lists(dev, shapes, dtypes)
    copies = [t.bfloat16() for t in p]
    for precise in (False, True):
        with pytest.raises(RuntimeError, match=r'sides of 1 to 1048576'):
            muon.step_(p, g, m, copies, lr=0.1, precise=precise)
    torch.cuda.synchronize()
    assert all((t == 0.5).all() for t in p + copies) and all((t == 0.25).all() for t in m)


def test_the_longest_side_runs(pkg, dev):
    from faster_yoco_amd import muon
    p, g, m = lists(dev, [(LONG - 1, 1), (2, LONG - 1)], [torch.float32] * 2)
    muon.step_(p, g, m, lr=0.1)
    assert all(t.isfinite().all() and (t != 0.5).all() for t in p)
    with pytest.raises(RuntimeError, match='1048576'):
        muon.orthogonalize(torch.ones(1, LONG, device=dev))


def test_an_optimizer_of_such_a_row_is_refused_when_it_is_made(pkg, dev):
    from faster_yoco_amd import muon, shard
    sh = shard.FlatShard([(4, 6), (LONG, 2), (9,)], dev)
    with pytest.raises(RuntimeError, match=r'row 1 .*1048576'):
        muon.MuonShardOptimizer(sh)
    muon.MuonShardOptimizer(sh, [0]).step()                       # Adam takes the long one
