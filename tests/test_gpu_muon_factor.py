"""The gradient factor of a step lies apart from what the step writes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_factor_in_what_is_written_is_refused(pkg, dev):
    from faster_yoco_amd import muon
    flat = torch.ones(200, device=dev)
    p, m, c = flat[:24].view(4, 6), flat[48:72].view(4, 6), torch.ones(4, 6, device=dev, dtype=torch.bfloat16)
    g = torch.ones(4, 6, device=dev)
    for at in (0, 23, 48, 71):
        with pytest.raises(RuntimeError, match='factor overlaps what is written'):
            muon.step_([p], [g], [m], [c], lr=0.1, factor=flat[at:at + 1])
    with pytest.raises(RuntimeError, match='factor overlaps what is written'):
        muon.step_([p], [g], [m], [c], lr=0.1, factor=c.view(-1)[:2].view(torch.float32))
    assert (flat == 1).all() and (c == 1).all()
    for factor in (flat[24:25], flat[47:48], flat[72], g.view(-1)[:1]):       # next to it, without dimensions, a gradient's
        muon.step_([p], [g], [m], [c], lr=0.1, factor=factor)
    assert (flat[:24] < 1).all() and (flat[24:48] == 1).all() and (flat[72:] == 1).all()
