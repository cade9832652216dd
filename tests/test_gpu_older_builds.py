"""The operators of a build without the residual stream's addition run, and the addition says that it is missing."""
import pytest

import older_builds

pytestmark = pytest.mark.gpu

CODE = '''
import torch
from faster_yoco_amd import norm
x = torch.ones(4, 128, device='cuda', dtype=torch.bfloat16)
st = torch.ones(4, device='cuda')
y, rstd = norm.rms_norm(x)
assert y.shape == x.shape and rstd.shape == (4,) and norm.rms_norm_backward(x, x, st)[0].shape == x.shape
for call in (lambda: norm.add_rms_norm(x, x), lambda: norm.add_rms_norm_backward(x, x, x, st)):
    try:
        call()
        raise SystemExit('no refusal')
    except RuntimeError as e:
        assert 'lacks' in str(e), e
print('refused')
'''


def test_the_addition_is_refused_alone(pkg, dev, tmp_path):
    from faster_yoco_amd import _lib
    res = older_builds.run(tmp_path, [n for n in _lib.SIGNATURES if 'z1_add_norm' not in n], CODE)
    assert res.returncode == 0 and res.stdout.split() == ['refused'], (res.stdout, res.stderr)
