"""Orthogonalised matrices on the GPU within the distances that are documented, whatever the spectrum: limits of their own against
the 64-bit form, which do not grow with what the stored operands leave.

Both limits are relative, in the 2-norm of all elements.

Single operands: 2e-3, about what a bf16 result's own rounding leaves (half a step of 2^-8 at most, 2^-8 / sqrt(3) at random over
values spread within their powers of two: 1.7e-3).  In 64-bit arithmetic with the operands rounded as they are stored, 18,000
spectra of one to three levels (65 x 65 to 352 x 704) leave 1.94e-3 at most; another draw of the same roundings differs by the
square root of its number of elements, 1 / 65: 1.97e-3.

Pairs: X's elements are off by up to 2^-22 of themselves, 2^-22 / sqrt(3) at random; of X_0, whose norm is 1, that goes into all
directions, and those of no size grow 3.4445^5 = 485 times: 6.7e-5, the later steps' roundings another 4 % of it (their squares
add, each 3.4445 times less).  A result of rank one has a norm of 0.68 at least: 1.0e-4.  Sums of up to 3 K / 16 additions in
fp32 add sqrt(3 K / 16) 2^-24 of what they sum, of up to 3.4 times X, in B X, where K is the shorter side, up to 520 here: 2.0e-6
a step, into all directions as well, 141 times by the end: 2.8e-4 were they all one way in every element, but their sizes are
the running sums', a third of that at random.  2e-4 in all."""
import pytest
import torch

import matrices as ref

pytestmark = pytest.mark.gpu

SINGLE, PAIRS = 2e-3, 2e-4
# thin ones, both sides of every border between the forms: 64 and 65 rows, a workgroup's matrices and larger ones
SHAPES = [(2, 2), (3, 5), (2, 9), (3, 2000), (2000, 3), (5, 400), (8, 4096), (16, 2048), (33, 96), (48, 1200), (64, 65), (65, 65), (96, 576), (576, 96), (352, 352), (64, 256),
          (256, 64), (64, 4096), (65, 66), (90, 130), (96, 300), (65, 4000), (128, 128), (128, 256), (512, 128), (150, 2000),
          (300, 520), (520, 300)]


def spectra(m, n, seed):
    g = torch.Generator().manual_seed(m * 5003 + n * 7 + seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    for rank in (1, 4):
        low = r(m, rank) @ r(rank, n)
        yield f'rank {rank}', low
        yield f'rank {rank} over noise', low + 1e-3 * r(m, n)
    for kind in ('noise', 'strong', 'falling', 'flat'):
        yield kind, ref.spectrum(m, n, kind, g)
    k = min(m, n)
    for j in {k, (k + 1) // 2, min(k, 28), min(k, 48), min(k, 60)}:            # equal singular values, and the rest none
        q = [torch.linalg.qr(r(s, j))[0] for s in (m, n)]
        yield f'{j} equal', q[0] @ q[1].t()


@pytest.mark.parametrize('m,n', SHAPES)
def test_documented_distances(pkg, dev, m, n):
    from faster_yoco_amd import muon
    for name, x in (s for seed in range(2) for s in spectra(m, n, seed)):
        x = x.float()
        want = ref.exact(x)
        for precise, limit in ((False, SINGLE), (True, PAIRS)):
            got = muon.orthogonalize(x.to(dev), dtype=torch.float32, precise=precise).cpu().double()
            off = float((got - want).norm() / want.norm())
            assert off <= limit, (name, precise, off)


@pytest.mark.parametrize('m,n', [(64, 256), (300, 520)])
def test_documented_distances_in_batches_and_steps(pkg, dev, m, n):
    """A batch whose tiles are larger, and the step's list: the same limits."""
    from faster_yoco_amd import muon
    x = [t.float() for _, t in spectra(m, n, 5)] * 5
    want = [ref.exact(t) for t in x]
    got = muon.orthogonalize(torch.stack(x).to(dev), dtype=torch.float32, precise=False)
    p = [torch.zeros(m, n, device=dev) for _ in x]
    muon.step_(p, [t.to(dev) for t in x], [torch.zeros_like(t) for t in p], lr=1.0, adjust=1.0, weight_decay=0.0, momentum=0.0,
               precise=False)
    for q, t, w in zip(got, p, want):
        assert float((q.cpu().double() - w).norm() / w.norm()) <= SINGLE
        assert float((t.cpu().double() + w).norm() / w.norm()) <= SINGLE


def test_other_coefficients(pkg, dev):
    """Few steps, many, of small and large growth: twelve of (1.5, -0.5, 0) grow small directions 130 times."""
    from faster_yoco_amd import muon
    for m, n in ((65, 4000), (300, 520)):
        for name, x in spectra(m, n, 2):
            for steps, c in ((1, ref.COEFFICIENTS), (3, ref.COEFFICIENTS), (12, (1.5, -0.5, 0.0))):
                want = ref.exact(x.float(), steps, c)
                got = muon.orthogonalize(x.float().to(dev), steps, c, precise=False).cpu().double()
                assert float((got - want).norm() / want.norm()) <= SINGLE, (name, steps)


def test_matrices_of_few_rows_beside_large_ones(pkg, dev):
    """One launch's tiles hold matrices with pairs and without (64-bit forms on the GPU: the large ones take seconds less)."""
    from faster_yoco_amd import muon
    shapes = [(40, 2000), (3, 5000), (9000, 64), (64, 256), (65, 600)] + [(2304, 2304)] * 3
    u = [next(x for name, x in spectra(m, n, i) if name == 'rank 1 over noise').float().to(dev) for i, (m, n) in enumerate(shapes)]
    p = [torch.zeros_like(t) for t in u]
    muon.step_(p, u, [torch.zeros_like(t) for t in u], lr=1.0, adjust=1.0, weight_decay=0.0, momentum=0.0, precise=False)
    for t, q in zip(u, p):
        want = ref.exact(t)
        off = float((q.double() + want).norm() / want.norm())
        assert off <= (PAIRS if min(t.shape) <= 64 else SINGLE), (t.shape, off)
