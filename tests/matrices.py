"""Plain 64-bit forms of the matrices' update, and the error bounds the tests of its kernels use.  Independent of the package.

Two bounds.  ``one_step_bound`` is a componentwise bound of one step's roundings, term by term.  Over several steps such a
bound grows by the largest slope of the polynomial each time and says little; there the tests compare with ``stored``, which
takes the same steps in 64 bits with every operand rounded as the kernels store it (sums exact, or fp32's).  The kernels' own
roundings are another draw of the same ones (their fp32 sums differ in the last bits, which moves some of the roundings that
follow), so their distance from the exact result is that of ``stored`` up to the draw: the tests allow four times it."""
import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
KX, KA, KB = 4096.0, 2048.0, 1024.0                   # the stored values' scales
U16, U32 = 2.0 ** -11, 2.0 ** -24                     # half an ulp, relative
TINY16 = 2.0 ** -25                                   # half of fp16's subnormal spacing
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def triples(coefficients, steps):
    return [coefficients] * steps if not hasattr(coefficients[0], '__len__') else list(coefficients)


def start(x, eps=1e-7):
    x = x.double()
    return x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)


def exact(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = start(x, eps)
    for a, b, c in triples(coefficients, steps):
        A = x @ x.mT.contiguous() if x.shape[-2] <= x.shape[-1] else x.mT.contiguous() @ x
        B = b * A + c * (A @ A)
        x = a * x + (B @ x if x.shape[-2] <= x.shape[-1] else x @ B)
    return x


def _h(v, scale):
    return (v * scale).half().to(v.dtype) / scale


def _pair(v, scale):
    hi = _h(v, scale)
    return hi, _h(v - hi, scale)


def _product(p, q, pairs):
    """p @ q of pairs (hi, lo) or of first halves alone.  In fp32 the sums are added as the kernels add them, 16 terms at a time
    and hi hi before hi lo before lo hi: N additions one after another, each off by up to U32 of the sum so far, are less exact
    than a library's blocked ones."""
    (ph, pl), (qh, ql) = p, q
    if not pairs:
        return ph @ qh
    acc = torch.zeros(ph.shape[0], qh.shape[1], dtype=ph.dtype)
    for a, b in ((ph, qh), (ph, ql), (pl, qh)):
        for k in range(0, a.shape[1], 16):
            acc = acc + (a[:, k:k + 16].double() @ b[k:k + 16].double()).float()
    return acc


def stored(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7, precise=False):
    """One matrix's steps with operands rounded as they are stored; precise: as pairs, and products and sums in fp32."""
    x = start(x, eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x.float() if precise else x
    for a, b, c in triples(coefficients, steps):
        hi, lo = _pair(x, KX)
        x = hi + lo
        A = _product((hi, lo), (hi.t(), lo.t()), precise)
        d = A.diagonal().clone()
        A = A - torch.diag(d)
        Ah, Al = _pair(A, KA)
        A = Ah + Al if precise else Ah
        S = _product((Ah, Al), (Ah, Al), precise)
        e = a + b * d + c * d * d + c * S.diagonal()
        B = c * S + (b + c * (d[:, None] + d)) * A
        B = B - torch.diag(B.diagonal())
        x = e[:, None] * x + _product(_pair(B, KB), (hi, lo), precise)
    x = x.t() if tall else x
    return x.double()


def one_step_bound(x, coefficients=COEFFICIENTS, eps=1e-7):
    """|kernel - exact| of one step on fp16 operands, element by element, before the result's own rounding.

    X's products take its first half, off by U16 |X| (and TINY16 / KX); A is then off by 2 U16 |X||X|^T and by its own
    rounding where it is stored; B by what that makes of b A + c A^2 and by its own rounding; sums of K terms by K U32 of the
    terms' sizes (several times over for the few operations around them); the linear term by X's pair, 2^-21."""
    x = start(x, eps)
    tall = x.shape[0] > x.shape[1]
    x = (x.t() if tall else x).abs().contiguous()
    a, b, c = (abs(v) for v in coefficients)
    r, n = x.shape
    dx = U16 * x + TINY16 / KX
    XX = x @ x.t()
    dA = dx @ x.t() + x @ dx.t() + dx @ dx.t() + (n + 8) * U32 * XX
    A, dS = XX, U16 * (XX + dA) + TINY16 / KA          # sizes: |A| <= |X||X|^T
    dA = dA + dS
    AA = A @ A
    dB = b * dA + c * (A @ dA + dA @ A + dA @ dA) + (r + 16) * U32 * (b * A + 3 * c * AA)
    B = b * A + c * AA
    dB = dB + U16 * (B + dB) + TINY16 / KB
    dX = dB @ x + (B + dB) @ dx + (r + 16) * U32 * (a * x + B @ x) + (2.0 ** -21) * (a * x + B @ x) + TINY16 / KX * (a + b + c)
    return dX.t() if tall else dX


def spectrum(m, n, kind, gen):
    """Test matrices: 'noise', 'strong' (a few large directions over small noise), 'falling' (singular values 1, 1/2, 1/3, ...),
    'flat' (nearly orthogonal)."""
    g = torch.randn(m, n, generator=gen, dtype=torch.float64)
    if kind == 'noise':
        return g
    k = min(m, n)
    if kind == 'strong':
        j = min(k, 4)
        return 0.02 * g + torch.randn(m, j, generator=gen, dtype=torch.float64) @ torch.randn(j, n, generator=gen, dtype=torch.float64)
    u, _, v = torch.linalg.svd(g, full_matrices=False)
    s = 1.0 / torch.arange(1, k + 1, dtype=torch.float64) if kind == 'falling' else 1 + 0.1 * torch.rand(k, generator=gen, dtype=torch.float64)
    return (u * s) @ v


def step(p, g, momentum, *, lr, mu, nesterov, weight_decay, rate, factor=1.0, eps=1e-7, steps=5, coefficients=COEFFICIENTS):
    """(p, momentum, the update) of one step in 64 bits."""
    g = g.double() * factor
    momentum = mu * momentum.double() + (1 - mu) * g
    u = mu * momentum + (1 - mu) * g if nesterov else momentum
    q = exact(u, steps, coefficients, eps)
    return p.double() * (1 - lr * weight_decay) - rate * q, momentum, q, u
