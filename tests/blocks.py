"""Plain 64-bit forms of the 8-bit formats, the norms and the products, on the CPU, and the error bounds the tests of the
kernels use.  Independent of the package."""
import torch

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
U = 2.0 ** -24                                        # half an ulp of fp32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # rounding, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # subnormal spacing
LARGEST = {t: torch.finfo(t).max for t in HALF}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]

# every e4m3 value by its code, and the finite magnitudes with the codes whose last bit is even marked
_CODES = torch.arange(256, dtype=torch.uint8).view(F8).double()
_MAGNITUDES = _CODES[:127]                            # codes 0x00 .. 0x7e, ascending


def up(n, m):
    return -(-n // m) * m


def e4m3_codes(v):
    """Codes of float64 values |v| <= 448, nearest, ties to the even code; NaN -> 0x7f."""
    a = v.abs().nan_to_num(0.0)
    hi = torch.searchsorted(_MAGNITUDES, a.contiguous()).clamp(max=126)        # first magnitude >= a
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - _MAGNITUDES[lo], _MAGNITUDES[hi] - a
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = code + 128 * torch.signbit(v)
    return torch.where(v.isnan(), torch.full_like(code, 127), code).to(torch.uint8)


def exponents(amax):
    """The least integer e >= -127 with amax <= 448 * 2^e, by trying each."""
    e = torch.full(amax.shape, -127.0, dtype=torch.float64)
    for k in range(-127, 121):
        e = torch.where(amax > 448 * 2.0 ** e, torch.full_like(e, k + 1.0), e)
    return e


def _codes(v, e):
    """Codes and e for v [..., 128-wide last dimension] with one e per [...]."""
    bad = ~v.isfinite()
    return e4m3_codes(torch.where(bad, torch.full_like(v, float('nan')), v) * 2.0 ** -e[..., None])


def pack(x):
    """(codes [rows, wide], scale bytes [rows, pitch]) of x [rows, dim]."""
    rows, dim = x.shape
    v = torch.zeros(rows, up(dim, 128), dtype=torch.float64)
    v[:, :dim] = x.double()
    v = v.view(rows, -1, 128)
    e = exponents(torch.where(v.isfinite(), v.abs(), torch.zeros_like(v)).amax(2))
    s = torch.full((rows, up(dim, 512) // 128), 127, dtype=torch.uint8)
    s[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return _codes(v, e).view(rows, -1), s


def pack_weight(w):
    N, K = w.shape
    n, k = up(N, 128), up(K, 128)
    v = torch.zeros(n, k, dtype=torch.float64)
    v[:N, :K] = w.double()
    t = v.view(n // 128, 128, k // 128, 128)
    e = exponents(torch.where(t.isfinite(), t.abs(), torch.zeros_like(t)).amax((1, 3)))
    q = _codes(t, e[:, None, :].expand(-1, 128, -1)).view(n, k)

    def bytes_(e, pitch):
        s = torch.full((e.shape[0], pitch), 127, dtype=torch.uint8)
        s[:, :e.shape[1]] = (e + 127).to(torch.uint8)
        return s
    return q[:N], bytes_(e, up(K, 512) // 128), q.t()[:K].contiguous(), bytes_(e.t(), up(N, 512) // 128)


def values(q, s, dim):
    """What codes and scale bytes stand for, float64 [rows, dim]."""
    v = _CODES[q.long()].view(q.shape[0], -1, 128)
    return (v * 2.0 ** (s.double()[:, :v.shape[1], None] - 127)).view(q.shape[0], -1)[:, :dim]


def weight_values(q, s, shape):
    N, K = shape
    e = s.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :q.shape[1]] - 127
    return (_CODES[q.long()] * 2.0 ** e)[:, :K]


def codes(t):
    return t.view(torch.uint8).cpu()


def same_codes(got, want):
    """Equal bytes, either NaN code for a NaN, either sign of zero for a zero."""
    g, w = _CODES[codes(got).long()], _CODES[want.long()]
    return bool(((g == w) | (g.isnan() & w.isnan())).all())


def rounded(ref, dtype):
    """How far rounding to dtype may take each value."""
    return HALF[dtype] * ref.abs() + TINY[dtype]


def norm(x, w, b, eps, center):
    x = x.double()
    mean = x.mean(1) if center else torch.zeros(x.shape[0], dtype=torch.float64)
    c = x - mean[:, None]
    rstd = 1 / torch.sqrt((c * c).mean(1) + eps)
    y = c * rstd[:, None]
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd


def norm_backward(dy, x, mean, rstd, w, center):
    dy, r = dy.double(), rstd.double()[:, None]
    xh = (x.double() - (mean.double()[:, None] if center else 0)) * r
    g = dy * w.double() if w is not None else dy
    c1 = g.mean(1, keepdim=True) if center else torch.zeros_like(r)
    return r * (g - c1 - xh * (g * xh).mean(1, keepdim=True)), (dy * xh).sum(0), dy.sum(0), xh, g
