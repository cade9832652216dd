"""Timed, checkable cases of the residual stream's norms and of the matrix update: the addition and norm in one pass with
its gradient, the orthogonalised update of a matrix, and the whole step of matrices under it.

``listed()`` are fixed cases, ``draw(rng)`` gives others of the same ranges.  ``prepare`` makes a case's inputs on the
GPU, ``run`` computes it: in elementary torch operations in 32 bits where ``own`` is false, through the package's
operators where it is true.  ``exact`` computes the same results from their definitions in 64 bits, and ``work`` is what
a pass cannot do without.

add norm    h = x + residual, rounded to their type; y = the layer norm (center) or RMS norm of h, in h's type or as
            8-bit rows; the 8-bit rows of h where checkpoint.
gradient    dx = the norm's gradient at h for dy, plus dh; it is the gradient of both x and residual.
orthogonal  X_0 = x / max(|x|_F, 1e-7), X_{k+1} = a X + b (X X^T) X + c (X X^T)^2 X, five times.
step        momentum = mu momentum + (1 - mu) g; u = mu momentum + (1 - mu) g; p = p (1 - lr wd) - lr 0.2
            sqrt(max(m, n)) orthogonal(u); the BF16 copy of p.

8-bit rows are held in blocks of 128 columns: e4m3 values, and for each block a power of two, the least 2^e with
max |x| <= 448 * 2^e.  A row's values are padded with zeros to whole blocks and its scales with ones to a multiple of four.
"""
import math

import torch

own = False

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 128
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BYTES = {'bf16': 2, 'fp16': 2, 'fp32': 4}

DIM, HIDDEN = 3072, 8192          # YOCO-3B's width and feed-forward width (faster_yoco_amd.configs)
EPS = 1e-5
STEPS, COEFFICIENTS = 5, (3.4445, -4.7750, 2.0315)
MU, DECAY = 0.95, 0.1


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # decoding one token: latency only; the stream is added and the next projection's 8-bit operand made
        {'name': 'add norm, one token', 'op': 'add_norm', 'rows': 1, 'dim': DIM, 'center': False, 'dtype': 'bf16',
         'y8': True, 'checkpoint': False},
        # an fp32 model of odd width
        {'name': 'add norm, odd', 'op': 'add_norm', 'rows': 777, 'dim': 1537, 'center': True, 'dtype': 'fp32',
         'y8': False, 'checkpoint': False},
        # four sequences of 2048 tokens in training: the stream, the projection's operand and the checkpoint in one pass
        {'name': 'add norm, checkpointed', 'op': 'add_norm', 'rows': 8192, 'dim': DIM, 'center': False, 'dtype': 'bf16',
         'y8': True, 'checkpoint': True},
        # one GPU's micro-batch of the pretraining recipe (2048 tokens), the stream kept in its own type
        {'name': 'add norm gradient', 'op': 'add_norm_grad', 'rows': 2048, 'dim': DIM, 'center': True, 'dtype': 'bf16',
         'checkpoint': False},
        # rows that start at any element
        {'name': 'add norm gradient, odd', 'op': 'add_norm_grad', 'rows': 4099, 'dim': 1001, 'center': False,
         'dtype': 'fp16', 'checkpoint': False},
        # eight sequences, the stream read back from its checkpoint
        {'name': 'add norm gradient, checkp.', 'op': 'add_norm_grad', 'rows': 16384, 'dim': DIM, 'center': False,
         'dtype': 'bf16', 'checkpoint': True},
        # a small model's matrix: latency only
        {'name': 'orthogonal, small', 'op': 'orthogonal', 'batch': 1, 'm': 64, 'n': 256, 'dtype': 'fp32', 'out': 'bf16'},
        # three odd matrices at once, in a type that holds more digits
        {'name': 'orthogonal, odd', 'op': 'orthogonal', 'batch': 3, 'm': 777, 'n': 401, 'dtype': 'fp16', 'out': 'fp16'},
        # the attention projections of one block
        {'name': 'orthogonal, projections', 'op': 'orthogonal', 'batch': 4, 'm': DIM, 'n': DIM, 'dtype': 'bf16',
         'out': 'bf16'},
        # one feed-forward weight
        {'name': 'orthogonal, feed-forward', 'op': 'orthogonal', 'batch': 1, 'm': HIDDEN, 'n': DIM, 'dtype': 'bf16',
         'out': 'bf16'},
        # the matrices of a small shard, fp32 gradients
        {'name': 'step, small shard', 'op': 'step', 'blocks': 1, 'dim': 1024, 'hidden': 4096, 'dtype': 'fp32', 'lr': 1e-4},
        # the matrices of two blocks of a pretraining shard
        {'name': 'step, two blocks', 'op': 'step', 'blocks': 2, 'dim': DIM, 'hidden': HIDDEN, 'dtype': 'bf16', 'lr': 1e-4},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('add_norm', 'add_norm_grad', 'orthogonal', 'step'))
    if op in ('add_norm', 'add_norm_grad'):
        rows, dim = _log(rng, 1, 16384), _log(rng, 64, HIDDEN)
        if rng.random() < 0.5:                # model widths are mostly whole blocks
            dim = max(1, dim // BLOCK) * BLOCK
        while rows * dim > 16384 * DIM:
            rows = max(1, rows // 2)
        case = {'op': op, 'rows': rows, 'dim': dim, 'center': rng.random() < 0.5,
                'dtype': rng.choice(('bf16', 'bf16', 'fp16', 'fp32'))}
        if op == 'add_norm':
            case['y8'] = rng.random() < 0.5
        return {**case, 'checkpoint': rng.random() < 0.5}
    m, n = _log(rng, 16, HIDDEN), _log(rng, 16, HIDDEN)
    if rng.random() < 0.5:                    # model widths are mostly whole blocks
        m, n = max(1, m // 64) * 64, max(1, n // 64) * 64
    if op == 'step':
        dim, hidden = min(m, n, DIM), max(m, n)
        return {'op': op, 'blocks': rng.choice((1, 1, 2)), 'dim': dim, 'hidden': hidden,
                'dtype': rng.choice(('bf16', 'fp32')), 'lr': _log(rng, 20, 120) * 1e-6}
    while min(m, n) > DIM:
        m, n = m // 2, n
    batch = _log(rng, 1, 8)
    while batch > 1 and batch * _products(m, n) > _products(DIM, HIDDEN):
        batch //= 2
    dtype = rng.choice(('bf16', 'bf16', 'fp16', 'fp32'))
    return {'op': op, 'batch': batch, 'm': m, 'n': n, 'dtype': dtype, 'out': 'fp16' if dtype == 'fp16' else 'bf16'}


def _shapes(case):
    """The matrices of `blocks` blocks: an attention projection and the feed-forward weights, one of them to each side."""
    d, h = case['dim'], case['hidden']
    return [(d, d), (h, d)] * case['blocks'] if case['blocks'] > 1 else [(d, d), (h, d), (d, h)]


def _products(m, n):
    """Multiplications and additions of the five iterations; the two symmetric products by one of their halves."""
    m, n = min(m, n), max(m, n)
    return STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    op, b = case['op'], BYTES[case['dtype']]
    if op == 'add_norm':
        n, T = case['rows'] * case['dim'], case['rows']
        return {'bytes': n * (3 * b + (1 if case['y8'] else b) + (1 if case['checkpoint'] else 0)) + 8 * T, 'flops': 9 * n}
    if op == 'add_norm_grad':
        n, T = case['rows'] * case['dim'], case['rows']
        return {'bytes': n * (3 * b + (1 if case['checkpoint'] else b)) + 8 * T, 'flops': 13 * n}
    if op == 'orthogonal':
        m, n = case['m'], case['n']
        return {'bytes': case['batch'] * m * n * (b + BYTES[case['out']]), 'flops': case['batch'] * _products(m, n)}
    shapes = _shapes(case)
    # the gradient is read, momentum and master read and written, the BF16 copy written
    return {'bytes': sum(m * n for m, n in shapes) * (b + 8 + 8 + 2), 'flops': sum(_products(m, n) for m, n in shapes)}


# ----------------------------------------------------------------------------------------------------------- inputs
def _stream(rows, dim, gen, dtype, size=1.0):
    """A residual stream: channels of different sizes, a few much larger than the rest, a small common offset."""
    dev = gen.device
    sizes = torch.exp(0.5 * torch.randn(dim, device=dev, generator=gen))
    sizes[torch.randint(0, dim, (max(1, dim // 256),), device=dev, generator=gen)] = 12.0
    return ((torch.randn(rows, dim, device=dev, generator=gen) * sizes + 0.1) * size).to(dtype)


def _gradient(rows, dim, gen, dtype):
    """Gradients of a mean loss: small, and tokens of different weight."""
    g = torch.randn(rows, dim, device=gen.device, generator=gen)
    return (g * 1e-3 * torch.exp(0.7 * torch.randn(rows, 1, device=gen.device, generator=gen))).to(dtype)


def _matrix(batch, m, n, gen, dtype):
    """A weight's gradient: a few strong directions of falling size over noise (fp16 ones under a loss scale)."""
    dev, r = gen.device, min(m, n, 32)
    size = 1.0 / torch.arange(1, r + 1, device=dev)
    u = torch.randn(batch, m, r, device=dev, generator=gen) * size
    v = torch.randn(batch, r, n, device=dev, generator=gen)
    return ((u @ v + 0.5 * torch.randn(batch, m, n, device=dev, generator=gen)) * (0.1 if dtype == torch.float16 else 1e-4)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed))
    dev, dtype, op = gen.device, DTYPES[case['dtype']], case['op']
    s = dict(case)
    if op in ('add_norm', 'add_norm_grad'):
        rows, dim = case['rows'], case['dim']
        s['w'] = (1 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dtype)
        s['b'] = (0.1 * torch.randn(dim, device=dev, generator=gen)).to(dtype) if case['center'] else None
        if op == 'add_norm':
            s['x'] = _stream(rows, dim, gen, dtype, 0.3)
            s['r'] = _stream(rows, dim, gen, dtype)
            return s
        h = _stream(rows, dim, gen, dtype)
        s['dy'], s['dh'] = _gradient(rows, dim, gen, dtype), _gradient(rows, dim, gen, dtype)
        v = h.float()
        s['mean'] = v.mean(1) if case['center'] else None
        if case['center']:
            v = v - s['mean'][:, None]
        s['rstd'] = torch.rsqrt(v.square().mean(1) + EPS)
        if case['checkpoint']:
            s['q'], s['s'] = _pack(h)
        else:
            s['h'] = h
        return s
    if op == 'orthogonal':
        s['x'] = _matrix(case['batch'], case['m'], case['n'], gen, dtype)
        return s
    for name in ('g', 'm', 'p', 'p16'):
        s[name] = []
    for m, n in _shapes(case):
        old = _matrix(1, m, n, gen, torch.float32)[0]
        s['m'].append(old)
        s['g'].append((old + _matrix(1, m, n, gen, torch.float32)[0]).to(dtype))
        s['p'].append(0.02 * torch.randn(m, n, device=dev, generator=gen))
        s['p16'].append(s['p'][-1].bfloat16())
    return s


# ------------------------------------------------------------------------------------------------------- plain form
def _ceil(n, m):
    return -(-n // m) * m


def _exponents(amax):
    """The least e >= -127 with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, ex = torch.frexp(amax)
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp_(min=-127)


def _pack(x):
    rows, dim = x.shape
    wide = _ceil(dim, BLOCK)
    v = torch.zeros(rows, wide, device=x.device)
    v[:, :dim] = x.float()
    v = v.view(rows, wide // BLOCK, BLOCK)
    e = _exponents(v.abs().amax(2))
    q = (v * torch.exp2(-e.float())[:, :, None]).to(F8).view(rows, wide)
    s = torch.full((rows, _ceil(wide // BLOCK, 4)), 127, dtype=torch.uint8, device=x.device)
    s[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return q, s.view(E8)


def _unpack(q, s, dim):
    rows, wide = q.shape
    scale = torch.exp2(s.view(torch.uint8).float() - 127)
    v = q.float().view(rows, wide // BLOCK, BLOCK) * scale[:, :wide // BLOCK, None]
    return v.view(rows, wide)[:, :dim]


def _orthogonal(x):
    """The iterates of matrices [..., m, n] in 32 bits, with the products over their shorter side."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.float().mT.contiguous() if tall else x.float()
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x / norm.clamp(min=1e-7).float()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = x @ x.mT.contiguous()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.mT if tall else x


def _plain(s):
    op, dtype = s['op'], DTYPES[s['dtype']]
    if op == 'add_norm':
        h = (s['x'].float() + s['r'].float()).to(dtype)
        x = h.float()
        mean = x.mean(1) if s['center'] else None
        c = x - mean[:, None] if s['center'] else x
        rstd = torch.rsqrt(c.square().mean(1) + EPS)
        y = c * rstd[:, None] * s['w'].float()
        if s['center']:
            y = y + s['b'].float()
        out = [h] + (list(_pack(y)) if s['y8'] else [y.to(dtype)])
        out += [mean, rstd] if s['center'] else [rstd]
        return out + (list(_pack(h)) if s['checkpoint'] else [])
    if op == 'add_norm_grad':
        x = _unpack(s['q'], s['s'], s['dim']) if s['checkpoint'] else s['h'].float()
        dy, r = s['dy'].float(), s['rstd'][:, None]
        xh = (x - s['mean'][:, None]) * r if s['center'] else x * r
        g = dy * s['w'].float()
        t = g - xh * (g * xh).mean(1, keepdim=True)
        if s['center']:
            t = t - g.mean(1, keepdim=True)
        out = [(t * r + s['dh'].float()).to(dtype), (dy * xh).sum(0).to(dtype)]
        return out + ([dy.sum(0).to(dtype)] if s['center'] else [])
    if op == 'orthogonal':
        return _orthogonal(s['x']).to(DTYPES[s['out']])
    for p, g, m, p16 in zip(s['p'], s['g'], s['m'], s['p16']):
        g = g.float()
        m.mul_(MU).add_(g, alpha=1 - MU)
        u = MU * m + (1 - MU) * g
        p.mul_(1 - s['lr'] * DECAY).sub_(_orthogonal(u), alpha=s['lr'] * 0.2 * math.sqrt(max(p.shape)))
        p16.copy_(p)
    return [s['p'], s['m'], s['p16']]


# --------------------------------------------------------------------------------------------- the package's operators
def _own(s):
    from faster_yoco_amd import act8, muon, norm
    op = s['op']
    if op == 'add_norm':
        if s['center']:
            out = norm.add_layer_norm(s['x'], s['r'], s['w'], s['b'], EPS, y8=s['y8'], checkpoint=s['checkpoint'])
        else:
            out = norm.add_rms_norm(s['x'], s['r'], s['w'], EPS, y8=s['y8'], checkpoint=s['checkpoint'])
        flat = []
        for t in out:
            flat += [t.q, t.s] if isinstance(t, act8.Act8) else [t]
        return flat
    if op == 'add_norm_grad':
        h = act8.Act8(s['q'], s['s'], s['dim']) if s['checkpoint'] else s['h']
        if s['center']:
            return list(norm.add_layer_norm_backward(s['dy'], s['dh'], h, s['mean'], s['rstd'], s['w'], bias=True))
        return list(norm.add_rms_norm_backward(s['dy'], s['dh'], h, s['rstd'], s['w']))
    if op == 'orthogonal':
        return muon.orthogonalize(s['x'], steps=STEPS, coefficients=COEFFICIENTS, dtype=DTYPES[s['out']])
    muon.step_(s['p'], s['g'], s['m'], s['p16'], lr=s['lr'], momentum=MU, nesterov=True, weight_decay=DECAY, adjust='rms',
               steps=STEPS, coefficients=COEFFICIENTS)
    return [s['p'], s['m'], s['p16']]


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------------------- 64-bit definition
def _grid(v):
    """v (64 bits, |v| <= 448) rounded to e4m3's values: three mantissa bits, exponents from -6, ties to even."""
    a = v.abs().clamp(min=2.0 ** -20)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_rows(x):
    """(values before scaling back, scales with their padding) of rows in blocks."""
    v = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
    amax = v.abs().amax(2)
    e = torch.ceil(torch.log2(amax / 448))
    e = torch.where(amax > torch.exp2(e) * 448, e + 1, e)
    e = torch.where(amax <= torch.exp2(e - 1) * 448, e - 1, e)
    s = torch.exp2(torch.where(amax > 0, e, torch.full_like(e, -127.0)).clamp(min=-127))
    return _grid(v / s[..., None]).flatten(1), torch.nn.functional.pad(s, (0, -s.shape[1] % 4), value=1.0)


def _exact_orthogonal(x):
    """From the definition, on whichever side the matrix is longer."""
    x = x.double()
    x = x / torch.clamp(torch.sqrt((x * x).sum((-2, -1), keepdim=True)), min=1e-7)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        if x.shape[-2] > x.shape[-1]:
            G = x.mT.contiguous() @ x
            x = a * x + x @ (b * G + c * (G @ G))
        else:
            G = x @ x.mT.contiguous()
            x = a * x + (b * G + c * (G @ G)) @ x
    return x


def exact(case, seed):
    st = prepare(case, seed)
    op = case['op']
    if op == 'orthogonal':
        return torch.stack([_exact_orthogonal(x) for x in st['x']])
    if op == 'step':
        ps, ms = [], []
        for p, g, m in zip(st['p'], st['g'], st['m']):
            m = MU * m.double() + (1 - MU) * g.double()
            u = MU * m + (1 - MU) * g.double()
            lr = case['lr']
            ps.append(p.double() - lr * DECAY * p.double() - lr * 0.2 * max(p.shape) ** 0.5 * _exact_orthogonal(u))
            ms.append(m)
        return [ps, ms, ps]
    n, w = case['dim'], st['w'].double()
    if op == 'add_norm':
        total = st['x'].double() + st['r'].double()
        h = total.to(DTYPES[case['dtype']]).double()
        mean = h.sum(1) / n
        c = h - mean[:, None] if case['center'] else h
        rstd = 1 / torch.sqrt((c * c).sum(1) / n + EPS)
        y = c * rstd[:, None] * w + (st['b'].double() if case['center'] else 0)
        out = [total] + (list(_exact_rows(y)) if case['y8'] else [y])
        out += [mean, rstd] if case['center'] else [rstd]
        return out + (list(_exact_rows(h)) if case['checkpoint'] else [])
    if case['checkpoint']:
        k = st['q'].shape[1] // BLOCK
        e = st['s'].view(torch.uint8)[:, :k].double() - 127
        h = (st['q'].double().unflatten(1, (k, BLOCK)) * torch.exp2(e)[..., None]).flatten(1)[:, :n]
    else:
        h = st['h'].double()
    dy, r = st['dy'].double(), st['rstd'].double()[:, None]
    xh = (h - (st['mean'].double()[:, None] if case['center'] else 0)) * r
    g = dy * w
    dx = r * (g - xh * ((g * xh).sum(1, keepdim=True) / n) - (g.sum(1, keepdim=True) / n if case['center'] else 0))
    return [dx + st['dh'].double(), (dy * xh).sum(0)] + ([dy.sum(0)] if case['center'] else [])
