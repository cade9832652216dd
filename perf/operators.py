"""Timed, checkable cases of the block-side operators: norms with their gradients, 8-bit activation checkpoints, and the
8-bit matrix products with their gradients.

``listed()`` are fixed cases, ``draw(rng)`` gives others of the same ranges.  ``prepare`` makes a case's inputs on the
GPU, ``run`` computes it: in elementary torch operations in 32 bits where ``own`` is false, through the package's
operators where it is true.  ``exact`` computes the same results from their definitions in 64 bits, and ``work`` is what
a pass cannot do without.

8-bit values are held in blocks of 128 along a row: e4m3 values, and for each block a power of two, the least 2^e with
max |x| <= 448 * 2^e.  A row's values are padded with zeros to whole blocks and its scales with ones to a multiple of
four.  A weight has one scale for each 128 x 128 block, and is kept in both orders.
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


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # decoding one token: latency only; the norm hands the next projection its 8-bit operand
        {'name': 'norm, one token', 'op': 'norm', 'rows': 1, 'dim': DIM, 'center': True, 'dtype': 'bf16', 'y8': True,
         'checkpoint': False},
        # four sequences of 2048 tokens in training: the projection's operand and the checkpoint in the same pass
        {'name': 'norm, checkpointed', 'op': 'norm', 'rows': 8192, 'dim': DIM, 'center': False, 'dtype': 'bf16',
         'y8': True, 'checkpoint': True},
        # one GPU's micro-batch of the pretraining recipe (2048 tokens), the input kept in its own type
        {'name': 'norm gradient', 'op': 'norm_grad', 'rows': 2048, 'dim': DIM, 'center': True, 'dtype': 'bf16',
         'checkpoint': False},
        # an fp32 model of odd width
        {'name': 'norm gradient, odd', 'op': 'norm_grad', 'rows': 777, 'dim': 1537, 'center': True, 'dtype': 'fp32',
         'checkpoint': False},
        # eight sequences, the input read back from its checkpoint
        {'name': 'norm gradient, checkpointed', 'op': 'norm_grad', 'rows': 16384, 'dim': DIM, 'center': False,
         'dtype': 'bf16', 'checkpoint': True},
        # rows that start at any element and end inside a block
        {'name': 'pack, odd', 'op': 'pack', 'rows': 4099, 'dim': 1001, 'dtype': 'fp16'},
        # a feed-forward activation recovered for a backward pass that wants it in its own type
        {'name': 'unpack', 'op': 'unpack', 'rows': 16384, 'dim': HIDDEN, 'dtype': 'bf16'},
        # after an optimizer update: one feed-forward weight, both orders
        {'name': 'pack weight', 'op': 'pack_weight', 'rows': HIDDEN, 'dim': DIM, 'dtype': 'bf16'},
        # decoding one token: the weight is read once
        {'name': 'product, one token', 'op': 'product', 'rows': 1, 'inner': DIM, 'outer': HIDDEN, 'dtype': 'bf16'},
        # a ragged micro-batch through a small odd projection: forward, input gradient and weight gradient
        {'name': 'projection, ragged', 'op': 'projection', 'rows': 333, 'inner': 1000, 'outer': 1501, 'dtype': 'bf16'},
        # the recipe's micro-batch through a feed-forward projection
        {'name': 'projection', 'op': 'projection', 'rows': 2048, 'inner': DIM, 'outer': HIDDEN, 'dtype': 'bf16'},
        # eight sequences at once
        {'name': 'projection, eight sequences', 'op': 'projection', 'rows': 16384, 'inner': DIM, 'outer': HIDDEN,
         'dtype': 'bf16'},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('norm', 'norm_grad', 'pack', 'unpack', 'pack_weight', 'product', 'projection'))
    dtype = rng.choice(('bf16', 'bf16', 'bf16', 'fp16', 'fp32'))
    rows, dim = _log(rng, 1, 16384), _log(rng, 64, HIDDEN)
    if rng.random() < 0.5:                    # model widths are mostly whole blocks
        dim = max(1, dim // BLOCK) * BLOCK
    if op == 'norm':
        y8 = rng.random() < 0.5
        return {'op': op, 'rows': rows, 'dim': dim, 'center': rng.random() < 0.5, 'dtype': dtype, 'y8': y8,
                'checkpoint': rng.random() < 0.5}
    if op == 'norm_grad':
        return {'op': op, 'rows': rows, 'dim': dim, 'center': rng.random() < 0.5, 'dtype': dtype,
                'checkpoint': rng.random() < 0.5}
    if op in ('pack', 'unpack'):
        return {'op': op, 'rows': rows, 'dim': dim, 'dtype': dtype}
    outer = _log(rng, 64, HIDDEN)
    if rng.random() < 0.5:
        outer = max(1, outer // BLOCK) * BLOCK
    if op == 'pack_weight':
        return {'op': op, 'rows': outer, 'dim': dim, 'dtype': dtype}
    if op == 'product':                       # serving: few tokens
        return {'op': op, 'rows': _log(rng, 1, 256), 'inner': dim, 'outer': outer, 'dtype': dtype}
    while rows * dim * outer > 16384 * DIM * HIDDEN:
        rows = max(1, rows // 2)
    return {'op': op, 'rows': rows, 'inner': dim, 'outer': outer, 'dtype': 'bf16'}


def work(case):
    b, op, T = BYTES[case['dtype']], case['op'], case['rows']
    if op in ('product', 'projection'):
        K, N = case['inner'], case['outer']
        forward = T * K * b + N * K + T * N * b
        if op == 'product':
            return {'bytes': forward, 'flops': 2 * T * N * K}
        # the input gradient reads dy and the weight and writes dx; the weight gradient reads the packed input again
        return {'bytes': forward + T * N * b + N * K + T * K * b + T * K + N * K * b, 'flops': 6 * T * N * K}
    n = T * case['dim']
    if op == 'norm':
        out = (1 if case['y8'] else b) + (1 if case['checkpoint'] else 0)
        return {'bytes': n * (b + out) + 8 * T, 'flops': 8 * n}
    if op == 'norm_grad':
        return {'bytes': n * (2 * b + (1 if case['checkpoint'] else b)) + 8 * T, 'flops': 12 * n}
    if op == 'pack_weight':
        return {'bytes': n * (b + 2), 'flops': 2 * n}
    return {'bytes': n * (b + 1), 'flops': 2 * n}


# ----------------------------------------------------------------------------------------------------------- inputs
def _stream(rows, dim, gen, dtype):
    """A residual stream: channels of different sizes, a few much larger than the rest, a small common offset."""
    dev = gen.device
    size = torch.exp(0.5 * torch.randn(dim, device=dev, generator=gen))
    big = torch.randint(0, dim, (max(1, dim // 256),), device=dev, generator=gen)
    size[big] = 12.0
    x = torch.randn(rows, dim, device=dev, generator=gen) * size + 0.1
    return x.to(dtype)


def _gradient(rows, dim, gen, dtype):
    """Gradients of a mean loss: small, and tokens of different weight."""
    g = torch.randn(rows, dim, device=gen.device, generator=gen)
    return (g * 1e-3 * torch.exp(0.7 * torch.randn(rows, 1, device=gen.device, generator=gen))).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed))
    dev, dtype, op, rows = gen.device, DTYPES[case['dtype']], case['op'], case['rows']
    s = dict(case)
    if op in ('norm', 'norm_grad'):
        dim = case['dim']
        x = _stream(rows, dim, gen, dtype)
        s['w'] = (1 + 0.2 * torch.randn(dim, device=dev, generator=gen)).to(dtype)
        s['b'] = (0.1 * torch.randn(dim, device=dev, generator=gen)).to(dtype) if case['center'] else None
        s['x'] = x
        if op == 'norm_grad':
            s['dy'] = _gradient(rows, dim, gen, dtype)
            v = x.float()
            s['mean'] = v.mean(1) if case['center'] else None
            if case['center']:
                v = v - s['mean'][:, None]
            s['rstd'] = torch.rsqrt(v.square().mean(1) + EPS)
            if case['checkpoint']:
                s['q'], s['s'] = _pack(x)
                s['x'] = None
    elif op == 'pack':
        s['x'] = _stream(rows, case['dim'], gen, dtype)
    elif op == 'unpack':
        s['q'], s['s'] = _pack(_stream(rows, case['dim'], gen, dtype))
    elif op == 'pack_weight':
        s['w'] = (0.02 * torch.randn(rows, case['dim'], device=dev, generator=gen)).to(dtype)
    else:
        s['x'] = _stream(rows, case['inner'], gen, dtype)
        w = 0.02 * torch.randn(case['outer'], case['inner'], device=dev, generator=gen)
        s['w8'] = _pack_weight(w.bfloat16())
        if op == 'projection':
            s['dy'] = _gradient(rows, case['outer'], gen, dtype)
    return s


# ------------------------------------------------------------------------------------------------------- plain form
def _ceil(n, m):
    return -(-n // m) * m


def _exponents(amax):
    """The least e >= -127 with amax <= 448 * 2^e (448 = 0.875 * 2^9)."""
    m, ex = torch.frexp(amax)
    e = torch.where(m <= 0.875, ex - 9, ex - 8)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp_(min=-127)


def _e8(e, columns):
    """Exponents [rows, blocks] as E8M0 bytes, padded with ones to `columns`."""
    out = torch.full((e.shape[0], columns), 127, dtype=torch.uint8, device=e.device)
    out[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return out.view(E8)


def _powers(s):
    """2^e of E8M0 bytes, in 32 bits."""
    return torch.exp2(s.view(torch.uint8).float() - 127)


def _pack(x):
    rows, dim = x.shape
    wide = _ceil(dim, BLOCK)
    v = torch.zeros(rows, wide, device=x.device)
    v[:, :dim] = x.float()
    v = v.view(rows, wide // BLOCK, BLOCK)
    e = _exponents(v.abs().amax(2))
    q = (v * torch.exp2(-e.float())[:, :, None]).to(F8).view(rows, wide)
    return q, _e8(e, _ceil(wide // BLOCK, 4))


def _unpack(q, s, dim):
    rows, wide = q.shape
    v = q.float().view(rows, wide // BLOCK, BLOCK) * _powers(s)[:, :wide // BLOCK, None]
    return v.view(rows, wide)[:, :dim]


def _pack_weight(w):
    N, K = w.shape
    n, k = _ceil(N, BLOCK), _ceil(K, BLOCK)
    v = torch.zeros(n, k, device=w.device)
    v[:N, :K] = w.float()
    v = v.view(n // BLOCK, BLOCK, k // BLOCK, BLOCK)
    e = _exponents(v.abs().amax(3).amax(1))
    v = (v * torch.exp2(-e.float())[:, None, :, None]).reshape(n, k)
    return {'q': v[:N].to(F8), 's': _e8(e, _ceil(k // BLOCK, 4)), 'qt': v.t()[:K].contiguous().to(F8),
            'st': _e8(e.t(), _ceil(n // BLOCK, 4)), 'shape': (N, K)}


def _weight(w8):
    N, K = w8['shape']
    k = _ceil(K, BLOCK) // BLOCK
    scale = _powers(w8['s'])[:, :k].repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)
    return (w8['q'].float() * scale)[:, :K]


def _plain(s):
    op, dtype = s['op'], DTYPES[s['dtype']]
    if op == 'norm':
        x = s['x'].float()
        mean = x.mean(1) if s['center'] else None
        c = x - mean[:, None] if s['center'] else x
        rstd = torch.rsqrt(c.square().mean(1) + EPS)
        y = c * rstd[:, None] * s['w'].float()
        if s['center']:
            y = y + s['b'].float()
        out = list(_pack(y)) if s['y8'] else [y.to(dtype)]
        out += [mean, rstd] if s['center'] else [rstd]
        return out + (list(_pack(s['x'])) if s['checkpoint'] else [])
    if op == 'norm_grad':
        x = _unpack(s['q'], s['s'], s['dim']) if s['checkpoint'] else s['x'].float()
        dy, r = s['dy'].float(), s['rstd'][:, None]
        xh = (x - s['mean'][:, None]) * r if s['center'] else x * r
        g = dy * s['w'].float()
        t = g - xh * (g * xh).mean(1, keepdim=True)
        if s['center']:
            t = t - g.mean(1, keepdim=True)
        out = [(t * r).to(dtype), (dy * xh).sum(0).to(dtype)]
        return out + ([dy.sum(0).to(dtype)] if s['center'] else [])
    if op == 'pack':
        return _pack(s['x'])
    if op == 'unpack':
        return _unpack(s['q'], s['s'], s['dim']).to(dtype)
    if op == 'pack_weight':
        w8 = _pack_weight(s['w'])
        return [w8['q'], w8['s'], w8['qt'], w8['st']]
    w = _weight(s['w8'])
    x = _unpack(*_pack(s['x']), s['inner'])
    y = (x @ w.t()).to(dtype)
    if op == 'product':
        return y
    dy = _unpack(*_pack(s['dy']), s['outer'])
    return [y, (dy @ w).to(dtype), (s['dy'].float().t() @ x).to(dtype)]


# --------------------------------------------------------------------------------------------- the package's operators
def _own(s):
    from faster_yoco_amd import act8, linear8, norm
    op, dtype = s['op'], DTYPES[s['dtype']]
    if op == 'norm':
        if s['center']:
            out = norm.layer_norm(s['x'], s['w'], s['b'], EPS, y8=s['y8'], checkpoint=s['checkpoint'])
        else:
            out = norm.rms_norm(s['x'], s['w'], EPS, y8=s['y8'], checkpoint=s['checkpoint'])
        flat = []
        for t in out:
            flat += [t.q, t.s] if isinstance(t, act8.Act8) else [t]
        return flat
    if op == 'norm_grad':
        x = act8.Act8(s['q'], s['s'], s['dim']) if s['checkpoint'] else s['x']
        if s['center']:
            return list(norm.layer_norm_backward(s['dy'], x, s['mean'], s['rstd'], s['w'], bias=True))
        return list(norm.rms_norm_backward(s['dy'], x, s['rstd'], s['w']))
    if op == 'pack':
        a = act8.pack(s['x'])
        return a.q, a.s
    if op == 'unpack':
        return act8.unpack(act8.Act8(s['q'], s['s'], s['dim']), dtype)
    if op == 'pack_weight':
        w = linear8.pack_weight(s['w'])
        return [w.q, w.s, w.qt, w.st]
    w = linear8.Weight8(s['w8']['q'], s['w8']['s'], s['w8']['qt'], s['w8']['st'], s['w8']['shape'])
    x = act8.pack(s['x'])
    y = linear8.matmul(x, w, dtype)
    if op == 'product':
        return y
    dx = linear8.matmul(act8.pack(s['dy']), w, dtype, transposed=True)
    return [y, dx, linear8.weight_grad(s['dy'], x, dtype)]


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------------------- 64-bit definition
def _grid(v):
    """v (64 bits, |v| <= 448) rounded to e4m3's values: three mantissa bits, exponents from -6, ties to even."""
    a = v.abs().clamp(min=2.0 ** -20)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_scales(amax):
    e = torch.ceil(torch.log2(amax / 448))
    e = torch.where(amax > torch.exp2(e) * 448, e + 1, e)
    e = torch.where(amax <= torch.exp2(e - 1) * 448, e - 1, e)
    return torch.exp2(torch.where(amax > 0, e, torch.full_like(e, -127.0)).clamp(min=-127))


def _exact_rows(x):
    """(values before scaling back, scales with their padding, the values stood for) of rows in blocks."""
    pad = -x.shape[1] % BLOCK
    v = torch.nn.functional.pad(x, (0, pad)).unflatten(1, (-1, BLOCK))
    s = _exact_scales(v.abs().amax(2))
    q = _grid(v / s[..., None])
    stood = (q * s[..., None]).flatten(1)[:, :x.shape[1]]
    return q.flatten(1), torch.nn.functional.pad(s, (0, -s.shape[1] % 4), value=1.0), stood


def exact(case, seed):
    st = prepare(case, seed)
    op = case['op']
    if op == 'unpack':
        k = st['q'].shape[1] // BLOCK
        e = st['s'].view(torch.uint8)[:, :k].double() - 127
        return (st['q'].double().unflatten(1, (k, BLOCK)) * torch.exp2(e)[..., None]).flatten(1)[:, :case['dim']]
    if op == 'pack':
        return _exact_rows(st['x'].double())[:2]
    if op == 'pack_weight':
        w = st['w'].double()
        N, K = w.shape
        v = torch.nn.functional.pad(w, (0, -K % BLOCK, 0, -N % BLOCK))
        s = _exact_scales(v.abs().unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK)).amax((1, 3)))
        q = _grid(v / s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1))
        four = lambda t: torch.nn.functional.pad(t, (0, -t.shape[1] % 4), value=1.0)  # noqa: E731
        return [q[:N], four(s), q.t()[:K].contiguous(), four(s.t())]
    if op in ('norm', 'norm_grad'):
        n = case['dim']
        w = st['w'].double()
        if op == 'norm':
            x = st['x'].double()
            mean = x.sum(1) / n
            c = x - mean[:, None] if case['center'] else x
            rstd = 1 / torch.sqrt((c * c).sum(1) / n + EPS)
            y = c * rstd[:, None] * w + (st['b'].double() if case['center'] else 0)
            out = list(_exact_rows(y)[:2]) if case['y8'] else [y]
            out += [mean, rstd] if case['center'] else [rstd]
            return out + (list(_exact_rows(x)[:2]) if case['checkpoint'] else [])
        if case['checkpoint']:
            k = st['q'].shape[1] // BLOCK
            e = st['s'].view(torch.uint8)[:, :k].double() - 127
            x = (st['q'].double().unflatten(1, (k, BLOCK)) * torch.exp2(e)[..., None]).flatten(1)[:, :n]
        else:
            x = st['x'].double()
        dy, r = st['dy'].double(), st['rstd'].double()[:, None]
        xh = (x - (st['mean'].double()[:, None] if case['center'] else 0)) * r
        g = dy * w
        dx = r * (g - xh * ((g * xh).sum(1, keepdim=True) / n) - (g.sum(1, keepdim=True) / n if case['center'] else 0))
        return [dx, (dy * xh).sum(0)] + ([dy.sum(0)] if case['center'] else [])
    w8 = st['w8']
    N, K = w8['shape']
    e = w8['s'].view(torch.uint8).double() - 127
    rows = torch.arange(N, device=e.device) // BLOCK
    columns = torch.arange(K, device=e.device) // BLOCK
    w = w8['q'].double()[:, :K] * torch.exp2(e[rows][:, columns])
    x = _exact_rows(st['x'].double())[2]
    if op == 'product':
        return x @ w.t()
    dy = st['dy'].double()
    return [x @ w.t(), _exact_rows(dy)[2] @ w, dy.t() @ x]
