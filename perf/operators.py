"""Layer norm, 8-bit activation checkpoints and 8-bit block-scaled products: the cases that are timed, each operator's plain form in
elementary torch operations, and its values in 64 bits.

An 8-bit block: 128 consecutive elements of a row share one power of two s = 2^q, the smallest with max |x| <= 448 s over the block's finite
elements; an element is kept as the e4m3 code nearest to x / s (ties to even).  Weights share one s over 128 x 128 elements."""
import math
import os
import sys

import torch

own = False

BLOCK = 128
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one sample through five members' hidden layer norm (the LeNet-5 head's width): latency only
        dict(name='norm token', op='norm', train=False, members=5, rows=1, width=120, dtype='float32'),
        # a training step's norm at an ordinary ensemble batch, odd width (no vector load fits), half precision
        dict(name='norm odd fp16', op='norm', train=True, members=5, rows=300, width=1001, dtype='float16'),
        # fp32 members, ordinary hidden width
        dict(name='norm fp32', op='norm', train=True, members=10, rows=2048, width=2048, dtype='float32'),
        # long batches of wide rows
        dict(name='norm long bf16', op='norm', train=True, members=2, rows=16384, width=8192, dtype='bfloat16'),
        # gelu of the MNIST-sized MLP, its input kept in 8 bits
        dict(name='gelu small fp32', op='act', act='gelu', members=5, rows=100, width=784, dtype='float32'),
        # silu of a wide hidden layer over a long batch
        dict(name='silu large bf16', op='act', act='silu', members=10, rows=4096, width=4096, dtype='bfloat16'),
        # weight gradient of a layer whose input was kept in 8 bits: ragged in every size
        dict(name='wgrad ragged fp32', op='wgrad', members=5, rows=300, inputs=784, outputs=513, dtype='float32'),
        # the same at a width where the matrix cores are full
        dict(name='wgrad large fp32', op='wgrad', members=8, rows=4096, inputs=2048, outputs=2048, dtype='float32'),
        # one token through eight members, weights laid out once
        dict(name='linear token bf16', op='serve', members=8, rows=1, inputs=4096, outputs=4096, dtype='bfloat16'),
        # a prompt through one model
        dict(name='linear prompt bf16', op='serve', members=1, rows=2048, inputs=8192, outputs=8192, dtype='bfloat16'),
        # a training step of the MNIST-sized ensemble's hidden layer, fp32 tensors, ragged
        dict(name='linear ragged fp32', op='train', members=5, rows=300, inputs=784, outputs=1200, dtype='float32'),
        # a training step of wide layers, 16-bit tensors
        dict(name='linear wide bf16', op='train', members=2, rows=8192, inputs=4096, outputs=8192, dtype='bfloat16'),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm; every other one rounded to a multiple of 8 where it is not small."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v > 64 and rng.random() < 0.5:
        v = v // 8 * 8
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(['norm', 'act', 'wgrad', 'serve', 'train'])
    c = dict(op=op, members=rng.randint(1, 10), dtype=rng.choice(sorted(TYPES)))
    if op in ('norm', 'act'):
        c.update(rows=_spread(rng, 1, 8192), width=_spread(rng, 16, 16384))     # (a norm over two or three values has next to no gradient)
        if op == 'norm':
            c['train'] = rng.random() < 0.75
        else:
            c['act'] = rng.choice(['gelu', 'silu', 'tanh', 'sigmoid', 'crater'])
        c['rows'] = max(1, min(c['rows'], (1 << 27) // (c['members'] * c['width'])))
        return c
    c.update(inputs=_spread(rng, 1, 8192), outputs=_spread(rng, 1, 8192))
    c['rows'] = rng.randint(1, 16) if op == 'serve' and rng.random() < 0.5 else _spread(rng, 1, 8192)
    c['rows'] = max(1, min(c['rows'], (1 << 35) // (c['members'] * c['inputs'] * c['outputs'])))
    return c


def _features(shape, gen, dtype):
    """Hidden features: normal values, a scale for each sample and a few channels that are larger than the rest."""
    x = torch.randn(shape, generator=gen, device='cuda')
    x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=gen, device='cuda'))
    x *= 1.0 + 9.0 * (torch.rand(shape[-1:], generator=gen, device='cuda') < 0.01)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    M, N, t = case['members'], case['rows'], TYPES[case['dtype']]
    s = {'case': case, 'eps': 1e-5}
    if case['op'] in ('norm', 'act'):
        D = case['width']
        s['x'] = _features((M, N, D), gen, t)
        if case['op'] == 'norm':
            s['weight'] = 1.0 + 0.2 * torch.randn((M, D), generator=gen, device='cuda')
            s['bias'] = 0.2 * torch.randn((M, D), generator=gen, device='cuda')
        if case.get('train', True):
            s['dy'] = (torch.randn((M, N, D), generator=gen, device='cuda') / N).to(t)
            for n in ('x', 'weight', 'bias'):
                if n in s:
                    s[n].requires_grad_(True)
        return s
    I, O = case['inputs'], case['outputs']
    s['scale'], s['bias_scale'] = 1.0 / math.sqrt(I), 1.0
    s['x'] = _features((M, N, I), gen, t)
    if case['op'] == 'wgrad':
        s['dy'] = (torch.randn((M, N, O), generator=gen, device='cuda') / N).to(t)
        return s
    W = torch.randn((M, O, I), generator=gen, device='cuda')
    s['bias'] = torch.randn((M, O), generator=gen, device='cuda')
    if case['op'] == 'serve':      # what a server keeps: the codes [M, O, I up to whole blocks] and the scale bytes
        s['codes'], s['scales'] = _weight_blocks(W)
        return s
    s['weight'] = W
    s['dy'] = (torch.randn((M, N, O), generator=gen, device='cuda') / N).to(t)
    for n in ('x', 'weight', 'bias'):
        s[n].requires_grad_(True)
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _exponent(amax):
    """q of s = 2^q: the smallest with amax <= 448 2^q, not below -126; 0 where the block is zero."""
    m, e = torch.frexp(amax)
    q = torch.clamp(e - 9 + (m > 0.875).to(torch.int32), min=-126)
    return torch.where(amax > 0, q, torch.zeros_like(q))


def _two(q):
    """2^q as float32, q in [-126, 127]."""
    return ((q + 127) << 23).view(torch.float32)


def _padded(x, multiple=BLOCK):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % multiple))


def _finite_max(a, dims):
    return torch.where(torch.isfinite(a), a.abs(), torch.zeros_like(a)).amax(dims)


def _rounded(x):
    """The values that x's 8-bit rows stand for, float32."""
    K = x.shape[-1]
    v = _padded(x.detach().float())
    v = v.view(v.shape[:-1] + (-1, BLOCK))
    q = _exponent(_finite_max(v, -1)).unsqueeze(-1)
    v = (v * _two(-q)).to(torch.float8_e4m3fn).float() * _two(q)
    return v.flatten(-2)[..., :K]


def _weight_blocks(W):
    """codes e4m3 [M, O, Ip] and scale bytes q + 127 [M, O / 128, up to whole fours of Ip / 128] of weights [M, O, I]."""
    M, O, I = W.shape
    v = torch.nn.functional.pad(W.detach().float(), (0, -I % BLOCK, 0, -O % BLOCK))
    v = v.view(M, v.shape[1] // BLOCK, BLOCK, v.shape[2] // BLOCK, BLOCK)
    q = _exponent(_finite_max(v, (2, 4)))
    codes = (v * _two(-q)[:, :, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.reshape(M, v.shape[1] * BLOCK, -1)[:, :O].contiguous()
    return codes, torch.nn.functional.pad((q + 127).to(torch.uint8), (0, -q.shape[-1] % 4)).contiguous()


def _weight_values(codes, scales, I):
    """float32 [M, O, I] of _weight_blocks' codes and scales."""
    M, O, Ip = codes.shape
    s = _two(scales[..., :Ip // BLOCK].to(torch.int32) - 127)
    s = s.repeat_interleave(BLOCK, 1)[:, :O].repeat_interleave(BLOCK, 2)
    return (codes.float() * s)[..., :I]


def _sums(a):
    """Sums over the rows of [M, N, D], float32 from 64 bits."""
    return a.sum(1, dtype=torch.float64).float()


def _plain_norm(s):
    x, w, b = s['x'].detach().float(), s['weight'].detach(), s['bias'].detach()
    t = s['x'].dtype
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + s['eps'])
    xh = d * r
    y = xh * w[:, None] + b[:, None]
    if 'dy' not in s:
        return {'y': y.to(t)}
    dy = s['dy'].float()
    g = dy * w[:, None]
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return {'y': y.to(t), 'dx': dx.to(t), 'dweight': _sums(dy * xh), 'dbias': _sums(dy)}


_CRATER, _HALF = math.sqrt(2.0) / 2.0 + 0.008274364699, math.sqrt(2.0) / 2.0


def _act(name, x):
    """(f(x), f'(x))."""
    if name == 'gelu':
        p = 0.5 * torch.special.erfc(-x * _HALF)
        return x * p, p + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == 'silu':
        p = 1.0 / (1.0 + torch.exp(-x))
        return x * p, p * (1.0 + x * (1.0 - p))
    if name == 'sigmoid':
        p = 1.0 / (1.0 + torch.exp(-x))
        return p, p * (1.0 - p)
    if name == 'tanh':
        p = torch.tanh(x)
        return p, 1.0 - p * p
    p = torch.tanh(_HALF * (x + 1.0))
    return _CRATER * x * (1.0 + p), _CRATER * (1.0 + p + x * _HALF * (1.0 - p * p))


def _plain_act(s):
    t, name = s['x'].dtype, s['case']['act']
    x = s['x'].detach().float()
    return {'y': _act(name, x)[0].to(t), 'dx': (s['dy'].float() * _act(name, _rounded(x))[1]).to(t)}


def _plain_wgrad(s, x8=None, dy=None):
    x8 = _rounded(s['x']) if x8 is None else x8
    dy = s['dy'].float() if dy is None else dy
    return {'dweight': s['scale'] * torch.matmul(dy.transpose(1, 2).contiguous(), x8), 'dbias': s['bias_scale'] * _sums(dy)}


def _product(a, w, s, bias):
    y = s['scale'] * torch.matmul(a, w.transpose(1, 2).contiguous())
    return y if bias is None else y + s['bias_scale'] * bias.detach()[:, None]


def _plain_serve(s):
    w = _weight_values(s['codes'], s['scales'], s['x'].shape[-1])
    return {'y': _product(_rounded(s['x']), w, s, s['bias']).to(s['x'].dtype)}


def _plain_train(s):
    t = s['x'].dtype
    x8, dy8 = _rounded(s['x']), _rounded(s['dy'])
    codes, scales = _weight_blocks(s['weight'])
    w = _weight_values(codes, scales, s['x'].shape[-1])
    y = _product(x8, w, s, s['bias'])
    dx = s['scale'] * torch.matmul(dy8, w)
    return {'y': y.to(t), 'dx': dx.to(t), **_plain_wgrad(s, x8)}


# ----------------------------------------------------------------------------------------------------------- the calls
def _package():
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'he-cka-ensembles_amd')
    if p not in sys.path:
        sys.path.insert(0, p)


def _own(s):
    _package()
    op = s['case']['op']
    if op == 'norm':
        from hyper_amd.layers.norm import layer_norm
        if 'dy' not in s:
            return {'y': layer_norm(s['x'], s['weight'], s['bias'], s['eps'])}
        y = layer_norm(s['x'], s['weight'], s['bias'], s['eps'])
        dx, dw, db = torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['dy'])
        return {'y': y.detach(), 'dx': dx, 'dweight': dw, 'dbias': db}
    if op == 'act':
        from hyper_amd.net.activation import checkpointed
        y = checkpointed(s['case']['act'], s['x'])
        dx, = torch.autograd.grad(y, (s['x'],), s['dy'])
        return {'y': y.detach(), 'dx': dx}
    from hyper_amd import block8
    if op == 'wgrad':
        dw, db = block8.weight_grad(s['dy'], block8.quantize(s['x']), scale=s['scale'], bias_scale=s['bias_scale'])
        return {'dweight': dw, 'dbias': db}
    if op == 'serve':
        w = block8.Weight8(s['codes'], s['scales'], inputs=s['x'].shape[-1])
        return {'y': block8.linear(s['x'], w, s['bias'], scale=s['scale'], bias_scale=s['bias_scale'])}
    y = block8.linear(s['x'], s['weight'], s['bias'], scale=s['scale'], bias_scale=s['bias_scale'])
    dx, dw, db = torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['dy'])
    return {'y': y.detach(), 'dx': dx, 'dweight': dw, 'dbias': db}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {'norm': _plain_norm, 'act': _plain_act, 'wgrad': _plain_wgrad, 'serve': _plain_serve,
                'train': _plain_train}[state['case']['op']](state)


# ----------------------------------------------------------------------------------------------------- bytes and flops
def work(case):
    M, N, b = case['members'], case['rows'], TYPES[case['dtype']].itemsize
    if case['op'] in ('norm', 'act'):
        n = M * N * case['width']
        if case['op'] == 'act':
            return {'bytes': 4 * n * b, 'flops': 40 * n}
        if not case['train']:
            return {'bytes': 2 * n * b + 8 * M * case['width'], 'flops': 8 * n}
        return {'bytes': 4 * n * b + 16 * M * case['width'], 'flops': 24 * n}
    I, O = case['inputs'], case['outputs']
    x, y, w = M * N * I * b, M * N * O * b, M * O * I
    if case['op'] == 'wgrad':
        return {'bytes': x + y + 4 * w + 4 * M * O, 'flops': 2 * w * N}
    if case['op'] == 'serve':
        return {'bytes': x + y + w + 4 * M * O, 'flops': 2 * w * N}
    return {'bytes': 2 * x + 2 * y + 8 * w + 8 * M * O, 'flops': 6 * w * N}


# ------------------------------------------------------------------------------------------------------- 64-bit values
def _near(v):
    """v, |v| <= 448, at the nearest value of three bits behind the leading one, the smallest step 2^-9; ties to even."""
    a = v.abs()
    top = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))).clamp(min=-6.0)
    step = torch.exp2(top - 3.0)
    return torch.round(v / step) * step


def _blocks64(v, rows, cols):
    """[M, R, K] in 64 bits with every rows x cols block rounded to its own scale."""
    M, R, K = v.shape
    p = torch.zeros((M, -(-R // rows) * rows, -(-K // cols) * cols), dtype=torch.float64, device=v.device)
    p[:, :R, :K] = v
    p = p.view(M, p.shape[1] // rows, rows, p.shape[2] // cols, cols)
    big = p.abs().amax((2, 4), keepdim=True)
    q = torch.ceil(torch.log2(torch.where(big > 0, big, torch.full_like(big, 448.0)) / 448.0)).clamp(min=-126.0)
    p = _near(p * torch.exp2(-q)) * torch.exp2(q)
    return p.reshape(M, p.shape[1] * rows, -1)[:, :R, :K]


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    with torch.no_grad():
        x = s['x'].double()
        if op == 'norm':
            w, b = s['weight'].double().unsqueeze(1), s['bias'].double().unsqueeze(1)
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            z = (x - mean) * torch.rsqrt(var + s['eps'])
            out = {'y': torch.addcmul(b, z, w)}
            if 'dy' in s:
                dy = s['dy'].double()
                g = dy * w
                D = x.shape[-1]
                inner = g - g.sum(-1, keepdim=True) / D - z * ((g * z).sum(-1, keepdim=True) / D)
                out.update(dx=inner * torch.rsqrt(var + s['eps']), dweight=(dy * z).sum(1), dbias=dy.sum(1))
            return out
        if op == 'act':
            out = {}
            with torch.enable_grad():
                for key, at in (('y', x), ('dx', _blocks64(x, 1, BLOCK))):
                    at = at.detach().requires_grad_(key == 'dx')
                    f = {'gelu': lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2.0)), 'silu': lambda v: v * torch.sigmoid(v),
                         'tanh': torch.tanh, 'sigmoid': torch.sigmoid,
                         'crater': lambda v: _CRATER * v * (1.0 + torch.tanh((v + 1.0) / math.sqrt(2.0)))}[case['act']](at)
                    out[key] = f.detach() if key == 'y' else torch.autograd.grad(f, at, s['dy'].double())[0]
            return out
        x8 = _blocks64(x, 1, BLOCK)
        out = {}
        if op != 'wgrad':
            if op == 'serve':
                M, O, Ip = s['codes'].shape
                q = s['scales'][..., :Ip // BLOCK].double() - 127.0
                w = (s['codes'].double().view(M, O, -1, BLOCK) * torch.exp2(q)[:, torch.arange(O, device=q.device) // BLOCK][..., None]).flatten(2)
                w = w[..., :x.shape[-1]]
            else:
                w = _blocks64(s['weight'].double(), BLOCK, BLOCK)
            out['y'] = torch.stack([a @ c.t() for a, c in zip(x8, w)]) * s['scale'] + s['bias_scale'] * s['bias'].double().unsqueeze(1)
        if op == 'train':
            out['dx'] = torch.stack([a @ c for a, c in zip(_blocks64(s['dy'].double(), 1, BLOCK), w)]) * s['scale']
        if op != 'serve':
            dy = s['dy'].double()
            out['dweight'] = torch.stack([a.t() @ c for a, c in zip(dy, x8)]) * s['scale']
            out['dbias'] = dy.sum(1) * s['bias_scale']
        return out
