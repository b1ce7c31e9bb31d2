"""Layer norm (hyper_amd.layers.layer_norm / LayerNorm, libhecka hecka_layernorm_*) against the formula in 64 bits.

Tolerances count roundings, u = 2^-24.  A sum of D values passes at most 40 additions per value (16 in a thread, 6 between lanes,
16 between waves, the scaling): |d mean| <= 40 u mean|x|, the variance is off by 42 u of itself and 1 / sqrt by 24 u, so
|d xh| <= u (40 mean|x| r + 26 |xh|).  The result is rounded once more to its type, by half a step."""
import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def formula(x, w, b, eps, dy=None):
    """64-bit values and the bounds of their errors; x [G, R, D], w / b [G, D] or None."""
    x = x.double()
    G, R, D = x.shape
    w = torch.ones(G, 1, D, dtype=torch.float64, device=x.device) if w is None else w.double().unsqueeze(1)
    b = torch.zeros_like(w) if b is None else b.double().unsqueeze(1)
    mu = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    dxh = U * (40 * x.abs().mean(-1, keepdim=True) * r + 26 * xh.abs())
    y = xh * w + b
    out = {'y': (y, w.abs() * dxh + 4 * U * (y.abs() + (xh * w).abs()))}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        dx = r * (g - m1 - xh * m2)
        ag, agx = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
        dm2 = 44 * U * agx + (g.abs() * dxh).mean(-1, keepdim=True)
        out['dx'] = (dx, r * (U * (6 * g.abs() + 44 * ag + 6 * (xh * m2).abs()) + xh.abs() * dm2 + dxh * m2.abs()) + 28 * U * dx.abs())
        out['dw'] = ((dy * xh).sum(1), (U * (R + 40) * (dy * xh).abs() + dy.abs() * dxh).sum(1))
        out['db'] = (dy.sum(1), U * (R + 40) * dy.abs().sum(1))
    return out


def held(got, want, what):
    val, tol = want
    half = HALF[got.dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[got.dtype] / 2      # below the normal range a step is fixed
    err = (got.double() - val).abs()
    over = err - (tol * (1 + half) + half * val.abs() + tiny)
    assert bool((over <= 0).all()), '%s: off by %.3g, over its bound by %.3g' % (what, float(err.max()), float(over.max()))


def data(G, R, D, dtype, seed=0, offset=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(G, R, D, generator=gen) * torch.exp(torch.randn(G, R, 1, generator=gen)) + offset).to(dtype)
    dy = torch.randn(G, R, D, generator=gen).to(dtype)
    return x.cuda(), dy.cuda(), (1 + 0.3 * torch.randn(G, D, generator=gen)).cuda(), torch.randn(G, D, generator=gen).cuda()


# one wave per row up to 1024, then 256, 512 and 1024 threads; a piece more and less than each of them holds; odd everywhere
WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 255, 257, 512, 1001, 1023, 1024, 1025, 2047, 2049, 4096, 4099, 8191, 8200, 16383, 16384]


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('D', WIDTHS)
def test_forward_and_gradients_against_the_formula(D, dtype):
    from hyper_amd.layers import layer_norm
    G, R = 3, 7
    x, dy, w, b = data(G, R, D, dtype, D)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = layer_norm(x, w, b, 1e-5)
    assert y.dtype == dtype and y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = formula(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for name, got in (('y', y.detach()), ('dx', dx), ('dw', dw), ('db', db)):
        held(got, want[name], name)


@gpu
@pytest.mark.parametrize('R', [1, 2, 3, 4, 5, 257, 3000])
def test_row_counts(R):
    from hyper_amd.layers import layer_norm
    for G, D in ((1, 96), (5, 1300), (2, 64), (3, 20)):
        x, dy, w, b = data(G, R, D, torch.float32, R)
        for t in (x, w, b):
            t.requires_grad_(True)
        y = layer_norm(x, w, b)
        got = (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
        want = formula(x.detach(), w.detach(), b.detach(), 1e-5, dy)
        for name, t in zip(('y', 'dx', 'dw', 'db'), got):
            held(t, want[name], '%s R=%d' % (name, R))


@gpu
def test_rows_far_from_zero_and_constant_rows():
    from hyper_amd.layers import layer_norm
    x, dy, w, b = data(2, 5, 300, torch.float32, 4, offset=1000.0)
    x[0, 1] = 3.5            # no spread at all: xh is zero exactly, y the bias
    x[1, 2] = 0.0
    x.requires_grad_(True)
    y = layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    want = formula(x.detach(), w, b, 1e-5, dy)
    held(y.detach(), want['y'], 'y')
    held(dx, want['dx'], 'dx')
    assert torch.equal(y[0, 1].detach(), b[0]) and torch.equal(y[1, 2].detach(), b[1])


@gpu
def test_a_bad_row_stays_alone():
    from hyper_amd.layers import layer_norm
    x, dy, w, b = data(2, 6, 130, torch.float32, 5)
    good = layer_norm(x, w, b)
    x[0, 2, 7] = float('nan')
    x[1, 3, 0] = float('inf')
    y = layer_norm(x, w, b)
    assert bool(y[0, 2].isnan().all()) and bool(y[1, 3].isnan().any())
    keep = torch.ones(2, 6, dtype=torch.bool)
    keep[0, 2] = keep[1, 3] = False
    assert torch.equal(y[keep], good[keep])


@gpu
def test_shared_weight_missing_parts_and_strides():
    from hyper_amd.layers import layer_norm
    x, dy, w, b = data(3, 10, 200, torch.float32, 6)
    x.requires_grad_(True)
    w1, b1 = w[0].clone().requires_grad_(True), b[0].clone().requires_grad_(True)
    y = layer_norm(x, w1, b1)
    dx, dw, db = torch.autograd.grad(y, (x, w1, b1), dy)
    want = formula(x.detach().view(1, 30, 200), w1.detach()[None], b1.detach()[None], 1e-5, dy.view(1, 30, 200))
    held(y.detach().view(1, 30, 200), want['y'], 'y')
    held(dw[None], want['dw'], 'shared dw')
    held(db[None], want['db'], 'shared db')
    # no affine part; only a weight; only some gradients
    y0 = layer_norm(x)
    held(y0.detach(), formula(x.detach(), None, None, 1e-5)['y'], 'plain')
    held(torch.autograd.grad(y0, x, dy)[0], formula(x.detach(), None, None, 1e-5, dy)['dx'], 'plain dx')
    wg = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(layer_norm(x.detach(), wg), wg, dy)
    held(dw, formula(x.detach(), w, None, 1e-5, dy)['dw'], 'dw alone')
    # a strided x and gradient, more axes, vectors
    xt = x.detach().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(layer_norm(xt, w, b), layer_norm(x.detach(), w, b))
    x4 = x.detach().view(3, 2, 5, 200)
    assert torch.equal(layer_norm(x4, w, b).view(3, 10, 200), layer_norm(x.detach(), w, b))
    assert torch.equal(layer_norm(x.detach()[0, 0], w1.detach(), b1.detach()), y.detach()[0, 0])
    # an expanded gradient
    y = layer_norm(x, w, b)
    dx1, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    dx2, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx1, dx2)


@gpu
def test_rows_past_two_to_the_thirty_one_elements():
    from hyper_amd.layers import layer_norm
    R, D, n = 131200, 16384, 3
    x, dy, w, b = data(1, n, D, torch.bfloat16, 6)
    w, b = w[0].clone().requires_grad_(True), b[0].clone().requires_grad_(True)
    far, fdy = torch.zeros(R, D, device='cuda', dtype=torch.bfloat16), torch.zeros(R, D, device='cuda', dtype=torch.bfloat16)
    far[-n:], fdy[-n:] = x[0], dy[0]
    x, far = x[0].requires_grad_(True), far.requires_grad_(True)
    y, want = layer_norm(far, w, b), layer_norm(x, w, b)
    assert y.numel() > 2 ** 31 and torch.equal(y[-n:], want) and torch.equal(y[0], b.bfloat16())
    got, ref = torch.autograd.grad(y, (far, w, b), fdy), torch.autograd.grad(want, (x, w, b), dy[0])
    assert torch.equal(got[0][-n:], ref[0]) and float(got[0][:-n].abs().max()) == 0
    # the sums over rows: n terms each (the other rows' are zeros), added in another order
    xh = (x.detach().double() - x.detach().double().mean(-1, keepdim=True)) / x.detach().double().std(-1, correction=0, keepdim=True)
    for g, r, m in zip(got[1:], ref[1:], ((dy[0].double() * xh).abs().sum(0), dy[0].double().abs().sum(0))):
        assert bool(((g - r).abs() <= 2 * n * 2.0 ** -24 * m.detach()).all())


@gpu
def test_gradient_against_differences():
    from hyper_amd.layers import layer_norm
    x, dy, w, b = data(2, 3, 24, torch.float32, 7)
    for t in (x, w, b):
        t.requires_grad_(True)
    grads = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    gen = torch.Generator().manual_seed(1)
    h = 1e-4
    for t, gr in zip((x, w, b), grads):
        way = torch.randn(t.shape, generator=gen).cuda()
        f = []
        for s in (h, -h):
            args = [a.detach().double() + (s * way.double() if a is t else 0.0) for a in (x, w, b)]
            f.append(float((formula(*args, 1e-5)['y'][0] * dy.double()).sum()))
        slope = (f[0] - f[1]) / (2 * h)
        # h^2 / 6 times the third derivative, of the order of the gradient's own size times 1e-8; the kernel's 1e-5 is larger
        assert abs(slope - float((gr.double() * way.double()).sum())) <= 1e-4 * float((gr.abs() * way.abs()).sum())


@gpu
def test_empty_inputs():
    from hyper_amd.layers import layer_norm
    w = torch.ones(2, 8, device='cuda', requires_grad=True)
    x = torch.zeros(2, 0, 8, device='cuda', requires_grad=True)
    y = layer_norm(x, w, None)
    assert y.shape == (2, 0, 8)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(dw))


@gpu
def test_same_bits_every_time_on_another_stream_and_in_a_graph():
    from hyper_amd.layers import layer_norm
    x, dy, w, b = data(4, 700, 1500, torch.bfloat16, 8)
    for t in (x, w, b):
        t.requires_grad_(True)

    def step():
        y = layer_norm(x, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)
    first = step()
    assert all(torch.equal(p, q) for p, q in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for k in range(3):
        with torch.no_grad():
            x.copy_(data(4, 700, 1500, torch.bfloat16, 20 + k)[0])
        for gr in graphs:
            gr.replay()
        want = step()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(p, q) for p, q in zip(want, o)), 'replay %d' % k


@gpu
def test_layer_in_an_ensemble():
    """LayerNorm between Linear layers of a fixed ensemble: its flat parameter row gives the function's result, and gradients."""
    from hyper_amd.generators.ensemble import FixedEnsembleModel
    from hyper_amd.layers import LayerNorm, Linear, SequentialModule, build_gen_module, layer_norm
    assert isinstance(build_gen_module({'name': 'layer_norm', 'num_features': 5}), LayerNorm)
    torch.manual_seed(0)
    model = FixedEnsembleModel(SequentialModule(modules=[Linear(20, 33), LayerNorm(33), Linear(33, 4)]), 3).cuda()
    names = [n for n, _ in model.named_parameters()]
    assert 'layer_generators.1.affine.self.fixed_parameters.weight' in names
    with torch.no_grad():
        for n, p in model.named_parameters():
            if '.1.affine' in n:
                p.normal_()
    x = torch.randn(3, 9, 20, device='cuda')
    for ids in (None, [2, 0]):      # all members in order, and a selection
        params = model.forward_params(model.sample_params(ids if ids is None else ids, device=x.device) if ids else None, device=x.device)
        xi = x if ids is None else x[ids]
        feats, out = model.target(params, xi)
        flat = params['1']['affine']['self']
        want = layer_norm(feats['0'], flat[:, :33].contiguous(), flat[:, 33:].contiguous())
        assert torch.equal(feats['1'], want)
        grads = torch.autograd.grad(out.square().sum(), [p for p in model.parameters()])
        assert all(bool(torch.isfinite(g).all()) and bool((g != 0).any()) for g in grads)


def test_refusals():
    from hyper_amd import _lib
    from hyper_amd.layers import LayerNorm, layer_norm
    with pytest.raises(RuntimeError, match='GPU'):
        layer_norm(torch.randn(2, 3))
    with pytest.raises(ValueError):
        LayerNorm(0)
    with pytest.raises(ValueError):
        LayerNorm(16385)
    L, one = _lib.lib(), 64
    assert L.hecka_layernorm_fwd(one, 7, 1, 1, 8, None, None, 0, 1e-5, one, None, None, None) == -1
    assert L.hecka_layernorm_fwd(one, 0, 1, 0, 8, None, None, 0, 1e-5, one, None, None, None) == -1
    assert L.hecka_layernorm_fwd(one, 0, 1, 1, 16385, None, None, 0, 1e-5, one, None, None, None) == -1
    assert L.hecka_layernorm_fwd(one, 0, 1, 1, 8, None, None, 0, 1e-5, one, one, None, None) == -1
    assert L.hecka_layernorm_fwd(None, 0, 1, 1, 8, None, None, 0, 1e-5, one, None, None, None) == -1
    assert L.hecka_layernorm_bwd_workspace_bytes(1, 4000, 100) > 0 and L.hecka_layernorm_bwd_workspace_bytes(0, 1, 1) == 0
    assert L.hecka_layernorm_bwd(one, one, 0, one, one, 1, 4000, 100, None, 0, one, one, one, 100, None, 0, None) == -3


@gpu
def test_refusals_on_the_gpu():
    from hyper_amd.layers import LayerNorm, layer_norm
    x, _, w, b = data(2, 3, 8, torch.float32)
    for bad in (dict(x=x.double()), dict(x=x.long()), dict(weight=w.half(), bias=None)):
        with pytest.raises(TypeError):
            layer_norm(**{'x': x, 'weight': w, 'bias': b, **bad})
    for bad in (dict(weight=w[:1], bias=b[:1]), dict(weight=w[:, :4], bias=b[:, :4]), dict(weight=None), dict(bias=b[0]),
                dict(x=torch.zeros(2, 3, 0, device='cuda')), dict(x=torch.zeros(1, 16385, device='cuda'), weight=None, bias=None)):
        with pytest.raises(ValueError):
            layer_norm(**{'x': x, 'weight': w, 'bias': b, **bad})
    with pytest.raises(RuntimeError):
        layer_norm(x, w.cpu(), b.cpu())
    with pytest.raises(ValueError):
        LayerNorm(9)({'affine': {'self': torch.ones(2, 18, device='cuda')}}, x)
    xg = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(layer_norm(xg, w, b).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):      # no second derivative
        g.sum().backward()
