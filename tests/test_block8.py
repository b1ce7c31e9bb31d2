"""8-bit blocks (hyper_amd.block8, net.activation.checkpointed, libhecka hecka_block8_*) against plain restatements in 64 bits.

u = 2^-24.  Codes and scales are held to the definition bit for bit.  Products of small whole numbers are exact in every path
(codes, sums and, for the 16-bit types, the matrix instruction), so their results are held to the rounded exact values bit for bit at
sizes and shapes where the kernels can go wrong; random values are held to bounds that count roundings."""
import math

import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- the definition, on the CPU
def exponent(big):
    """q of the smallest power of two with big <= 448 2^q, not below -126; 0 for a block of zeros (numbers, not tensors)."""
    if big == 0:
        return 0
    q = math.frexp(big)[1] - 9
    while big > math.ldexp(448.0, q):
        q += 1
    while q > -126 and big <= math.ldexp(448.0, q - 1):
        q -= 1
    return max(q, -126)


def e4m3(v):
    """The code's value nearest to v (64 bits, |v| <= 448), ties to even; NaN for what is not finite."""
    a = v.abs()
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), torch.clamp(e - 1, min=-6) - 3)
    return torch.where(torch.isfinite(v), torch.round(v / step) * step, torch.full_like(v, math.nan))


def blocks(x, rows, cols):
    """(values, scale bytes) of x [G, R, K], 64 bits on the CPU, with every rows x cols block on its own scale."""
    x = x.detach().cpu().double()
    G, R, K = x.shape
    out, nr, nc = x.clone(), -(-R // rows), -(-K // cols)
    byte = torch.zeros(G, nr, nc, dtype=torch.uint8)
    for g in range(G):
        for r in range(nr):
            for c in range(nc):
                at = (g, slice(r * rows, (r + 1) * rows), slice(c * cols, (c + 1) * cols))
                b = x[at]
                fin = b[torch.isfinite(b)]
                q = exponent(float(fin.abs().max()) if fin.numel() else 0.0)
                top = 240.0 if q == 120 else 448.0      # 256 2^120 is no fp32 number: a finite element stays finite
                out[at] = e4m3(torch.where(torch.isfinite(b), (b * 2.0 ** -q).clamp(-top, top), b)) * 2.0 ** q
                byte[g, r, c] = q + 127
    return out, byte


def same(a, b):
    """Equal values, NaN equal to NaN."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def features(shape, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=gen))
    return x.to(dtype)


def whole(shape, seed, most=4):
    """Small whole numbers times a power of two for each row: their codes are exact, as every sum of their products."""
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=gen).float()


# ----------------------------------------------------------------------------------------------------------- quantisation
@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('K', [1, 3, 8, 127, 128, 129, 500, 513, 784])
def test_codes_and_scales_are_the_definition(K, dtype):
    from hyper_amd import block8
    x = features((2, 5, K), dtype, K)
    x[0, 1] = 0
    if K > 2:
        x[1, 0, 0], x[1, 1, 1], x[1, 2, 2] = math.nan, math.inf, -math.inf
    q = block8.quantize(x.cuda())
    val, byte = blocks(x, 1, 128)
    nb = block8.row_blocks(K)
    assert q.codes.shape == (10, nb * 128) and q.scales.shape == (10, block8.scale_stride(K)) and q.shape == x.shape
    assert torch.equal(q.scales.cpu()[:, :nb].reshape(2, 5, nb), byte)
    assert bool((q.scales.cpu()[:, nb:] == 127).all())
    codes = q.codes.cpu().view(torch.float8_e4m3fn).double().view(2, 5, nb, 128) * torch.ldexp(torch.ones((), dtype=torch.float64), byte.int() - 127)[..., None]
    codes = codes.view(2, 5, -1)
    assert same(codes[..., :K], val) and bool((q.codes.cpu().view(2, 5, -1)[..., K:] == 0).all())
    for t in TYPES:
        out = block8.dequantize(q, t)
        assert out.dtype == t and out.shape == x.shape
        want = val.to(t) if t != torch.float16 else val.float().half()
        assert same(out.cpu(), want)


@gpu
def test_every_binade_and_every_tie():
    """All fp32 binades as the block's largest value, both sides of 448 2^q, and every midpoint of two codes."""
    from hyper_amd import block8
    rows = []
    for e in range(-149, 128):
        for m in (1.0, 1.75, 1.7500001, 1.9999999):
            r = torch.zeros(128)
            r[0] = min(math.ldexp(m, e), 3.4028234e38)
            r[1] = -r[0] / 3
            r[2] = r[0] / 300
            rows.append(r)
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = ((codes[1:] + codes[:-1]) / 2).float()
    r = torch.zeros(2, 128)
    r[0, :126], r[0, 127] = mid, 448.0
    r[1, :126], r[1, 127] = -mid * 2.0 ** 20, 448.0 * 2.0 ** 20
    x = torch.stack(rows + [r[0], r[1]])[None]
    q = block8.quantize(x.cuda())
    val, byte = blocks(x, 1, 128)
    assert torch.equal(q.scales.cpu()[:, 0], byte.view(-1))
    assert same(block8.dequantize(q).cpu().double(), val)


@gpu
def test_the_largest_finite_values_stay_finite():
    from hyper_amd import block8
    for t in TYPES:
        big = torch.finfo(t).max
        x = torch.tensor([[big, -big, 1.0, 0.0]], dtype=t, device='cuda')
        back = block8.dequantize(block8.quantize(x))
        assert bool(torch.isfinite(back).all()) and float((back - x)[0, :2].abs().max()) <= 2.0 ** -4 * big
        W = x.view(1, 1, 4)
        assert bool(torch.isfinite(block8.quantize_weight(W).codes.view(torch.float8_e4m3fn).float()).all())
        y = block8.linear(x.view(1, 1, 4), block8.quantize_weight(torch.ones(1, 1, 4, device='cuda')), scale=0.5)
        assert float(y.float().abs().max()) < big      # the largest values cancel


@gpu
def test_strided_rows_and_single_vectors():
    from hyper_amd import block8
    x = features((6, 300), torch.bfloat16, 3).cuda()
    for v in (x[::2], x[:, 5:200], x.t(), x[1], x[2:2], x.view(2, 3, 300)[:, 1:]):
        a, b = block8.quantize(v), block8.quantize(v.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and a.shape == v.shape
        assert block8.dequantize(a).shape == v.shape


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,O,I', [(1, 1, 1), (2, 130, 257), (1, 128, 128), (3, 5, 700), (1, 513, 3), (2, 256, 384)])
def test_weight_codes_both_ways(M, O, I, dtype):
    from hyper_amd import block8
    W = features((M, O, I), dtype, O + I)
    if O > 4 and I > 2:
        W[0, 4, 2] = math.nan
    w = block8.quantize_weight(W.cuda())
    val, byte = blocks(W, 128, 128)
    nI, nO = block8.row_blocks(I), block8.row_blocks(O)
    assert torch.equal(w.scales.cpu()[..., :nI], byte) and bool((w.scales.cpu()[..., nI:] == 127).all())
    assert torch.equal(w.scales_t.cpu()[..., :nO], byte.transpose(1, 2)) and bool((w.scales_t.cpu()[..., nO:] == 127).all())
    s = torch.ldexp(torch.ones((), dtype=torch.float64), byte.int() - 127).repeat_interleave(128, 1)[:, :O].repeat_interleave(128, 2)[..., :I]
    assert same(w.codes.cpu().view(torch.float8_e4m3fn).double()[..., :I] * s, val)
    assert torch.equal(w.codes_t.cpu()[..., :O], w.codes.cpu()[..., :I].transpose(1, 2))
    assert bool((w.codes.cpu()[..., I:] == 0).all()) and bool((w.codes_t.cpu()[..., O:] == 0).all())
    alone = block8.quantize_weight(W.cuda(), transposed=False)
    assert alone.codes_t is None and torch.equal(alone.codes, w.codes) and torch.equal(alone.scales, w.scales)


# ------------------------------------------------------------------------------------------------------------ activations
def act64(name, x):
    h = math.sqrt(0.5)
    if name == 'gelu':
        p = 0.5 * torch.erfc(-x * h)
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if name in ('silu', 'sigmoid'):
        p = torch.sigmoid(x)
        return (x * p, p * (1 + x * (1 - p))) if name == 'silu' else (p, p * (1 - p))
    if name == 'tanh':
        return torch.tanh(x), 1 - torch.tanh(x) ** 2
    c, p = h + 0.008274364699, torch.tanh(h * (x + 1))
    return c * x * (1 + p), c * (1 + p + x * h * (1 - p * p))


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('name', ['gelu', 'silu', 'tanh', 'sigmoid', 'crater'])
def test_checkpointed_activation(name, dtype):
    """y: the function at x.  dx: dy times the slope at the blocks' values.  The functions below them (erfc, exp, tanh) are off by a
    few u and see an argument off by 2 u of itself, whose effect on y is at most 2 u |x| max|f'|, on the slope 2 u max|x f''|; 32 u
    (1 + |x|) covers value and slope of all five."""
    from hyper_amd.net.activation import checkpointed
    for shape in ((3, 5, 257), (2, 128), (1, 1), (7,), (2, 2, 3, 130)):
        x = (features(shape, torch.float32, 1) * 2).clamp(-30, 30).to(dtype)
        dy = torch.randn(shape, generator=torch.Generator().manual_seed(2)).to(dtype)
        xg = x.cuda().requires_grad_(True)
        y = checkpointed(name, xg)
        dx, = torch.autograd.grad(y, xg, dy.cuda())
        assert y.dtype == dtype and dx.dtype == dtype and y.shape == shape and dx.shape == shape
        x8 = blocks(x.reshape(1, -1, shape[-1]), 1, 128)[0].view(shape)
        tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[dtype]
        for got, at, f, n in ((y.detach(), x.double(), 1.0, 0), (dx, x8, dy.double(), 1)):
            want = act64(name, at)[n] * f
            f = f if torch.is_tensor(f) else torch.ones_like(want)
            tol = 32 * U * (1 + at.abs()) * f.abs() + HALF[dtype] * want.abs() + tiny
            assert bool(((got.cpu().double() - want).abs() <= tol * (1 + HALF[dtype])).all()), (shape, n)


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_without_gradients_the_same_results_and_nothing_kept(dtype):
    from hyper_amd import block8
    from hyper_amd.layers import layer_norm
    from hyper_amd.net.activation import checkpointed
    x = features((2, 33, 300), dtype, 1).cuda().requires_grad_(True)
    W, b = torch.randn(2, 70, 300, device='cuda', requires_grad=True), torch.randn(2, 70, device='cuda', requires_grad=True)
    w1, b1 = torch.randn(2, 300, device='cuda', requires_grad=True), torch.randn(2, 300, device='cuda', requires_grad=True)
    calls = [lambda n=n: checkpointed(n, x) for n in ('gelu', 'silu', 'tanh', 'sigmoid', 'crater')]
    calls += [lambda: block8.linear(x, W, b), lambda: block8.linear(x[0], W, b, scale=0.5), lambda: layer_norm(x, w1, b1), lambda: layer_norm(x)]
    for call in calls:
        y = call()
        with torch.no_grad():
            z = call()
        assert y.requires_grad and not z.requires_grad and torch.equal(y.detach(), z)
        with torch.inference_mode():
            assert torch.equal(call(), z)
    v = x.detach().transpose(1, 2)
    assert torch.equal(checkpointed('gelu', v), checkpointed('gelu', v.contiguous()))
    assert checkpointed('gelu', x.detach()[:, :0]).shape == (2, 0, 300)


@gpu
def test_checkpointed_activation_keeps_bytes_and_takes_extremes():
    from hyper_amd.net.activation import checkpointed
    x = torch.randn(64, 4096, device='cuda', requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = checkpointed('gelu', x)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 4
    assert kept <= 1.1 * x.numel(), kept
    for name in ('gelu', 'silu', 'tanh', 'sigmoid', 'crater'):
        v = torch.tensor([[-3e38, -1e4, -100.0, -0.0, 0.0, 100.0, 1e4, 3e38]], device='cuda')
        y = checkpointed(name, v)
        assert bool(torch.isfinite(y[:, :7]).all()), (name, y)
    assert checkpointed('silu', torch.zeros(0, 4, device='cuda')).shape == (0, 4)


# --------------------------------------------------------------------------------------------------------------- products
# (M, N, O, I): one row to the token kernel's sixteen and past it, a tile less and more, odd everywhere, one of each, long sums
SHAPES = [(1, 1, 1, 1), (2, 1, 40, 200), (3, 16, 33, 129), (2, 17, 31, 128), (1, 5, 300, 1000), (2, 128, 128, 128), (1, 129, 257, 385),
          (5, 100, 10, 784), (1, 300, 130, 64), (2, 257, 128, 640), (1, 64, 7, 4099), (1, 513, 515, 130)]


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I', SHAPES)
def test_whole_numbers_come_out_exact(M, N, O, I, dtype):
    """Training (y, dx, dW, db) and serving of whole numbers: every rounding is that of the result."""
    from hyper_amd import block8
    x, W, b = whole((M, N, I), 1), whole((M, O, I), 2), whole((M, O), 3, 50)
    dy = whole((M, N, O), 4)
    xg, Wg, bg = x.to(dtype).cuda().requires_grad_(True), W.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    y = block8.linear(xg, Wg, bg, scale=0.25, bias_scale=2.0)
    dx, dW, db = torch.autograd.grad(y, (xg, Wg, bg), dy.to(dtype).cuda())
    xd, Wd, dyd = x.double(), W.double(), dy.double()
    want = {'y': 0.25 * torch.bmm(xd, Wd.transpose(1, 2).contiguous()) + 2.0 * b.double()[:, None], 'dx': 0.25 * torch.bmm(dyd, Wd),
            'dW': 0.25 * torch.bmm(dyd.transpose(1, 2).contiguous(), xd), 'db': 2.0 * dyd.sum(1)}
    for name, got in (('y', y.detach()), ('dx', dx), ('dW', dW), ('db', db)):
        assert got.dtype == (dtype if name in ('y', 'dx') else torch.float32)
        assert torch.equal(got.cpu(), want[name].to(got.dtype)), name
    w = block8.quantize_weight(W.cuda(), transposed=False)
    assert torch.equal(block8.linear(x.to(dtype).cuda(), w, b.cuda(), scale=0.25, bias_scale=2.0).cpu(), want['y'].to(dtype))
    q = block8.quantize(x.to(dtype).cuda())
    assert torch.equal(block8.linear(q, w, scale=0.25).cpu(), (want['y'] - 2.0 * b.double()[:, None]).to(dtype))


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(2, 3, 70, 300), (1, 200, 150, 1100), (3, 300, 784, 513), (1, 1030, 20, 40)])
def test_random_values_within_counted_roundings(M, N, O, I, dtype):
    """fp32 results: the products are exact, each of the K / 32 instructions and the 32 sums inside one rounds by u of the sum of
    magnitudes at most.  16-bit results: inside a group of eight the fp8 instruction cuts each product at 2^-13 of the largest, seven of
    them at most, so 7 * 2^-13 of the sum of magnitudes - and, as these cuts have the sign of their product and no more than half a
    step each on average, a 2-norm below 2^-14 of the result's own for values of mixed sign, where the half step is 2^-8 or 2^-11."""
    from hyper_amd import block8
    x, W, dy = features((M, N, I), dtype, 1), features((M, O, I), torch.float32, 2), features((M, N, O), dtype, 3)
    b = torch.randn(M, O, generator=torch.Generator().manual_seed(4))
    xg, Wg, bg = x.cuda().requires_grad_(True), W.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    y = block8.linear(xg, Wg, bg, scale=0.5, bias_scale=0.5)
    dx, dW, db = torch.autograd.grad(y, (xg, Wg, bg), dy.cuda())
    x8, w8, dy8 = blocks(x, 1, 128)[0], blocks(W, 128, 128)[0], blocks(dy, 1, 128)[0]
    dyd = dy.double()
    tr = lambda t: t.transpose(1, 2).contiguous()   # noqa: E731
    cases = {'y': (x8, tr(w8), y.detach(), 0.5 * b.double()[:, None], I), 'dx': (dy8, w8, dx, 0.0, O), 'dW': (tr(dyd), x8, dW, 0.0, N)}
    for name, (p, q, got, add, K) in cases.items():
        want, mags = 0.5 * torch.bmm(p, q) + add, 0.5 * torch.bmm(p.abs(), q.abs())
        err = (got.cpu().double() - want).abs()
        fp8 = got.dtype != torch.float32
        tol = U * (3 * K / 32 + 40) * mags + 4 * U * want.abs() + (7 * 2.0 ** -13 * mags if fp8 else 0.0)
        tol = tol + HALF[got.dtype] * (want.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
        finite = torch.isfinite(got.cpu().double())      # an fp16 result past 65504
        assert bool((err[finite] <= tol[finite]).all()) and (got.dtype == torch.float16 or bool(finite.all())), (name, float((err / tol)[finite].max()))
        rel = float(err[finite].norm() / want[finite].norm())
        assert rel <= (2.0 ** -14 if fp8 else 0.0) + (HALF[got.dtype] if got.dtype != torch.float32 else 1e-6), (name, rel)
    assert bool(((db.cpu().double() - 0.5 * dyd.sum(1)).abs() <= U * (N + 40) * dyd.abs().sum(1)).all())


@gpu
def test_token_and_prompt_paths_agree():
    """Row 5 of a batch gives the same fp32 result alone, among sixteen and among seventeen: both paths make the same codes and
    exact products; they add them up in another order."""
    from hyper_amd import block8
    x, W = features((2, 40, 1000), torch.float32, 1).cuda(), features((2, 90, 1000), torch.float32, 2).cuda()
    w = block8.quantize_weight(W)
    full = block8.linear(x, w).double()
    mags = torch.bmm(block8.dequantize(block8.quantize(x)).double().abs().cpu(), blocks(W, 128, 128)[0].abs().transpose(1, 2).contiguous()).cuda()
    for n in (1, 2, 15, 16, 17, 33):
        part = block8.linear(x[:, 5:5 + n] if n < 33 else x[:, :n], w).double()
        at = slice(5, 5 + n) if n < 33 else slice(0, n)
        assert bool(((part - full[:, at]).abs() <= U * 140 * mags[:, at]).all()), n


@gpu
def test_shared_rows_and_their_gradient():
    """x [N, I] through all members: its gradient is the members' sum."""
    from hyper_amd import block8
    for N in (5, 40):
        x, W, dy = whole((N, 200), 1), whole((3, 50, 200), 2), whole((3, N, 50), 3)
        xg, Wg = x.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
        y = block8.linear(xg, Wg)
        dx, dW = torch.autograd.grad(y, (xg, Wg), dy.cuda())
        assert torch.equal(y.detach().cpu().double(), torch.matmul(x.double(), W.double().transpose(1, 2).contiguous()))
        assert torch.equal(dx.cpu().double(), torch.bmm(dy.double(), W.double()).sum(0)) and dx.shape == x.shape
        assert torch.equal(dW.cpu().double(), torch.matmul(dy.double().transpose(1, 2).contiguous(), x.double()))
        w = block8.quantize_weight(W.cuda())
        assert torch.equal(block8.linear(x.cuda(), w), y.detach())
        dW2, db2 = block8.weight_grad(dy.cuda(), block8.quantize(x.cuda()))
        assert torch.equal(dW2, dW) and torch.equal(db2.cpu().double(), dy.double().sum(1))


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('shared', [False, True])
@pytest.mark.parametrize('M,N,O,I', [(30, 400, 1000, 300), (30, 400, 300, 1000)])
def test_large_tiles_with_ragged_edges(M, N, O, I, shared, dtype):
    """Tiles of 256 x 256 in y and dW, or in dx (whose sum over the members they also write)."""
    from hyper_amd import block8
    x, W, b, dy = whole((N, I) if shared else (M, N, I), 1), whole((M, O, I), 2), whole((M, O), 3, 50), whole((M, N, O), 4)
    xg, Wg, bg = x.to(dtype).cuda().requires_grad_(True), W.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    y = block8.linear(xg, Wg, bg, scale=0.25, bias_scale=2.0)
    dx, dW, db = torch.autograd.grad(y, (xg, Wg, bg), dy.to(dtype).cuda())
    xd = x.float().expand(M, N, I)      # sums of whole numbers below 2^24: exact in fp32 as well
    assert torch.equal(y.detach().cpu(), (0.25 * torch.bmm(xd, W.transpose(1, 2).contiguous()) + 2.0 * b[:, None]).to(dtype))
    want = 0.25 * torch.bmm(dy, W)
    assert torch.equal(dx.cpu(), (want.sum(0) if shared else want).to(dtype))
    assert torch.equal(dW.cpu(), 0.25 * torch.bmm(dy.transpose(1, 2).contiguous(), xd)) and torch.equal(db.cpu(), 2.0 * dy.sum(1))


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(1, 64, 130, 5000), (2, 33, 71, 2100), (1, 17, 3, 8200), (1, 300, 8, 2048)])
def test_long_sums_shared_out(M, N, O, I, dtype):
    """Few tiles and many blocks of K: the slabs' sum, its bias and rounding, and the same bits on every call."""
    from hyper_amd import _lib, block8
    assert _lib.lib().hecka_block8_linear_workspace_bytes(M, N, O, I, M, TYPES.index(dtype)) > 0
    x, W, b = whole((M, N, I), 1), whole((M, O, I), 2), whole((M, O), 3, 50)
    q, w = block8.quantize(x.to(dtype).cuda()), block8.quantize_weight(W.cuda())
    for bias in (None, b):
        y = block8.linear(q, w, None if bias is None else bias.cuda(), scale=0.25, bias_scale=2.0)
        want = 0.25 * torch.bmm(x.double(), W.double().transpose(1, 2).contiguous()) + (0.0 if bias is None else 2.0 * bias.double()[:, None])
        assert torch.equal(y.cpu(), want.to(dtype))
    x = features((M, N, I), dtype, 5).cuda()
    assert torch.equal(block8.linear(block8.quantize(x), w), block8.linear(block8.quantize(x), w))


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(3, 40, 50, 201), (2, 33, 4099, 35), (7, 1, 1, 1), (40, 700, 300, 129)])
def test_gradient_of_shared_rows_is_rounded_once(M, N, O, I, dtype):
    """The members' sum in fp32, also where the sum over outputs is long and shared out."""
    from hyper_amd import block8
    x, W, dy = whole((N, I), 1), whole((M, O, I), 2), whole((M, N, O), 3)
    xg = x.to(dtype).cuda().requires_grad_(True)
    dx, = torch.autograd.grad(block8.linear(xg, W.cuda(), scale=0.5), xg, dy.to(dtype).cuda())
    assert dx.dtype == dtype and torch.equal(dx.cpu(), (0.5 * torch.bmm(dy.double(), W.double()).sum(0)).to(dtype))


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_any_part_of_the_gradients(dtype):
    """Every choice of what requires a gradient and of what is asked for gives the bits of the whole step; strided x, W in a flat row."""
    from hyper_amd import block8
    M, N, O, I = 2, 21, 30, 140
    flat = torch.randn(M, O * I + 17, device='cuda')
    x0, b0, dy = features((M, N, 2 * I), dtype, 1).cuda()[:, :, :I], torch.randn(M, O, device='cuda'), features((M, N, O), dtype, 2).cuda()
    for shared in (False, True):
        whole_step = None
        for need in (7, 1, 2, 4, 3, 5, 6):
            x = (x0[0] if shared else x0).detach().requires_grad_(bool(need & 1))
            W = flat[:, :O * I].view(M, O, I).detach().requires_grad_(bool(need & 2))
            b = b0.detach().requires_grad_(bool(need & 4))
            y = block8.linear(x, W, b, scale=0.5, bias_scale=0.25)
            for ask in range(1, 8):
                if ask & ~need:
                    continue
                got = torch.autograd.grad(y, [t for i, t in enumerate((x, W, b)) if ask >> i & 1], dy, retain_graph=True)
                if whole_step is None and ask == need == 7:
                    whole_step = got
                if whole_step is not None:
                    want = [g for i, g in enumerate(whole_step) if ask >> i & 1]
                    assert all(torch.equal(p, q) for p, q in zip(got, want)), (shared, need, ask)


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_gradient_of_the_bias_alone(dtype):
    from hyper_amd import block8
    for M, N, O in ((2, 5, 7), (1, 5000, 33), (3, 130, 300)):
        b, dy = whole((M, O), 1).cuda().requires_grad_(True), whole((M, N, O), 2).to(dtype)
        y = block8.linear(torch.randn(M, N, 20, device='cuda', dtype=dtype), torch.randn(M, O, 20, device='cuda'), b, bias_scale=0.5)
        db, = torch.autograd.grad(y, b, dy.cuda())
        assert torch.equal(db.cpu().double(), 0.5 * dy.double().sum(1))
        if dtype == torch.float32:
            from hyper_amd.layers.linear import BatchedLinearCheckpoint
            y = BatchedLinearCheckpoint.apply(torch.randn(M, N, 20, device='cuda'), torch.randn(M, O, 20, device='cuda'), b, 1.0, 0.5)
            assert torch.equal(torch.autograd.grad(y, b, dy.cuda())[0], db)


@gpu
def test_not_a_number_reaches_its_row_and_column_only():
    from hyper_amd import block8
    for dtype in TYPES:
        for N in (4, 40):
            x, W, dy = whole((1, N, 300), 1).to(dtype), whole((1, 60, 300), 2), whole((1, N, 60), 3).to(dtype)
            good = block8.linear(x.cuda(), block8.quantize_weight(W.cuda()))
            gW, gb = block8.weight_grad(dy.cuda(), block8.quantize(x.cuda()))
            x[0, 2, 131] = math.inf
            y = block8.linear(x.cuda(), block8.quantize_weight(W.cuda()))
            dW, db = block8.weight_grad(dy.cuda(), block8.quantize(x.cuda()))
            assert bool(y[0, 2].isnan().all()) and torch.equal(y[0, :2], good[0, :2]) and torch.equal(y[0, 3:], good[0, 3:])
            assert bool(dW[0, :, 131].isnan().all()) and torch.equal(dW[0, :, :131], gW[0, :, :131]) and torch.equal(db, gb)


@gpu
def test_weight_gradient_cut_over_rows():
    """Few tiles over many rows: the pieces' sums, the same bits on every call, and fp16 / fp32 terms that reach past bf16."""
    from hyper_amd import _lib, block8
    M, N, O, I = 1, 5000, 40, 70
    assert _lib.lib().hecka_block8_wgrad_workspace_bytes(M, N, O, I) > 0
    for dtype in TYPES:
        x = whole((M, N, I), 1)
        dy = (whole((M, N, O), 2, 2000) / 1024).to(dtype)      # eleven bits: more than one bf16 term holds
        dW, db = block8.weight_grad(dy.cuda(), block8.quantize(x.to(dtype).cuda()), scale=2.0, bias_scale=0.5)
        again = block8.weight_grad(dy.cuda(), block8.quantize(x.to(dtype).cuda()), scale=2.0, bias_scale=0.5)
        assert torch.equal(dW, again[0]) and torch.equal(db, again[1])
        want, wb = 2.0 * torch.bmm(dy.double().transpose(1, 2).contiguous(), x.double()), 0.5 * dy.double().sum(1)
        assert bool(((dW.cpu().double() - want).abs() <= U * 64 * 2.0 * torch.bmm(dy.double().abs().transpose(1, 2).contiguous(), x.double().abs())).all())
        assert bool(((db.cpu().double() - wb).abs() <= U * 200 * dy.double().abs().sum(1)).all())


@gpu
def test_gradients_against_differences_of_the_rounded_function():
    """y is linear in the blocks' values and the gradient is taken through the rounding (its slope counts as one): with values that
    are their own codes, a change by whole codes has to change the loss by gradient times change, exactly."""
    from hyper_amd import block8
    x, W, dy = whole((2, 30, 140), 1, 2), whole((2, 35, 140), 2, 2), whole((2, 30, 35), 3, 2)
    x[..., 0::64], W[..., 0::64] = 4.0, 4.0      # fixes every block's scale
    xg, Wg = x.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    dx, dW = torch.autograd.grad(block8.linear(xg, Wg), (xg, Wg), dy.cuda())
    loss = lambda a, c: float((block8.linear(a.cuda(), c.cuda()).double() * dy.cuda().double()).sum())   # noqa: E731
    base = loss(x, W)
    for (m, i, j) in ((0, 3, 5), (1, 29, 139), (0, 0, 127)):
        d = x.clone()
        d[m, i, j] += 1
        assert loss(d, W) - base == float(dx[m, i, j])
        d = W.clone()
        d[m, i, j] += 1
        assert loss(x, d) - base == float(dW[m, i, j])


@gpu
def test_far_rows_of_a_large_checkpoint():
    """Offsets past 2^31 codes: the last rows of a checkpoint of 2.2e9 elements."""
    from hyper_amd import block8
    K, R = 4096, 540000
    x = torch.zeros(R, K, device='cuda', dtype=torch.bfloat16)
    x[-3:] = features((3, K), torch.bfloat16, 1).cuda()
    q = block8.quantize(x)
    tail = block8.quantize(x[-3:])
    assert torch.equal(q.codes[-3:], tail.codes) and torch.equal(q.scales[-3:], tail.scales) and int(q.codes[:-3].max()) == 0
    del x
    back = block8._values(q, torch.bfloat16)
    assert torch.equal(back[-3:], block8.dequantize(tail)) and float(back[:-3].abs().max()) == 0
    W = whole((1, 8, K), 2)
    y = block8.linear(block8.Rows8(q.codes, q.scales, (1, R, K), torch.bfloat16), block8.quantize_weight(W.cuda()))
    want = block8.linear(block8.Rows8(tail.codes, tail.scales, (1, 3, K), torch.bfloat16), block8.quantize_weight(W.cuda()))
    assert torch.equal(y[0, -3:], want[0]) and float(y[0, :-3].abs().max()) == 0


@gpu
def test_far_outputs_and_far_weights():
    """Results and gradients of more than 2^31 elements, and weights of as many: their last rows."""
    from hyper_amd import block8
    N, O, I, n = 140000, 16384, 40, 5
    x, W, dy = whole((1, n, I), 1).bfloat16().cuda(), whole((1, O, I), 2).cuda(), whole((1, n, O), 3).bfloat16().cuda()
    big = torch.zeros(1, N, I, device='cuda', dtype=torch.bfloat16)
    big[:, -n:] = x
    x, big = x.requires_grad_(True), big.requires_grad_(True)
    W.requires_grad_(True)
    y, want = block8.linear(big, W), block8.linear(x, W)
    assert y.numel() > 2 ** 31 and torch.equal(y[:, -n:], want) and float(y[:, :-n].detach().amax()) == 0
    far = torch.zeros_like(y)
    far[:, -n:] = dy
    dx, dW = torch.autograd.grad(y, (big, W), far)
    wx, wW = torch.autograd.grad(want, (x, W), dy)
    assert torch.equal(dx[:, -n:], wx) and float(dx[:, :-n].abs().max()) == 0 and torch.equal(dW, wW)
    del y, far, dx, big
    O, I = 131200, 16384
    W = torch.zeros(1, O, I, device='cuda', dtype=torch.bfloat16)
    W[:, -n:] = whole((1, n, I), 4).bfloat16().cuda()
    w, few = block8.quantize_weight(W), block8.quantize_weight(W[:, -128:].contiguous())
    assert w.codes.numel() > 2 ** 31 and torch.equal(w.codes[:, -n:], few.codes[:, -n:])
    for rows in (1, 20):
        x = whole((1, rows, I), 5).bfloat16().cuda()
        y = block8.linear(x, w)
        assert torch.equal(y[:, :, -128:], block8.linear(x, few)) and float(y[:, :, :-n].abs().max()) == 0


@gpu
def test_empty_batches():
    from hyper_amd import block8
    x = torch.zeros(2, 0, 30, device='cuda', requires_grad=True)
    W = torch.ones(2, 5, 30, device='cuda', requires_grad=True)
    b = torch.ones(2, 5, device='cuda', requires_grad=True)
    y = block8.linear(x, W, b)
    dx, dW, db = torch.autograd.grad(y, (x, W, b), torch.zeros(2, 0, 5, device='cuda'))
    assert y.shape == (2, 0, 5) and dx.shape == x.shape and not dW.any() and not db.any()
    assert block8.linear(x.detach(), block8.quantize_weight(W), b.detach()).shape == (2, 0, 5)


@gpu
def test_same_bits_on_another_stream_and_in_two_graphs():
    from hyper_amd import block8
    from hyper_amd.net.activation import checkpointed
    x = features((2, 300, 500), torch.float32, 1).cuda().requires_grad_(True)
    W = features((2, 130, 500), torch.float32, 2).cuda().requires_grad_(True)
    b = torch.randn(2, 130, device='cuda', requires_grad=True)
    dy = features((2, 300, 130), torch.float32, 3).cuda()

    def step():
        y = block8.linear(checkpointed('gelu', x), W, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, W, b), dy)
    first = step()
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
            x.copy_(features((2, 300, 500), torch.float32, 30 + k))
        for g in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(p, q) for p, q in zip(want, o)), 'replay %d' % k


# --------------------------------------------------------------------------------------------------------------- refusals
def test_refusals_without_a_gpu():
    from hyper_amd import _lib, block8
    from hyper_amd.net.activation import checkpointed
    for call in (lambda: block8.quantize(torch.randn(2, 3)), lambda: checkpointed('gelu', torch.randn(3)),
                 lambda: block8.quantize_weight(torch.randn(1, 2, 3)), lambda: block8.linear(torch.randn(1, 2, 3), torch.randn(1, 2, 3))):
        with pytest.raises(RuntimeError, match='GPU'):
            call()
    with pytest.raises(ValueError):
        checkpointed('relu', torch.randn(3))
    with pytest.raises(TypeError):
        block8.quantize([1.0])
    L, p, odd = _lib.lib(), 4096, 4097
    assert L.hecka_block8_quantize(p, 9, 1, 8, 8, 0, p, p, None, None) == -1
    assert L.hecka_block8_quantize(p, 0, 1, 8, 7, 0, p, p, None, None) == -1
    assert L.hecka_block8_quantize(p, 0, 1, 8, 8, 1, p, p, None, None) == -1
    assert L.hecka_block8_quantize(p, 0, 1, 8, 8, 6, p, p, p, None) == -1
    assert L.hecka_block8_quantize(p, 0, 1, 8, 8, 0, odd, p, None, None) == -1
    assert L.hecka_block8_quantize(p, 0, 1, 8, 8, 0, None, None, None, None) == -1
    assert L.hecka_block8_quantize(p, 0, 1, 8, 8, 1, p, None, p, None) == -1
    assert L.hecka_block8_values(p, p, None, 0, 1, 8, 1, p, None) == -1
    assert L.hecka_block8_values(p, p, None, 0, 0, 8, 0, p, None) == -1
    assert L.hecka_block8_weight(p, 0, 1, 8, 8, 64, p, p, p, None, None) == -1
    assert L.hecka_block8_weight(p, 0, 2, 8, 8, 63, p, p, None, None, None) == -1
    assert L.hecka_block8_weight(p, 0, 0, 8, 8, 64, p, p, None, None, None) == -1
    assert L.hecka_block8_linear(p, p, 2, p, p, 3, 8, 8, 8, None, 0, 1.0, 0.0, p, 0, 3, None, 0, None) == -1
    assert L.hecka_block8_linear(p, p, 1, p, p, 1, 8, 8, (1 << 22) + 1, None, 0, 1.0, 0.0, p, 0, 1, None, 0, None) == -1
    assert L.hecka_block8_linear(odd, p, 1, p, p, 1, 8, 8, 8, None, 0, 1.0, 0.0, p, 0, 1, None, 0, None) == -1
    assert L.hecka_block8_linear(p, p, 1, p, p, 3, 8, 8, 8, None, 0, 1.0, 0.0, p, 0, 2, None, 0, None) == -1      # a sum over some members
    assert L.hecka_block8_linear(p, p, 1, p, p, 3, 8, 8, 8, p, 8, 1.0, 1.0, p, 0, 1, None, 0, None) == -1         # a sum with a bias
    need = L.hecka_block8_linear_workspace_bytes(1, 64, 1024, 8192, 1, 0)
    assert need > 0 and need % (64 * 1024 * 4) == 0                                                               # slabs of a split K
    assert L.hecka_block8_linear(p, p, 1, p, p, 1, 64, 1024, 8192, None, 0, 1.0, 0.0, p, 0, 1, p, need - 1, None) == -3
    assert L.hecka_block8_linear_workspace_bytes(3, 8, 8, 8, 1, 1) == 3 * 64 * 4 and L.hecka_block8_linear_workspace_bytes(3, 8, 8, 8, 3, 2) == 0
    assert L.hecka_block8_linear_token(p, 0, 1, p, p, 1, 17, 8, 8, None, 0, 1.0, 0.0, p, None) == -1
    assert L.hecka_block8_wgrad(p, 0, p, p, 1, 1, 5000, 8, 8, 1.0, 1.0, p, p, None, 0, None) == -3
    assert L.hecka_block8_wgrad_workspace_bytes(1, 0, 8, 8) == 0
    assert L.hecka_block8_train_bytes(0, 2, 3, 8, 8, 8, 0, 1, 1) == 0 and L.hecka_block8_train_bytes(0, 2, 2, 8, 8, 8, 0, 0, 0) == 0
    kept, ws = (L.hecka_block8_train_bytes(i, 2, 2, 8, 8, 8, 0, 1, 1) for i in (0, 1))
    fwd = lambda xm=2, k=kept, n=ws: L.hecka_block8_train_fwd(p, 0, xm, 8, p, 0, 64, 2, 8, 8, 8, None, 0, 1.0, 0.0, 1, 1, p, p, k, p, n, None)   # noqa: E731
    assert fwd(xm=3) == -1 and fwd(k=kept - 1) == -3 and fwd(n=ws - 1) == -3
    bwd = lambda dx, dw, db, need=1, k=kept, n=1 << 30: L.hecka_block8_train_bwd(p, 0, 2, 2, 8, 8, 8, 1.0, 0.0, need, need, p, k, dx, dw, db, p, n, None)   # noqa: E731
    assert bwd(p, None, None, need=0) == -1 and bwd(None, None, p) == -1 and bwd(p, p, p, k=kept - 1) == -3 and bwd(p, p, p, n=0) == -3


@gpu
def test_refusals_on_the_gpu():
    from hyper_amd import block8
    x, W = torch.randn(2, 5, 30, device='cuda'), torch.randn(2, 7, 30, device='cuda')
    w = block8.quantize_weight(W)
    q = block8.quantize(x)
    bad = [lambda: block8.linear(x[:, :, :29], W), lambda: block8.linear(x[:1], W), lambda: block8.linear(x, w, torch.zeros(2, 8, device='cuda')),
           lambda: block8.linear(x, W, torch.zeros(2, 7, device='cuda', dtype=torch.float16)), lambda: block8.linear(x, W[0]),
           lambda: block8.weight_grad(torch.zeros(2, 6, 7, device='cuda'), q), lambda: block8.weight_grad(torch.zeros(3, 5, 7, device='cuda'), q),
           lambda: block8.quantize(torch.zeros(3, 0, device='cuda')), lambda: block8.quantize_weight(torch.zeros(1, 0, 3, device='cuda')),
           lambda: block8.Weight8(w.codes, w.scales, 300), lambda: block8.Weight8(w.codes, w.scales[:, :, :1], 30),
           lambda: block8.Weight8(w.codes.float(), w.scales, 30),
           lambda: block8.Rows8(q.codes, q.scales, (2, 6, 30), torch.float32), lambda: block8.Rows8(q.codes[:, :64], q.scales, (2, 5, 30), torch.float32),
           lambda: block8.Rows8(q.codes, q.scales.cpu(), (2, 5, 30), torch.float32), lambda: block8.Rows8(q.codes, q.scales, (2, 5, 30), torch.float64), lambda: block8.Weight8(w.codes, w.scales, 30, w.codes_t)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: block8.quantize(x.double()), lambda: block8.linear(x.double(), W), lambda: block8.dequantize(q, torch.float64),
                 lambda: block8.dequantize(x), lambda: block8.weight_grad(torch.zeros(2, 5, 7, device='cuda'), x)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError, match='serve'):
        block8.linear(x.clone().requires_grad_(True), w)
    with pytest.raises(RuntimeError):
        block8.linear(x, w, torch.zeros(2, 7))
    xg = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(block8.linear(xg, W).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
