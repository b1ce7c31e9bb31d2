"""8-bit blocks where a looser look would miss a fault: every 16-bit value as a block's largest, results past fp16's range, every part of the gradients
against the whole step, far results of either sign."""
import math

import pytest
import torch

from test_block8 import HALF, TYPES, U, blocks, exponent, features, same, whole

gpu = pytest.mark.gpu


def largest_of_blocks(dtype):
    """[n, 256]: row i's two blocks have the i-th positive value v of `dtype` as their largest (fp32: four values a binade).  The first holds parts of v
    down to 2^-20 of it, the second every midpoint of two codes at v's scale."""
    if dtype == torch.float32:
        v = torch.tensor([min(math.ldexp(m, e), 3.4028234e38) for e in range(-149, 128) for m in (1.0, 1.75, 1.7500001, 1.9999999)], dtype=torch.float32)
    else:
        v = torch.arange(1, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    gen = torch.Generator().manual_seed(1)
    d = v.double()[:, None]
    parts = d * torch.ldexp(torch.rand((len(v), 128), generator=gen, dtype=torch.float64) * 2 - 1, torch.randint(-20, 1, (len(v), 128), generator=gen))
    parts[:, :4] = torch.cat([d, -d / 3, d / 300, -d], 1)
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2 * torch.where(torch.arange(126) % 2 == 0, 1.0, -1.0)
    q = torch.tensor([exponent(float(a)) for a in v])
    ties = torch.cat([d, -d, mid * torch.ldexp(torch.ones(1, dtype=torch.float64), q)[:, None]], 1)
    top = torch.finfo(dtype).max
    return torch.cat([parts, ties], 1).clamp(-top, top).to(dtype)


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_every_largest_value(dtype):
    """Codes, scales and values bit for bit the definition's, subnormal blocks among them; the codes that the serving kernel makes by itself too."""
    from hyper_amd import block8
    x = largest_of_blocks(dtype)
    q = block8.quantize(x.cuda())
    val, byte = blocks(x[None], 1, 128)
    assert torch.equal(q.scales.cpu()[:, :2], byte[0])
    got = q.codes.cpu().view(torch.float8_e4m3fn).double().view(-1, 2, 128) * torch.ldexp(torch.ones((), dtype=torch.float64), byte[0].int() - 127)[..., None]
    assert same(got.view(-1, 256), val[0])
    for t in TYPES:
        want = val[0].to(t) if t != torch.float16 else val[0].float().half()
        if t == torch.float16:      # 65536 comes back as what fp16 holds
            want = torch.where(val[0].abs() == 65536.0, torch.sign(val[0]) * 65504.0, val[0]).half()
        assert same(block8.dequantize(q, t).cpu(), want), t
    w = block8.quantize_weight(torch.ones(1, 1, 256, device='cuda'), transposed=False)
    scale = 2.0 ** -12
    small = x[x[:, 0].double() < 1e35]      # no sum of 256 passes fp32
    for at in range(0, len(small), 4001):      # sixteen rows at a time by the kernel that makes its codes, and by the one that takes them: sums in another order
        rows = small[at:at + 16].cuda()
        a, b = block8.linear(rows, w, scale=scale).double(), block8.linear(block8.quantize(rows), w, scale=scale).double()
        mags = rows.double().abs().sum(1)[None, :, None] * scale
        tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
        assert bool(((a - b).abs() <= 300 * U * mags + 2 * HALF[dtype] * a.abs() + tiny).all())


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(3, 250), (130, 40)])
def test_every_largest_value_of_a_weight(rows, cols, dtype):
    from hyper_amd import block8
    v = largest_of_blocks(dtype)
    v = v[::max(1, len(v) // 150)]
    W = v[:, :1].double()[:, None] * torch.empty(len(v), rows, cols, dtype=torch.float64).uniform_(-1, 1, generator=torch.Generator().manual_seed(2))
    W[:, rows - 1, cols - 1] = v[:, 0].double()
    W = W.to(dtype)
    w = block8.quantize_weight(W.cuda())
    val, byte = blocks(W, 128, 128)
    nb = byte.shape[-1]
    assert torch.equal(w.scales.cpu()[..., :nb], byte)
    s = torch.ldexp(torch.ones((), dtype=torch.float64), byte.int() - 127).repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)[..., :cols]
    assert same(w.codes.cpu().view(torch.float8_e4m3fn).double()[..., :cols] * s, val)


@gpu
@pytest.mark.parametrize('products', ['exact', 'fp8'])
def test_what_passes_the_range_of_fp16_is_infinite_and_nothing_else(products):
    """A result is an infinity only where the value and its bound reach 65520, halfway to the step past the last number, of that sign; never NaN."""
    from hyper_amd import block8
    M, N, O, I = 2, 150, 140, 700
    x, W, dy = features((M, N, I), torch.float16, 1), features((M, O, I), torch.float32, 2), features((M, N, O), torch.float16, 3)
    xg, Wg = x.cuda().requires_grad_(True), W.cuda()
    y = block8.linear(xg, Wg, products=products)
    dx, = torch.autograd.grad(y, xg, dy.cuda())
    x8, w8, dy8 = blocks(x, 1, 128)[0], blocks(W, 128, 128)[0], blocks(dy, 1, 128)[0]
    wt = w8.transpose(1, 2).contiguous()
    for got, p, q, K in ((y.detach(), x8, wt, I), (dx, dy8, w8, O), (block8.linear(x.cuda()[:, :16], block8.quantize_weight(Wg)), x8[:, :16], wt, I)):
        got, want, mags = got.cpu().double(), torch.bmm(p, q), torch.bmm(p.abs(), q.abs())
        tol = U * (3 * K / 32 + 40) * mags + 4 * U * want.abs() + (7 * 2.0 ** -13 * mags if products == 'fp8' else 0.0)
        infinite = torch.isinf(got)
        assert bool(infinite.any()) and not bool(got.isnan().any())
        assert bool((want[infinite] * torch.sign(got[infinite]) + tol[infinite] >= 65520).all())
        fine = ~infinite
        assert bool((want[fine].abs() - tol[fine] <= 65520).all())
        t = tol[fine] + HALF[torch.float16] * (want[fine].abs() + tol[fine]) + 2.0 ** -25
        assert bool(((got[fine] - want[fine]).abs() <= t).all())


@gpu
@pytest.mark.parametrize('dtype,products', [(t, 'exact') for t in TYPES] + [(t, 'fp8') for t in TYPES[1:]], ids=str)
def test_parts_of_the_gradients_are_the_whole_steps(dtype, products):
    """Each choice of what requires a gradient and of what is asked for, against the step in which everything is."""
    from hyper_amd import block8
    for M, N, O, I in ((2, 21, 30, 140), (1, 700, 261, 130)):
        x0, W0, b0, dy = features((M, N, I), dtype, 1).cuda(), torch.randn(M, O, I, device='cuda'), torch.randn(M, O, device='cuda'), features((M, N, O), dtype, 2).cuda()
        for shared in (False, True):
            def step(need):
                t = [v.detach().clone().requires_grad_(bool(need >> i & 1)) for i, v in enumerate((x0[0] if shared else x0, W0, b0))]
                return t, block8.linear(*t, scale=0.5, bias_scale=0.25, products=products)
            t, y = step(7)
            full = torch.autograd.grad(y, t, dy)
            assert all(bool((g != 0).any()) for g in full)
            for need in range(1, 8):
                t, z = step(need)
                assert torch.equal(z, y)
                for ask in range(1, 8):
                    if not ask & ~need:
                        got = torch.autograd.grad(z, [v for i, v in enumerate(t) if ask >> i & 1], dy, retain_graph=True)
                        assert all(torch.equal(p, q) for p, q in zip(got, [g for i, g in enumerate(full) if ask >> i & 1])), (shared, need, ask)


@gpu
@pytest.mark.parametrize('products', ['exact', 'fp8'])
def test_far_results_of_either_sign(products):
    """A result of more than 2^31 elements: nothing but zeros in front of its last rows, below or above."""
    from hyper_amd import block8
    N, O, I, n = 140000, 16384, 40, 5
    x, W = -whole((1, n, I), 1).abs().bfloat16().cuda(), whole((1, O, I), 2).abs().cuda()
    big = torch.zeros(1, N, I, device='cuda', dtype=torch.bfloat16)
    big[:, -n:] = x
    with torch.no_grad():
        y, want = block8.linear(big, W, products=products), block8.linear(x, W, products=products)
    assert y.numel() > 2 ** 31 and torch.equal(y[:, -n:], want) and bool((want < 0).any())
    assert float(y[:, :-n].amax()) == 0 and float(y[:, :-n].amin()) == 0
