"""The checkpointed activations (net.activation.checkpointed) where they are small: errors relative to the value, against the function in 64 bits.

u = 2^-24.  The exponential is off by 3 u, a reciprocal that one Newton step follows by u, each product by u.  sigmoid: 3 + 1 + 1 u; silu a product
more: 6 u.  gelu: 0.24 u of its polynomial's fit, 10 u of its evaluation (worst of 6e6 arguments in fp32 arithmetic, the reciprocal a unit off either
way) and 3 u of the exponential: 16 u.  crater: sigmoid, two products and a rounded constant, 8 u, and its exponent is a rounded z = sqrt 2 (x + 1),
three roundings of it: 3 u |z| more.  Then half a step of the result's type.  Hardware exponentials below 2^-126 are zero: sigmoid, silu = x
sigmoid, crater = 1.43 x sigmoid and gelu = x Phi, Phi < 0.03 e^(-x^2 / 2) there, lose at most max(1, 1.43 |x|) 2^-126 by that; a result below its type's
normal range is off by half of that range's step."""
import math

import pytest
import torch

from test_block8 import HALF, TYPES, U, act64, blocks

gpu = pytest.mark.gpu
NAMES = ['gelu', 'silu', 'sigmoid', 'crater']
REL = {'gelu': 16 * U, 'silu': 6 * U, 'sigmoid': 5 * U, 'crater': 8 * U}
STEP = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}      # half of the smallest step


def values64(name, x):
    """y in 64 bits without cancellation: erfc, and 1 + tanh z = 2 sigmoid(2 z)."""
    if name == 'crater':
        return 2 * (math.sqrt(0.5) + 0.008274364699) * x * torch.sigmoid(math.sqrt(2.0) * (x + 1))
    return act64(name, x)[0]


def held(name, x, y):
    want, at = values64(name, x.double()), x.double()
    rel = REL[name] + (3 * U * (math.sqrt(2.0) * (at + 1)).abs() if name == 'crater' else 0.0)
    half = HALF[x.dtype]
    lost = torch.clamp(1.43 * at.abs(), min=1.0) * 2.0 ** -126 * (1 + half) + STEP[x.dtype]
    over = (y.double() - want).abs() - ((rel + half * (1 + rel)) * want.abs() + lost)
    assert bool((over <= 0).all()), (name, float(at[over.argmax()]), float(y[over.argmax()]), float(want[over.argmax()]))


@gpu
@pytest.mark.parametrize('name', NAMES)
def test_fp32_is_right_relative_to_the_value(name):
    from hyper_amd.net.activation import checkpointed
    gen = torch.Generator().manual_seed(1)
    x = torch.exp(torch.rand(1 << 18, generator=gen) * math.log(3e4) - math.log(1e3))      # 0.001 .. 30
    x = torch.cat([-x, x, torch.linspace(-15, 15, 1 << 18)]).cuda()
    held(name, x, checkpointed(name, x))
    xg = x.clone().requires_grad_(True)
    assert torch.equal(checkpointed(name, xg).detach(), checkpointed(name, x))


@gpu
def test_the_slope_of_gelu_far_down():
    """dx at x's 8-bit values: Phi + x phi, each good to 16 u of itself; they have opposite signs below zero."""
    from hyper_amd.net.activation import checkpointed
    x = -torch.linspace(0.0, 13.0, 4096).cuda().requires_grad_(True)
    dx, = torch.autograd.grad(checkpointed('gelu', x), x, torch.ones_like(x))
    at = blocks(x.detach().view(1, 32, 128), 1, 128)[0].view(-1)
    below, bell = 0.5 * torch.erfc(-at * math.sqrt(0.5)), at * torch.exp(-0.5 * at * at) / math.sqrt(2 * math.pi)
    assert bool(((dx.cpu().double() - below - bell).abs() <= 16 * U * (below + bell.abs()) + 2.0 ** -126).all())


@gpu
@pytest.mark.parametrize('dtype', TYPES[1:], ids=str)
@pytest.mark.parametrize('name', NAMES)
def test_every_16_bit_value(name, dtype):
    """All finite 16-bit arguments: the exponential's own error is no part of a 16-bit result's either."""
    from hyper_amd.net.activation import checkpointed
    x = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x) & (x.float().abs() < 80)].cuda()
    held(name, x, checkpointed(name, x))


@gpu
@pytest.mark.parametrize('name', ['silu', 'sigmoid'])
def test_above_zero_a_rounding_or_two_and_no_more(name):
    """x > 0: q = e^-x moves 1 / (1 + q) by 3 u q at most; the quotient is rounded once (u, and 2^-40 of its Newton step), silu's product once more."""
    from hyper_amd.net.activation import checkpointed
    x = torch.linspace(0.0, 30.0, 1 << 20).cuda()
    at = x.double()
    off = (checkpointed(name, x).double() - values64(name, at)).abs() / values64(name, at).clamp(min=1e-30)
    assert bool((off <= ((2.0 if name == 'silu' else 1.0) + 3 * torch.exp(-at) + 1e-3) * U).all()), float((off / U).max())


@gpu
@pytest.mark.parametrize('dtype', TYPES[1:], ids=str)
@pytest.mark.parametrize('name', NAMES + ['tanh'])
def test_a_16_bit_result_is_the_fp32_one_rounded(name, dtype):
    """One arithmetic for all types: for every finite 16-bit argument the fp32 result, rounded once - y and, of 8-bit values, the slope."""
    from hyper_amd.net.activation import checkpointed
    x = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)].cuda()
    assert torch.equal(checkpointed(name, x).float().nan_to_num(), checkpointed(name, x.float()).to(dtype).float().nan_to_num())
    s, f = x[x.abs() < 100].requires_grad_(True), x[x.abs() < 100].float().requires_grad_(True)
    g, h = (torch.autograd.grad(checkpointed(name, t), t, torch.ones_like(t))[0] for t in (s, f))
    assert torch.equal(g, h.to(dtype))
