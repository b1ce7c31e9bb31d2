"""The checkpointed activations (net.activation.checkpointed) where they are small: errors relative to the value, against the function in 64 bits.

u = 2^-24.  The exponential is off by 3 u, a reciprocal by 2 u, each product and sum by u.  sigmoid: 3 + 2 + 2 u; silu a product more;
gelu 0.24 u of its polynomial's fit, 10 u of its evaluation (worst of 6e6 arguments in fp32 arithmetic, the reciprocal a unit off either way) and
3 u of the exponential.  16 u for all of them; crater's exponent is a rounded z = sqrt 2 (x + 1), three roundings of it: 3 u |z| more.  Then half a
step of the result's type, and below the normal range (hardware exponentials end at 2^-126) what that range ends with."""
import math

import pytest
import torch

from test_block8 import HALF, TYPES, U, act64, blocks

gpu = pytest.mark.gpu
NAMES = ['gelu', 'silu', 'sigmoid', 'crater']
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def values64(name, x):
    """y in 64 bits without cancellation: erfc, and 1 + tanh z = 2 sigmoid(2 z)."""
    if name == 'crater':
        return 2 * (math.sqrt(0.5) + 0.008274364699) * x * torch.sigmoid(math.sqrt(2.0) * (x + 1))
    return act64(name, x)[0]


def held(name, x, y):
    want, at = values64(name, x.double()), x.double()
    rel = 16 * U + (3 * U * (math.sqrt(2.0) * (at + 1)).abs() if name == 'crater' else 0.0)
    half = HALF[x.dtype]
    over = (y.double() - want).abs() - ((rel + half * (1 + rel)) * want.abs() + TINY[x.dtype])
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
