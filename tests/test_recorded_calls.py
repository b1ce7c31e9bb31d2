"""Layer norm, checkpointed activations and block8 under forward-mode gradients and torch.jit.trace: a launch outside of autograd's nodes would
drop the tangent, or leave the recording with its uninitialised result.  The launches themselves are stubbed out: no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture
def launches(monkeypatch):
    """Entry points that were launched; their sizes in bytes are those of the real library."""
    from hyper_amd import _lib, block8
    from hyper_amd.layers import norm
    seen = []
    monkeypatch.setattr(_lib, 'call', lambda name, device, *args: seen.append(name))
    monkeypatch.setattr(block8, '_check', lambda t, what: None)
    monkeypatch.setattr(norm, '_check_layer_norm', lambda x, affine: None)
    return seen


def calls():
    """(name, a call of x [2, 3, 8]) without gradients: what needs no node of its own."""
    from hyper_amd import block8
    from hyper_amd.layers import LayerNorm, layer_norm
    from hyper_amd.net.activation import checkpointed
    W, b, w = torch.randn(2, 5, 8), torch.randn(2, 5), torch.randn(2, 8)
    return [('layer_norm', lambda x: layer_norm(x)), ('layer_norm, members', lambda x: layer_norm(x, w, w)),
            ('LayerNorm', lambda x: LayerNorm(8)({'affine': {'self': torch.randn(2, 16)}}, x)[1]),
            ('checkpointed', lambda x: checkpointed('silu', x)), ('linear', lambda x: block8.linear(x, W, b)), ('linear, shared', lambda x: block8.linear(x[0], W))]


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('case', range(6))
def test_a_tangent_is_refused_and_not_dropped(case, grad, launches):
    name, call = calls()[case]
    x = torch.randn(2, 3, 8)
    with torch.set_grad_enabled(grad):
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match='jvp'):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
            assert call(x).shape[0] == 2      # without a tangent: as ever
        del launches[:]
        assert call(x).shape[0] == 2 and launches


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('case', range(6))
def test_a_trace_launches_again(case, grad, launches):
    name, call = calls()[case]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, torch.randn(2, 3, 8), check_trace=False)
        del launches[:]
        traced(torch.randn(2, 3, 8))
    assert launches, '%s: the recording holds no launch' % name


def test_codes_are_not_recorded(launches):
    from hyper_amd import block8
    u8 = dict(dtype=torch.uint8)
    q = block8.Rows8._made(torch.zeros(6, 128, **u8), torch.zeros(6, 4, **u8), (2, 3, 8), torch.float32)
    w = block8.Weight8._made(torch.zeros(2, 5, 128, **u8), torch.zeros(2, 1, 4, **u8), 8, None, None)
    b = torch.randn(2, 5)
    for call in (lambda x: block8.quantize(x).codes, lambda x: block8.dequantize(q) + x, lambda x: block8.quantize_weight(x).codes,
                 lambda x: block8.weight_grad(x, q)[0], lambda x: block8.linear(x, w), lambda x: block8.linear(q, w, b) + x.sum()):
        with pytest.raises(RuntimeError, match='trace'):
            torch.jit.trace(call, torch.randn(2, 3, 8), check_trace=False)
    with forward_ad.dual_level():
        for dual in (lambda t: block8.linear(forward_ad.make_dual(t, t), w), lambda t: block8.linear(t, w, forward_ad.make_dual(b, b)),
                     lambda t: block8.linear(q, w, forward_ad.make_dual(b, b))):
            with pytest.raises(RuntimeError, match='tangents'):
                dual(torch.randn(2, 3, 8))


@pytest.mark.gpu
def test_traced_calls_on_the_gpu():
    """The recorded functions give the eager results for other inputs than the example's."""
    from hyper_amd import block8
    from hyper_amd.layers import layer_norm
    from hyper_amd.net.activation import checkpointed
    W, b, w = torch.randn(2, 70, 300, device='cuda'), torch.randn(2, 70, device='cuda'), torch.randn(2, 300, device='cuda')
    for call in (lambda x: layer_norm(x, w, w), lambda x: checkpointed('gelu', x), lambda x: block8.linear(x, W, b)):
        with torch.no_grad():
            traced = torch.jit.trace(call, torch.randn(2, 9, 300, device='cuda'), check_trace=False)
            for k in range(2):
                x = torch.randn(2, 9, 300, device='cuda')
                assert torch.equal(traced(x), call(x))
