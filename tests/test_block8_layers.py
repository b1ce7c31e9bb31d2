"""The 8-bit and layer-norm layers together, as an ensemble uses them: an MLP of LayerNorm, Linear(compute / checkpoint) and
checkpointed activations against a plain restatement in 64 bits (rounding to 8-bit blocks as an identity in the backward pass)."""
import copy

import pytest
import torch

from test_block8 import act64, blocks

gpu = pytest.mark.gpu
M, N = 3, 37


class Act(torch.autograd.Function):
    """y = act(x), slope at x's 8-bit rows."""

    @staticmethod
    def forward(ctx, x, name):
        ctx.save_for_backward(blocks(x, 1, 128)[0])
        ctx.name = name
        return act64(name, x)[0]

    @staticmethod
    def backward(ctx, g):
        return g * act64(ctx.name, ctx.saved_tensors[0])[1], None


class Linear(torch.autograd.Function):
    """y = s x W^T + t b.  compute: products of rounded operands; else exact products and the weight gradient from rounded x."""

    @staticmethod
    def forward(ctx, x, W, b, s, t, compute):
        x8 = blocks(x, 1, 128)[0]
        w = blocks(W, 128, 128)[0] if compute else W
        ctx.save_for_backward(x8, w)
        ctx.cfg = (s, t, compute)
        return s * torch.bmm(x8 if compute else x, w.transpose(1, 2).contiguous()) + t * b[:, None]

    @staticmethod
    def backward(ctx, g):
        x8, w = ctx.saved_tensors
        s, t, compute = ctx.cfg
        return s * torch.bmm(blocks(g, 1, 128)[0] if compute else g, w), s * torch.bmm(g.transpose(1, 2).contiguous(), x8), t * g.sum(1), None, None, None


CONFIG = {'name': 'mlp', 'activation': 'gelu', 'norm': 'layer_norm', 'layers': [
    {'in': 150, 'out': 200, 'norm': None}, {'in': 200, 'out': 140, 'act': 'silu'}, {'in': 140, 'out': 10, 'last': True, 'compute': 'fp32', 'checkpoint': None}]}


def build(compute, checkpoint):
    from hyper_amd.generators.ensemble import FixedEnsembleModel
    from hyper_amd.layers import build_gen_module
    import hyper_amd.target  # noqa: F401
    torch.manual_seed(0)
    cfg = dict(copy.deepcopy(CONFIG), compute=compute, checkpoint=checkpoint)
    return FixedEnsembleModel(build_gen_module(cfg), M).cuda()


def predict(model, x):
    return model(model.forward_params(model.sample_params(list(range(model.size)), device=x.device)), x)[1]


def restated(model, params, x, compute, checkpoint):
    h = x
    for i, (name, mod) in enumerate(model.target._modules.items()):
        if type(mod).__name__ == 'LayerNorm':
            w, b = params[name + '.affine.self.fixed_parameters.weight'], params[name + '.affine.self.fixed_parameters.bias']
            mu = h.mean(-1, keepdim=True)
            h = (h - mu) / torch.sqrt(((h - mu) ** 2).mean(-1, keepdim=True) + mod.eps) * w[:, None] + b[:, None]
            continue
        W, b = params[name + '.self.fixed_parameters.weight'], params[name + '.self.fixed_parameters.bias']
        if mod.compute == 'e4m3' or mod.checkpoint:
            h = Linear.apply(h, W, b, mod.scale, mod.bias_scale, mod.compute == 'e4m3')
        else:
            h = mod.scale * torch.bmm(h, W.transpose(1, 2).contiguous()) + mod.bias_scale * b[:, None]
        if mod.act is not None:
            h = Act.apply(h, mod.act_name) if mod.checkpoint else act64(mod.act_name, h)[0]
    return h


@gpu
@pytest.mark.parametrize('compute,checkpoint', [('e4m3', None), ('fp32', 'e4m3'), ('e4m3', 'e4m3')])
def test_mlp_of_an_ensemble(compute, checkpoint):
    """Predictions and every parameter's gradient.  The blocks round values that the two sides compute with fp32 differences, about
    1e-6 of themselves: one of 1e5 codes may then fall to the other side of a tie, which moves its value by 2^-3.  Each tensor holds
    under 2e4 codes, so at most a handful move; one in a row of 140 shifts what depends on it by 2^-3 / sqrt(140) of one row in 111."""
    model = build(compute, checkpoint)
    gen = torch.Generator().manual_seed(5)
    x, dy = torch.randn(M, N, 150, generator=gen), torch.randn(M, N, 10, generator=gen)
    named = dict(model.named_parameters())
    pre = 'layer_generators.'
    assert all(k.startswith(pre) for k in named)
    pred = predict(model, x.cuda())
    grads = torch.autograd.grad(pred, list(named.values()), dy.cuda())
    p64 = {k[len(pre):]: v.detach().cpu().double().requires_grad_(True) for k, v in named.items()}
    want = restated(model, p64, x.double(), compute, checkpoint)
    gw = torch.autograd.grad(want, list(p64.values()), dy.double())
    assert float((pred.detach().cpu().double() - want.detach()).norm() / want.detach().norm()) <= 2e-3
    for (k, _), g, w in zip(named.items(), grads, gw):
        assert float((g.cpu().double() - w).norm() / w.norm()) <= 2e-3, k
    if compute == 'fp32':      # a checkpoint changes no result: predictions are the plain layer's bit for bit but for the activation's own last place
        plain = build('fp32', None)
        assert float((predict(plain, x.cuda()) - pred).detach().abs().max()) <= 1e-5 * float(pred.detach().abs().max())


@gpu
def test_checkpoint_keeps_less():
    """Memory that a forward pass leaves behind for its backward pass: a byte per saved element and layer instead of eight."""
    from hyper_amd.layers.linear import Linear as Layer
    x = torch.randn(2, 512, 1024, device='cuda')
    params = torch.randn(2, 2048 * 1024 + 2048, device='cuda', requires_grad=True)
    kept = {}
    for name, kw in (('plain', {}), ('checkpoint', dict(checkpoint='e4m3'))):
        layer = Layer(1024, 2048, act='gelu', **kw)
        h = x * 1.0
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        _, y = layer({'self': params}, h)
        x_bytes = h.numel() * 4
        del h
        kept[name] = torch.cuda.memory_allocated() - before - y.numel() * 4
        y.sum().backward()
    # plain: the activation's input (4 bytes) stays, and so does x; with checkpoints: 1 byte for each, the fp32 x is free again
    assert kept['plain'] >= 2 * 512 * 2048 * 4 and kept['checkpoint'] <= kept['plain'] - 0.7 * 2 * 512 * 2048 * 4 - 0.7 * x_bytes, kept


@gpu
def test_training_step_in_a_graph_equals_eager():
    model = build('e4m3', 'e4m3')
    named = [p for p in model.parameters()]
    x, dy = torch.randn(M, N, 150, device='cuda'), torch.randn(M, N, 10, device='cuda')

    def step():
        pred = predict(model, x)
        return [pred.detach()] + list(torch.autograd.grad(pred, named, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for k in range(3):
        x.copy_(torch.randn(M, N, 150, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, want)), k


@gpu
def test_16_bit_features_through_the_layers():
    """compute='e4m3' and LayerNorm take bf16 / fp16 features with fp32 parameters; gradients come back in their own types."""
    from hyper_amd.layers import LayerNorm, Linear as Layer, SequentialModule
    from hyper_amd.generators.ensemble import FixedEnsembleModel
    torch.manual_seed(1)
    model = FixedEnsembleModel(SequentialModule(modules=[LayerNorm(96), Layer(96, 64, act='silu', compute='e4m3', checkpoint='e4m3')]), 2).cuda()
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(2, 50, 96, device='cuda', dtype=dtype, requires_grad=True)
        y = predict(model, x)
        assert y.dtype == dtype
        grads = torch.autograd.grad(y.float().square().sum(), [x] + list(model.parameters()))
        assert grads[0].dtype == dtype and all(g.dtype == torch.float32 for g in grads[1:]) and all(bool(torch.isfinite(g).all()) for g in grads)


def test_refusals():
    from hyper_amd.layers import Activation, Linear as Layer, build_gen_module
    import hyper_amd.target  # noqa: F401
    for call in (lambda: Layer(3, 4, compute='int8'), lambda: Layer(3, 4, checkpoint='fp16'), lambda: Activation('relu', checkpoint='e4m3'),
                 lambda: Activation('gelu', checkpoint='int8'), lambda: build_gen_module({'name': 'mlp', 'norm': 'batch', 'layers': [{'in': 3, 'out': 4}, {'in': 4, 'out': 2}]})):
        with pytest.raises(ValueError):
            call()
    mods = list(build_gen_module({'name': 'mlp', 'layers': [{'in': 3, 'out': 4}, {'in': 4, 'out': 2}]})._modules.values())
    assert [type(m).__name__ for m in mods] == ['Linear', 'Linear'] and mods[0].compute == 'fp32' and mods[0].checkpoint is None
