"""block8.linear's products: exact unless the caller asks for the fp8 matrix instruction, which has to pass what the exact ones pass."""
import pytest
import torch

import test_block8 as base
from test_block8 import HALF, TYPES, U, blocks, features

gpu = pytest.mark.gpu
TYPES16 = TYPES[1:]


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(1, 200, 150, 1100), (3, 300, 784, 513), (1, 40, 130, 5000), (20, 300, 520, 900)])
def test_products_are_added_in_fp32(M, N, O, I, dtype):
    """All types: each of the K / 32 instructions, the 32 sums inside one and the joins of shared-out sums round by u of the sum of
    magnitudes at most; then one rounding to the result's type."""
    from hyper_amd import block8
    x, W, dy = features((M, N, I), dtype, 1), features((M, O, I), torch.float32, 2), features((M, N, O), dtype, 3)
    if dtype == torch.float16:
        x, dy = x.clamp(-30, 30), dy.clamp(-30, 30)
    xg, Wg = x.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    y = block8.linear(xg, Wg, scale=2.0 ** -8)
    dx, = torch.autograd.grad(y, xg, dy.cuda())
    x8, w8, dy8 = blocks(x, 1, 128)[0], blocks(W, 128, 128)[0], blocks(dy, 1, 128)[0]
    tr = lambda t: t.transpose(1, 2).contiguous()   # noqa: E731
    served = block8.linear(x.cuda(), block8.quantize_weight(W.cuda(), transposed=False), scale=2.0 ** -8)
    for name, p, q, got, K in (('y', x8, tr(w8), y.detach(), I), ('dx', dy8, w8, dx, O), ('served', x8, tr(w8), served, I)):
        want, mags = 2.0 ** -8 * torch.bmm(p, q), 2.0 ** -8 * torch.bmm(p.abs(), q.abs())
        tol = U * (3 * K / 32 + 40) * mags + 4 * U * want.abs()
        tol = tol + HALF[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        over = (got.cpu().double() - want).abs() - tol
        assert bool((over <= 0).all()), (name, float(over.max()))


@pytest.fixture
def fp8(monkeypatch):
    from hyper_amd import block8
    exact = block8.linear
    monkeypatch.setattr(block8, 'linear', lambda x, *args, **kw: exact(x, *args, **dict(kw, products='fp8' if x.dtype in TYPES16 else 'exact')))


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
@pytest.mark.parametrize('M,N,O,I', base.SHAPES)
def test_fp8_whole_numbers(M, N, O, I, dtype, fp8):
    base.test_whole_numbers_come_out_exact(M, N, O, I, dtype)


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(2, 3, 70, 300), (1, 200, 150, 1100), (3, 300, 784, 513), (1, 1030, 20, 40)])
def test_fp8_random_values(M, N, O, I, dtype, fp8):
    base.test_random_values_within_counted_roundings(M, N, O, I, dtype)


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
@pytest.mark.parametrize('shared', [False, True])
@pytest.mark.parametrize('M,N,O,I', [(30, 400, 1000, 300), (30, 400, 300, 1000)])
def test_fp8_large_tiles(M, N, O, I, shared, dtype, fp8):
    base.test_large_tiles_with_ragged_edges(M, N, O, I, shared, dtype)


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(1, 64, 130, 5000), (2, 33, 71, 2100), (1, 17, 3, 8200), (1, 300, 8, 2048)])
def test_fp8_long_sums(M, N, O, I, dtype, fp8):
    base.test_long_sums_shared_out(M, N, O, I, dtype)


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(3, 40, 50, 201), (2, 33, 4099, 35), (7, 1, 1, 1), (40, 700, 300, 129)])
def test_fp8_shared_rows(M, N, O, I, dtype, fp8):
    base.test_gradient_of_shared_rows_is_rounded_once(M, N, O, I, dtype)


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
def test_fp8_any_part_and_bad_values(dtype, fp8):
    base.test_any_part_of_the_gradients(dtype)
    base.test_without_gradients_the_same_results_and_nothing_kept(dtype)
    base.test_not_a_number_reaches_its_row_and_column_only()
    base.test_far_outputs_and_far_weights() if dtype == torch.bfloat16 else None


@gpu
@pytest.mark.parametrize('dtype', TYPES16, ids=str)
def test_fp8_in_a_graph(dtype):
    """The training step through the layer, eager and replayed; both products from the same codes."""
    from hyper_amd.generators.ensemble import FixedEnsembleModel
    from hyper_amd.layers import Linear, SequentialModule
    torch.manual_seed(0)
    model = FixedEnsembleModel(SequentialModule(modules=[Linear(300, 200, act='silu', compute='fp8', checkpoint='e4m3')]), 2).cuda()
    x, dy = torch.randn(2, 90, 300, device='cuda').to(dtype).requires_grad_(True), torch.randn(2, 90, 200, device='cuda').to(dtype)

    def step():
        y = model(model.forward_params(model.sample_params([0, 1], device=x.device)), x)[1]
        return [y.detach()] + list(torch.autograd.grad(y, [x] + list(model.parameters()), dy))
    first = step()
    exact = block8_step(model, x, dy)
    assert all(float((a.double() - b.double()).norm() / b.double().norm()) <= 2.0 ** -7 for a, b in zip(first, exact))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(2, 90, 300, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, want)), k


def block8_step(model, x, dy):
    layer = list(model.target._modules.values())[0]
    layer.compute = 'e4m3'
    try:
        y = model(model.forward_params(model.sample_params([0, 1], device=x.device)), x)[1]
        return [y.detach()] + list(torch.autograd.grad(y, [x] + list(model.parameters()), dy))
    finally:
        layer.compute = 'fp8'


def test_refusals_without_a_gpu():
    from hyper_amd import _lib, block8
    from hyper_amd.layers import Linear
    assert Linear(3, 4, compute='fp8').compute == 'fp8'
    with pytest.raises(ValueError):
        Linear(3, 4, compute='bf16')
    for products, dtype in (('fp8', torch.float32), ('fp16', torch.bfloat16), (None, torch.bfloat16)):
        with pytest.raises(ValueError):
            block8._products('block8.linear', products, dtype)
    L, p = _lib.lib(), 4096
    for bad in (0x100, 0x103, 0x201, -1):      # fp32 has exact products only
        assert L.hecka_block8_linear(p, p, 1, p, p, 1, 8, 8, 8, None, 0, 1.0, 0.0, p, bad, 1, None, 0, None) == -1
        assert L.hecka_block8_train_bytes(0, 2, 2, 8, 8, 8, bad, 1, 1) == 0
        assert L.hecka_block8_train_fwd(p, bad, 2, 8, p, 0, 64, 2, 8, 8, 8, None, 0, 1.0, 0.0, 1, 1, p, p, 1 << 20, p, 1 << 20, None) == -1
        assert L.hecka_block8_train_bwd(p, bad, 2, 2, 8, 8, 8, 1.0, 0.0, 1, 1, p, 1 << 20, p, None, None, p, 1 << 20, None) == -1
    assert L.hecka_block8_quantize(p, 0x101, 1, 8, 8, 0, p, p, None, None) == -1 and L.hecka_block8_wgrad(p, 0x101, p, p, 1, 1, 8, 8, 8, 1.0, 1.0, p, p, p, 1 << 20, None) == -1
    assert L.hecka_block8_train_bytes(0, 2, 2, 8, 8, 8, 0x101, 1, 1) == L.hecka_block8_train_bytes(0, 2, 2, 8, 8, 8, 1, 1, 1) > 0


@gpu
def test_refusals_on_the_gpu():
    from hyper_amd import block8
    x, W = torch.randn(1, 20, 30, device='cuda'), torch.randn(1, 7, 30, device='cuda')
    w = block8.quantize_weight(W, transposed=False)
    for call in (lambda: block8.linear(x, W, products='fp8'), lambda: block8.linear(x, w, products='fp8'), lambda: block8.linear(x[:, :3], w, products='fp8'),
                 lambda: block8.linear(block8.quantize(x), w, products='fp8'), lambda: block8.linear(x.half(), W, products='e4m3')):
        with pytest.raises(ValueError):
            call()


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_transposed_codes_multiply_with_the_weights_themselves(dtype):
    """quantize_weight's codes_t as a Weight8: the product that the input gradient is, bit for bit; without them half of the bytes."""
    from hyper_amd import block8
    for M, N, O, I in ((2, 40, 300, 140), (2, 3, 300, 140)):
        x, W, dy = features((M, N, I), dtype, 1).cuda().requires_grad_(True), torch.randn(M, O, I, device='cuda'), features((M, N, O), dtype, 2).cuda()
        dx, = torch.autograd.grad(block8.linear(x, W, scale=0.5), x, dy)
        w = block8.quantize_weight(W)
        back = block8.Weight8(w.codes_t, w.scales_t, w.outputs)
        assert torch.equal(block8.linear(block8.quantize(dy), back, scale=0.5), dx)
        alone = block8.quantize_weight(W, transposed=False)
        assert alone.codes_t is None and alone.scales_t is None and alone.nbytes() == w.codes.numel() + w.scales.numel()
