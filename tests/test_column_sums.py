"""Bias gradients (block8.weight_grad, block8.linear, Linear(checkpoint)) over many rows: as accurate as over few.

A large gradient in the first row and small ones in all others, each below half a step of the large one: a sum that runs down the rows in
fp32 loses every one of them.  u = 2^-24.  The rows of one step (64 at most) are added by at most three matrix instructions, each off by u of the
sum of magnitudes it adds up for its rounding and 32 u for the sums inside it (the large one stands in one step, so that is 99 u times
what the others of that step are worth plus 3 u of the large one); steps and pieces are added exactly but for u of the result and of each of two pieces."""
import pytest
import torch

from test_block8 import TYPES, U

gpu = pytest.mark.gpu
# (M, N, O, I): 512 tiles that are never cut, large tiles, rows cut into pieces, odd widths, one column of tiles (a wave has several of them)
SHAPES = [(4, 8000, 2048, 1024), (8, 6000, 2048, 2048), (1, 9000, 40, 70), (2, 7001, 301, 130), (130, 1500, 256, 256)]


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I', SHAPES)
def test_small_gradients_behind_a_large_one(M, N, O, I, dtype):
    from hyper_amd import block8
    big, small = (2.0 ** 15, 2.0 ** -16) if dtype == torch.float16 else (2.0 ** 30, 2.0 ** -1)
    dy = torch.full((M, N, O), small, dtype=dtype, device='cuda')
    dy[:, 0] = big
    dy[:, :, 1::2] *= -1
    q = block8.quantize(torch.ones(M, N, I, dtype=dtype, device='cuda'))
    dW, db = block8.weight_grad(dy, q, scale=1.0, bias_scale=0.5)
    want = 0.5 * dy[0].double().sum(0)
    assert bool(((db.double() - want).abs() <= 0.5 * (6 * U * big + 99 * U * 64 * small)).all()), float((db.double() - want).abs().max() / want.abs().max() / U)
    again = block8.weight_grad(dy, q, scale=1.0, bias_scale=0.5)
    assert torch.equal(db, again[1]) and torch.equal(dW, again[0])


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_random_rows_to_the_accuracy_of_a_few(dtype):
    """2-norm over 2 x 4096 columns of 20000 rows of mixed sign: a step's sum is off by u / 2 of its own on average, and as many steps as add
    up to the result add up to its error: u, and u for fp16's and fp32's further terms; the last rounding."""
    from hyper_amd import block8
    dy = torch.randn(2, 20000, 4096, generator=torch.Generator('cuda').manual_seed(1), device='cuda').to(dtype)
    _, db = block8.weight_grad(dy, block8.quantize(torch.zeros(2, 20000, 300, dtype=dtype, device='cuda')))
    want = dy.sum(1, dtype=torch.float64)
    assert float((db.double() - want).norm() / want.norm()) <= 3 * U


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_what_is_not_finite_stays_in_its_column(dtype):
    from hyper_amd import block8
    for M, N, O, I in ((1, 700, 130, 40), (4, 700, 2048, 1024)):
        dy = torch.randn(M, N, O, device='cuda').to(dtype)
        q = block8.quantize(torch.randn(M, N, I, device='cuda').to(dtype))
        good = block8.weight_grad(dy, q)[1]
        dy[0, 300, 5], dy[0, 10, 7], dy[0, 20, 7] = float('nan'), float('inf'), float('-inf')
        if dtype == torch.bfloat16:
            dy[0, 699, 9] = float('-inf')      # one term: an infinity is itself
        db = block8.weight_grad(dy, q)[1]
        assert bool(db[0, 5].isnan()) and bool(db[0, 7].isnan())
        keep = torch.ones(M, O, dtype=torch.bool, device='cuda')
        keep[0, 5] = keep[0, 7] = False
        if dtype == torch.bfloat16:
            assert float(db[0, 9]) == float('-inf')
            keep[0, 9] = False
        assert torch.equal(db[keep], good[keep])
