"""Every kernel that block8's products choose between, compared with exact values where its loops are in full swing: many blocks of K, many rows.

The rules of choice (csrc/hecka_block8_gemm.hip: linear_plan, linear_run, token_run, wgrad_plan) are restated here, and each test says which kernel its
sizes are meant to reach: a rule that changes has to bring its sizes along.  Operands are whole numbers up to 2, times a power of two from 1 to 8 for every
row and block of 128 (128 x 128 of a weight): a scale of another row or block gives other results, and all sums are exact - at most 2^14
products up to 2^2 of 2^0 to 2^6, so 22 bits."""
import pytest
import torch

from test_block8 import TYPES

gpu = pytest.mark.gpu


def cdiv(a, b):
    return -(-a // b)


def large_rounds(M, R, C):
    return cdiv(M * cdiv(R, 256) * cdiv(C, 256), 256)


def linear_kernel(M, N, O, K, fp8):
    """(tile, blocks of K for each workgroup, workgroups that share K, steps ahead) of results [M, N, O]."""
    nblk, tiles = cdiv(K, 128), M * cdiv(N, 128) * cdiv(O, 128)
    if large_rounds(M, N, O) * (512 if fp8 else 900) <= tiles:
        return 256, cdiv(nblk, 4) * 4, 1, 1
    splits, share = 1, cdiv(nblk, 4) * 4
    if 256 // tiles > 1:
        splits = min(256 // tiles, max(1, nblk // 8))
        share = cdiv(cdiv(nblk, splits), 4) * 4
        splits = cdiv(nblk, share)
    return 128, share, splits, 3 if fp8 and share >= 16 and tiles * splits <= 256 else 1


def token_kernel(M, O, K):
    """(16-row tiles of a wave, waves of a workgroup)."""
    rows16, nblk = M * cdiv(O, 16), cdiv(K, 128)
    if rows16 >= 512:
        return (2, 4) if rows16 >= 1024 or nblk < 16 else (2, 8)
    if rows16 >= 128:
        return (1, 4) if nblk < 16 else (1, 8)
    return (1, 4) if nblk <= 4 else (1, 8) if nblk < 32 else (1, 16)


def wgrad_kernel(M, N, O, I, dtype):
    """(tile, workgroups that share the rows, whole 16-byte pieces of dy)."""
    whole = O % (4 if dtype == torch.float32 else 8) == 0
    tiles = M * cdiv(O, 128) * cdiv(I, 128)
    if whole and large_rounds(M, O, I) * 700 <= tiles:
        return 256, 1, whole
    splits = min(1 if tiles >= 512 else 512 // tiles, cdiv(N, 256))
    return 128, cdiv(N, cdiv(cdiv(N, splits), 64) * 64), whole


def scaled(shape, seed, blocks):
    """Whole numbers of [-2, 2] times 2^0 .. 2^3, another for each of `blocks` (block of the rows, of the columns)."""
    gen = torch.Generator().manual_seed(seed)
    G, R, C = shape
    v = torch.randint(-2, 3, shape, generator=gen).float()
    e = torch.randint(0, 4, (G, cdiv(R, blocks[0]), cdiv(C, blocks[1])), generator=gen)
    return v * torch.ldexp(torch.ones(()), e).repeat_interleave(blocks[0], 1)[:, :R].repeat_interleave(blocks[1], 2)[..., :C]


def t(a):
    return a.transpose(1, 2).contiguous()


def check(M, N, O, I, dtype, products, train=True):
    from hyper_amd import block8
    x, W, b = scaled((M, N, I), 1, (1, 128)), scaled((M, O, I), 2, (128, 128)), torch.randint(-9, 10, (M, O)).float()
    want = 0.25 * torch.bmm(x, t(W)) + 2.0 * b[:, None]      # exact in fp32
    xg, Wg, bg = x.to(dtype).cuda(), W.cuda(), b.cuda()
    q, w = block8.quantize(xg), block8.quantize_weight(Wg, transposed=False)
    assert len(q.scales[:, 0].unique()) >= min(4, M * N) // 2      # there are scales to mix up
    assert torch.equal(block8.linear(q, w, bg, 0.25, 2.0, products).cpu(), want.to(dtype)), 'served'
    if not train:
        return
    dy = scaled((M, N, O), 3, (1, 128))
    for v in (xg, Wg, bg):
        v.requires_grad_(True)
    y = block8.linear(xg, Wg, bg, 0.25, 2.0, products)
    assert torch.equal(y.detach().cpu(), want.to(dtype)), 'y'
    dx, dW, db = torch.autograd.grad(y, (xg, Wg, bg), dy.to(dtype).cuda())
    assert torch.equal(dx.cpu(), (0.25 * torch.bmm(dy, W)).to(dtype)), 'dx'
    assert torch.equal(dW.cpu(), 0.25 * torch.bmm(t(dy), x)), 'dW'
    assert torch.equal(db.cpu(), 2.0 * dy.sum(1)), 'db'


ALL = [(d, 'exact') for d in TYPES] + [(d, 'fp8') for d in TYPES[1:]]


# blocks of K: an odd number, one past a multiple of four and eight, one more than a share holds, a last share of one block
@gpu
@pytest.mark.parametrize('dtype', TYPES[1:], ids=str)
@pytest.mark.parametrize('M,N,O,I,shares', [(1, 1000, 2100, 2100, 1), (1, 1000, 2100, 4100, 1), (2, 900, 1900, 2300, 1), (1, 1000, 2100, 2432, 1), (1, 64, 8192, 8192, 4),
                                             (1, 64, 8192, 6200, 4), (1, 100, 8100, 8300, 4)])
def test_three_steps_ahead(M, N, O, I, shares, dtype):
    tile, share, splits, ahead = linear_kernel(M, N, O, I, True)
    assert (tile, splits, ahead) == (128, shares, 3)
    check(M, N, O, I, dtype, 'fp8', train=False)


@gpu
@pytest.mark.parametrize('dtype,products', ALL, ids=str)
@pytest.mark.parametrize('M,N,O,I,dx', [(18, 500, 1656, 1600, 256), (20, 400, 1504, 1530, 256), (30, 400, 1000, 2200, None), (30, 400, 1000, 1152, None)])
def test_large_tiles_over_many_blocks(M, N, O, I, dx, dtype, products):
    """256 x 256 tiles: the second and third dword of scales, their slots used again, odd and even numbers of blocks; dW's over many rows."""
    assert linear_kernel(M, N, O, I, products == 'fp8')[0] == 256 and cdiv(I, 128) >= 8
    assert dx is None or linear_kernel(M, N, I, O, products == 'fp8')[0] == dx
    assert wgrad_kernel(M, N, O, I, dtype)[0] == 256
    check(M, N, O, I, dtype, products)


@gpu
@pytest.mark.parametrize('dtype,products', ALL, ids=str)
@pytest.mark.parametrize('M,N,O,I', [(2, 300, 1000, 1300), (7, 300, 520, 2200), (1, 513, 2052, 1100), (1, 77, 4100, 5000)])
def test_small_tiles_over_many_blocks(M, N, O, I, dtype, products):
    assert linear_kernel(M, N, O, I, products == 'fp8')[0] == 128 and cdiv(I, 128) >= 8
    check(M, N, O, I, dtype, products)


TOKENS = [(3, 3001, 2100, (2, 8)), (5, 4099, 300, (2, 4)), (3, 3001, 700, (2, 4)), (2, 8200, 2600, (2, 4)), (2, 1101, 2100, (1, 8)), (2, 1101, 700, (1, 4)), (1, 70, 400, (1, 4)),
          (1, 70, 1300, (1, 8)), (1, 300, 5000, (1, 16))]


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,O,I,kernel', TOKENS)
def test_token_kernels(M, O, I, kernel, dtype):
    from hyper_amd import block8
    assert token_kernel(M, O, I) == kernel
    W, b = scaled((M, O, I), 2, (128, 128)), torch.randint(-9, 10, (M, O)).float()
    w = block8.quantize_weight(W.cuda(), transposed=False)
    for N in (1, 5, 16):
        x = scaled((M, N, I), N, (1, 128))
        want = (0.25 * torch.bmm(x, t(W)) + 2.0 * b[:, None]).to(dtype)
        assert torch.equal(block8.linear(x.to(dtype).cuda(), w, b.cuda(), 0.25, 2.0).cpu(), want), N
        want = (0.25 * torch.bmm(x[:1].expand(M, N, I), t(W))).to(dtype)
        assert torch.equal(block8.linear(x[0].to(dtype).cuda(), w, scale=0.25).cpu(), want), 'shared, %d' % N
        if dtype != torch.float32:
            assert torch.equal(block8.linear(x[0].to(dtype).cuda(), w, scale=0.25, products='fp8').cpu(), want)


@gpu
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('M,N,O,I,kernel', [(3, 1000, 2048, 2048, (256, 1)), (40, 333, 300, 520, (128, 1)), (2, 1500, 264, 264, (128, 6)), (2, 1500, 261, 300, (128, 6)),
                                             (3, 700, 1999, 2000, (128, 1))])
def test_weight_gradient_kernels(M, N, O, I, kernel, dtype):
    """Large tiles, small ones alone and in pieces of the rows, with whole and with ragged rows of dy."""
    from hyper_amd import block8
    tile, splits, whole = wgrad_kernel(M, N, O, I, dtype)
    assert (tile, splits) == kernel and whole == (O % 4 == 0 if dtype == torch.float32 else O % 8 == 0)
    x, dy = scaled((M, N, I), 1, (1, 128)), scaled((M, N, O), 3, (1, 128))
    dW, db = block8.weight_grad(dy.to(dtype).cuda(), block8.quantize(x.to(dtype).cuda()), 0.25, 2.0)
    assert torch.equal(dW.cpu(), 0.25 * torch.bmm(t(dy), x)) and torch.equal(db.cpu(), 2.0 * dy.sum(1))


def test_the_rules_by_their_workspaces():
    """What a workspace's size says of the library's own choice: the numbers of shares of linear_kernel and wgrad_kernel."""
    from hyper_amd import _lib
    L = _lib.lib()
    for M, N, O, I in [(1, 1000, 2100, 2100), (1, 64, 8192, 8192), (1, 64, 8192, 6200), (1, 100, 8100, 8300), (18, 500, 1656, 1600), (30, 400, 1000, 2200), (2, 300, 1000, 1300), (1, 77, 4100, 5000), (7, 300, 520, 2200),
                       (1, 17, 3, 8200), (1, 1, 1, 1), (2, 128, 128, 2048)]:
        for number, fp8 in ((0, False), (1, False), (2, False), (0x101, True), (0x102, True)):
            splits = linear_kernel(M, N, O, I, fp8)[2]
            assert L.hecka_block8_linear_workspace_bytes(M, N, O, I, M, number) == (4 * splits * M * N * O if splits > 1 else 0), (M, N, O, I, number)
        need = max(s * M * O * (I + 1) * 4 if s > 1 else 0 for s in (wgrad_kernel(M, N, o, I, torch.float32)[1] for o in (O, O)))
        assert L.hecka_block8_wgrad_workspace_bytes(M, N, O, I) >= need
