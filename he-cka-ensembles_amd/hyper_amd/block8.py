"""8-bit blocks: activations and weights kept as e4m3 codes with one power-of-two scale for every 128 elements of a row (128 x 128
of a weight), and the products that work on the codes (libhecka hecka_block8_*; no counterpart in the reference, which is fp32
only).

    q = quantize(x)                          # Rows8: a checkpoint of x in a byte per element
    dequantize(q)                            # the values that it stands for
    w = quantize_weight(W, transposed=False) # Weight8: laid out once by a program that serves
    y = linear(x, w, bias)                   # x (or Rows8) times w^T
    y = linear(x, W, bias)                   # W a float tensor: training - gradients for x, W and bias
    dW, db = weight_grad(dy, q)              # the weight gradient from the checkpoint

A value is off by at most half a step of its code: 2^-4 of itself, or 2^-10 of the block's scale where that is more.
Everything is fp32 / bf16 / fp16 on the GPU; there is no CPU path.  `layers.Linear(compute='e4m3')`, `layers.Linear(
checkpoint='e4m3')` and `layers.Activation(checkpoint='e4m3')` are the layers on top."""
import torch

from . import _lib

BLOCK = 128
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
FP8 = 0x100          # added to a 16-bit type: products by the fp8 matrix instruction
ACTIVATIONS = {'gelu': 1, 'silu': 2, 'tanh': 3, 'sigmoid': 4, 'crater': 5}
_MOST = 1 << 22      # sizes of a product


def row_blocks(K):
    return -(-K // BLOCK)


def scale_stride(K):
    """Scale bytes of a row of K elements: one per block, up to whole dwords."""
    return -(-row_blocks(K) // 4) * 4


def _check(t, what):
    if not torch.is_tensor(t):
        raise TypeError('%s: expected a tensor, got %s' % (what, type(t).__name__))
    if not t.is_cuda:
        raise RuntimeError('%s: needs GPU tensors; there is no CPU path' % what)
    if t.dtype not in DTYPES:
        raise TypeError('%s: float32, bfloat16 or float16, got %s' % (what, t.dtype))


def _not_traced(what):
    """torch.jit.trace records nodes of autograd's only; codes made outside of one would be the example's."""
    if torch._C._is_tracing():
        raise RuntimeError('%s: torch.jit.trace cannot record it' % what)


def _check_rows(q, what):
    if not isinstance(q, Rows8):
        raise TypeError('%s: expected Rows8, got %s' % (what, type(q).__name__))


def _same_device(what, *ts):
    if any(t is not None and t.device != ts[0].device for t in ts):
        raise RuntimeError('%s: tensors on different devices (%s)' % (what, ', '.join(str(t.device) for t in ts if t is not None)))


def _ptr(t):
    return t.data_ptr() if t is not None else None


class Rows8(object):
    """Rows [..., K] in 8-bit blocks: `codes` uint8 [rows, Kp] (Kp = K up to whole blocks), `scales` uint8 [rows, S], the
    shape and dtype of what was put in."""

    def __init__(self, codes, scales, shape, dtype):
        shape = torch.Size(shape)
        if len(shape) < 1 or shape[-1] == 0 or dtype not in DTYPES:
            raise ValueError('Rows8: rows of shape %s, %s' % (tuple(shape), dtype))
        rows = shape.numel() // shape[-1]
        for t, name, width in ((codes, 'codes', row_blocks(shape[-1]) * BLOCK), (scales, 'scales', scale_stride(shape[-1]))):
            if t.dtype != torch.uint8 or tuple(t.shape) != (rows, width) or not t.is_contiguous() or not t.is_cuda or t.device != codes.device:
                raise ValueError('Rows8: %s have to be contiguous uint8 (%d, %d) on one GPU, got %s %s' % (name, rows, width, t.dtype, tuple(t.shape)))
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype

    @classmethod
    def _made(cls, codes, scales, shape, dtype):
        """Of tensors that quantize laid out: nothing to check."""
        q = cls.__new__(cls)
        q.codes, q.scales, q.shape, q.dtype = codes, scales, torch.Size(shape), dtype
        return q

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def dequantize(self, dtype=None):
        return dequantize(self, dtype)


class Weight8(object):
    """Weights [M, O, I] in 8-bit blocks of 128 x 128.  codes [M, O, Ip] (uint8 or float8_e4m3fn, contiguous), scales uint8 [M,
    ceil(O / 128), S(I)]: byte e, 1 to 254, stands for 2^(e - 127).  codes_t [M, I, Op] / scales_t (or None): the same codes transposed, for a
    program that multiplies with W as well as with W^T, by Weight8(w.codes_t, w.scales_t, w.outputs).  linear reads codes and scales alone, and
    its training makes codes of its own."""

    def __init__(self, codes, scales, inputs, codes_t=None, scales_t=None):
        for t, n in ((codes, 'codes'), (codes_t, 'codes_t')):
            if t is None and n == 'codes_t':
                continue
            if t.dtype not in (torch.uint8, torch.float8_e4m3fn) or t.dim() != 3 or not t.is_contiguous() or not t.is_cuda:
                raise ValueError('Weight8: %s has to be a contiguous uint8 or float8_e4m3fn GPU tensor [members, rows, columns]' % n)
        M, O, Ip = codes.shape
        if not 0 < inputs <= Ip or Ip != row_blocks(inputs) * BLOCK:
            raise ValueError('Weight8: %d columns of codes for %d inputs' % (Ip, inputs))
        if (codes_t is None) != (scales_t is None):
            raise ValueError('Weight8: codes_t and scales_t come together')
        want = [(scales, (M, row_blocks(O), scale_stride(inputs)))]
        if codes_t is not None:
            if tuple(codes_t.shape) != (M, inputs, row_blocks(O) * BLOCK) or codes_t.device != codes.device:
                raise ValueError('Weight8: codes_t has the wrong shape or device, %s on %s' % (tuple(codes_t.shape), codes_t.device))
            want.append((scales_t, (M, row_blocks(inputs), scale_stride(O))))
        for t, shape in want:
            if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != codes.device:
                raise ValueError('Weight8: scales have to be contiguous uint8 %s on the codes\' device, got %s %s'
                                 % (shape, t.dtype, tuple(t.shape)))
        self.codes, self.scales, self.codes_t, self.scales_t = codes, scales, codes_t, scales_t
        self.members, self.outputs, self.inputs = M, O, inputs

    @classmethod
    def _made(cls, codes, scales, inputs, codes_t, scales_t):
        """Of tensors that quantize_weight laid out: nothing to check."""
        w = cls.__new__(cls)
        w.codes, w.scales, w.codes_t, w.scales_t = codes, scales, codes_t, scales_t
        w.members, w.outputs, w.inputs = codes.shape[0], codes.shape[1], inputs
        return w

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return sum(t.numel() for t in (self.codes, self.scales, self.codes_t, self.scales_t) if t is not None)


def _rows(x):
    """(x as rows that one stride describes, number of rows, stride)."""
    K = x.shape[-1]
    R = x.numel() // K
    if x.is_contiguous():
        return x, R, K
    flat = x.reshape(-1, K) if x.dim() != 2 else x      # a view where one stride reaches every row, else a copy
    if flat.stride(1) != 1 or flat.stride(0) < K:
        flat = flat.contiguous()
    return flat, R, flat.stride(0)


def _quantize(x, act=0, keep=True):
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError('block8.quantize: needs rows of at least one element, got %s' % (tuple(x.shape),))
    K = x.shape[-1]
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype) if act else None
    rows, R, ld = _rows(x) if x.numel() else (x, 0, K)
    codes = scales = None
    if keep:
        codes = torch.empty((R, row_blocks(K) * BLOCK), device=x.device, dtype=torch.uint8)
        scales = torch.empty((R, scale_stride(K)), device=x.device, dtype=torch.uint8)
    if R:
        _lib.call('hecka_block8_quantize', x.device, rows.data_ptr(), DTYPES[x.dtype], R, K, ld, act, _ptr(codes), _ptr(scales), _ptr(y))
    if not keep:
        return None, y
    return Rows8._made(codes, scales, x.shape, x.dtype), y


def _values(q, dtype, act=0, dy=None):
    out = torch.empty(q.shape, device=q.device, dtype=dtype)
    if out.numel():
        _lib.call('hecka_block8_values', q.device, q.codes.data_ptr(), q.scales.data_ptr(), _ptr(dy), DTYPES[dtype],
                  q.codes.shape[0], q.shape[-1], act, out.data_ptr())
    return out


def quantize(x):
    """x [..., K] (any strides) as Rows8; no gradient passes."""
    _check(x, 'block8.quantize')
    _not_traced('block8.quantize')
    return _quantize(x.detach())[0]


def dequantize(q, dtype=None):
    """The values that a Rows8 stands for, in its own dtype or `dtype`."""
    _check_rows(q, 'block8.dequantize')
    _not_traced('block8.dequantize')
    dtype = q.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise TypeError('block8.dequantize: float32, bfloat16 or float16, got %s' % dtype)
    return _values(q, dtype)


def _members_apart(W):
    """W [M, O, I] with whole members: a member's slice of a flat parameter row is read in place."""
    M, O, I = W.shape
    return W.contiguous() if W.stride()[1:] != (I, 1) or (M > 1 and W.stride(0) < O * I) else W


def quantize_weight(W, transposed=True):
    """W [M, O, I] as Weight8; transposed=False leaves out codes_t and scales_t, half of its bytes, which linear does not read."""
    _check(W, 'block8.quantize_weight')
    _not_traced('block8.quantize_weight')
    return _quantize_weight(W, transposed)


def _quantize_weight(W, transposed=True):
    if W.dim() != 3 or 0 in W.shape:
        raise ValueError('block8.quantize_weight: needs [members, outputs, inputs] without zero sizes, got %s' % (tuple(W.shape),))
    W = _members_apart(W.detach())
    M, O, I = W.shape
    u8 = dict(device=W.device, dtype=torch.uint8)
    codes = torch.empty((M, O, row_blocks(I) * BLOCK), **u8)
    scales = torch.empty((M, row_blocks(O), scale_stride(I)), **u8)
    codes_t = torch.empty((M, I, row_blocks(O) * BLOCK), **u8) if transposed else None
    scales_t = torch.empty((M, row_blocks(I), scale_stride(O)), **u8) if transposed else None
    _lib.call('hecka_block8_weight', W.device, W.data_ptr(), DTYPES[W.dtype], M, O, I, W.stride(0), codes.data_ptr(),
              scales.data_ptr(), _ptr(codes_t), _ptr(scales_t))
    return Weight8._made(codes, scales, I, codes_t, scales_t)


def _members(q, M, what):
    """Members of rows [members, N, I] or, shared by all, [N, I]."""
    if len(q.shape) == 2:
        return 1
    if len(q.shape) != 3 or q.shape[0] != M:
        raise ValueError('%s: rows have shape %s, expected (%d, N, inputs) or (N, inputs)' % (what, tuple(q.shape), M))
    return M


def _bstride(b):
    return b.stride(0) if b is not None else 0


def _bias_rows(b):
    return b if b is None or b.stride(1) == 1 else b.contiguous()


def _products(what, products, dtype):
    """The library's number for results of `dtype` by the wanted products."""
    if products not in ('exact', 'fp8'):
        raise ValueError("%s: products are 'exact' or 'fp8', got %r" % (what, products))
    if products == 'fp8' and dtype == torch.float32:
        raise ValueError('%s: the fp8 instruction is for bfloat16 and float16; float32 results are exact products' % what)
    return DTYPES[dtype] + (FP8 if products == 'fp8' else 0)


def _product(q, codes, scales, M, O, I, bias, alpha, beta, dtype, number):
    N = q.shape[-2]
    y = torch.empty((M, N, O), device=q.device, dtype=dtype)
    if y.numel():
        nbytes = _lib.lib().hecka_block8_linear_workspace_bytes(M, N, O, I, M, number)
        ws = torch.empty((nbytes // 4,), device=q.device, dtype=torch.float32) if nbytes else None
        _lib.call('hecka_block8_linear', q.device, q.codes.data_ptr(), q.scales.data_ptr(), 1 if len(q.shape) == 2 else M,
                  codes.data_ptr(), scales.data_ptr(), M, N, O, I, _ptr(bias), _bstride(bias), alpha, beta, y.data_ptr(), number,
                  M, _ptr(ws), nbytes)
    return y


def _weight_grad(dy, q, alpha, beta, want_bias=True):
    M, N, O = dy.shape
    I = q.shape[-1]
    dW = torch.empty((M, O, I), device=dy.device, dtype=torch.float32)
    db = torch.empty((M, O), device=dy.device, dtype=torch.float32) if want_bias else None
    if N == 0:
        return dW.zero_(), db.zero_() if db is not None else None
    if dW.numel():
        nbytes = _lib.lib().hecka_block8_wgrad_workspace_bytes(M, N, O, I)
        ws = torch.empty((nbytes // 4,), device=dy.device, dtype=torch.float32) if nbytes else None
        _lib.call('hecka_block8_wgrad', dy.device, dy.data_ptr(), DTYPES[dy.dtype], q.codes.data_ptr(), q.scales.data_ptr(),
                  1 if len(q.shape) == 2 else M, M, N, O, I, alpha, beta, dW.data_ptr(), _ptr(db), _ptr(ws), nbytes)
    return dW, db


def _bias_grad(dy, scale):
    """The column sums alone, fp32 in a fixed order: those beside the weight gradient of rows of one zero."""
    N = dy.shape[1]
    codes = torch.zeros((N, BLOCK + scale_stride(1)), device=dy.device, dtype=torch.uint8).view(-1)
    one = Rows8._made(codes[:N * BLOCK], codes[N * BLOCK:], (N, 1), dy.dtype)
    return _weight_grad(dy, one, 0.0, scale)[1]


def weight_grad(dy, rows, scale=1.0, bias_scale=1.0):
    """(dW, db) = (scale dy^T x, bias_scale sum of dy over the rows), fp32, of y = scale x W^T + bias_scale b, from dy [M, N, O] and
    x kept as Rows8 [M, N, I] (or [N, I], shared by all members); no gradient passes."""
    _check(dy, 'block8.weight_grad')
    _not_traced('block8.weight_grad')
    _check_rows(rows, 'block8.weight_grad')
    if dy.dim() != 3:
        raise ValueError('block8.weight_grad: dy has to be [members, N, outputs], got %s' % (tuple(dy.shape),))
    _members(rows, dy.shape[0], 'block8.weight_grad')
    if rows.shape[-2] != dy.shape[1]:
        raise ValueError('block8.weight_grad: %d rows of dy for %d in the checkpoint' % (dy.shape[1], rows.shape[-2]))
    _same_device('block8.weight_grad', dy, rows)
    _sizes('block8.weight_grad', dy.shape[0], dy.shape[1], dy.shape[2], rows.shape[-1])
    return _weight_grad(dy.detach().contiguous(), rows, scale, bias_scale)


def _sizes(what, M, N, O, I):
    if max(N, O, I) > _MOST or M > 65535:
        raise ValueError('%s: sizes up to %d and 65535 members, got M = %d, N = %d, O = %d, I = %d' % (what, _MOST, M, N, O, I))
    if min(M, O, I) == 0:
        raise ValueError('%s: zero members, outputs or inputs' % what)


class _Linear8(torch.autograd.Function):
    """y[m] = scale x8[m] W8[m]^T + bias_scale b[m]; t: _products' number.  Keeps the codes of x and W (a byte per element each) and nothing else; the
    backward's products are dx = scale dy8 W8 and dW = scale dy^T x8 (dy as it is, x from the checkpoint)."""

    @staticmethod
    def forward(ctx, x, W, b, scale, bias_scale, t):
        M, O, I = W.shape
        N, xm = x.shape[-2], 1 if x.dim() == 2 else M
        need_dx, need_dw, _ = ctx.needs_input_grad[:3]
        y = torch.empty((M, N, O), device=x.device, dtype=x.dtype)
        kept = None
        if N:
            rows, _, ld = _rows(x)
            W = _members_apart(W)
            size = _lib.lib().hecka_block8_train_bytes
            nk, nw = size(0, M, xm, N, O, I, t, need_dx, need_dw), size(1, M, xm, N, O, I, t, need_dx, need_dw)
            if nk:
                kept = torch.empty((nk,), device=x.device, dtype=torch.uint8)
            ws = torch.empty((nw,), device=x.device, dtype=torch.uint8)
            _lib.call('hecka_block8_train_fwd', x.device, rows.data_ptr(), t, xm, ld, W.data_ptr(), DTYPES[W.dtype], W.stride(0), M, N, O, I,
                      _ptr(b), _bstride(b), scale, bias_scale, need_dx, need_dw, y.data_ptr(), _ptr(kept), nk, ws.data_ptr(), nw)
        # a tensor that autograd frees with the graph; only the codes that a gradient will ask for
        ctx.save_for_backward(kept)
        ctx.cfg = (x.shape, x.dtype, W.shape, W.dtype, b is not None, scale, bias_scale, need_dx, need_dw, t)
        return y

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        kept, = ctx.saved_tensors
        xshape, xdtype, (M, O, I), wdtype, has_bias, scale, bias_scale, need_dx, need_dw, t = ctx.cfg
        N, xm = dy.shape[1], 1 if len(xshape) == 2 else M
        dy = dy.contiguous()
        dx = dW = db = None
        want_x, want_w, want_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], has_bias and ctx.needs_input_grad[2]      # may be fewer now
        if want_x:
            dx = torch.empty(xshape, device=dy.device, dtype=xdtype)
        if want_w:
            dW = torch.empty((M, O, I), device=dy.device, dtype=torch.float32)
            db = torch.empty((M, O), device=dy.device, dtype=torch.float32) if want_b else None
        elif want_b:
            db = _bias_grad(dy, bias_scale)
        if N == 0:
            return dx, dW.zero_().to(wdtype) if want_w else None, db.zero_() if want_b else None, None, None, None
        if want_x or want_w:
            nw = _lib.lib().hecka_block8_train_bytes(2, M, xm, N, O, I, t, want_x, want_w)
            ws = torch.empty((nw,), device=dy.device, dtype=torch.uint8) if nw else None
            _lib.call('hecka_block8_train_bwd', dy.device, dy.data_ptr(), t, xm, M, N, O, I, scale, bias_scale, need_dx, need_dw, kept.data_ptr(),
                      kept.numel(), _ptr(dx), _ptr(dW), _ptr(db) if want_w else None, _ptr(ws), nw)
        return dx, dW.to(wdtype) if want_w else None, db, None, None, None


def _check_bias(what, b, M, O):
    if b is None:
        return
    _check(b, what)
    if b.dtype != torch.float32 or tuple(b.shape) != (M, O):
        raise ValueError('%s: bias has to be float32 (%d, %d), got %s %s' % (what, M, O, b.dtype, tuple(b.shape)))


def linear(x, weight, bias=None, scale=1.0, bias_scale=1.0, products='exact'):
    """y[m] = scale x[m] W[m]^T + bias_scale b[m] in 8-bit blocks; x [M, N, I], or [N, I] shared by all members; bias fp32 [M, O].

    weight: a float tensor [M, O, I] - training: its codes are made here, x's are the checkpoint; or a Weight8 - serving: no
    gradients, x may be Rows8 (then the result has the dtype it was made from), and up to 16 rows take one launch that makes the
    codes of x on the way.

    products: 'exact' - of the blocks' values, added in fp32 - or, for bf16 / fp16 x, 'fp8' - the fp8 matrix instruction, nearly twice as
    fast, which cuts each product 13 bits below the largest of eight (1.5e-5 of the result); up to 16 rows served are exact with either."""
    what = 'block8.linear'
    if isinstance(weight, Weight8):
        w = weight
        M, O, I = w.members, w.outputs, w.inputs
        _not_traced(what)
        if not isinstance(x, Rows8):
            _check(x, what)
            if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
                raise RuntimeError('block8.linear: weights in codes serve only (no gradients): pass the float weights to train')
        if _lib.tangents(x, bias):
            raise RuntimeError('block8.linear: weights in codes serve only (no tangents)')
        xm = _members(x, M, what)
        if x.shape[-1] != I:
            raise ValueError('%s: rows of %d elements for %d inputs' % (what, x.shape[-1], I))
        _check_bias(what, bias, M, O)
        _same_device(what, x, w, bias)
        N = x.shape[-2]
        _sizes(what, M, N, O, I)
        number = _products(what, products, x.dtype)
        b = _bias_rows(bias.detach() if bias is not None else None)
        if isinstance(x, Rows8) or N > 16:
            q = x if isinstance(x, Rows8) else _quantize(x.detach())[0]
            return _product(q, w.codes, w.scales, M, O, I, b, scale, bias_scale, q.dtype, number)
        x = x.detach().contiguous()
        y = torch.empty((M, N, O), device=x.device, dtype=x.dtype)
        if N:
            _lib.call('hecka_block8_linear_token', x.device, x.data_ptr(), DTYPES[x.dtype], xm, w.codes.data_ptr(), w.scales.data_ptr(),
                      M, N, O, I, _ptr(b), _bstride(b), scale, bias_scale, y.data_ptr())
        return y
    _check(x, what)
    _check(weight, what)
    if weight.dim() != 3:
        raise ValueError('%s: weight has to be [members, outputs, inputs], got %s' % (what, tuple(weight.shape)))
    M, O, I = weight.shape
    _members(x, M, what)
    if x.shape[-1] != I:
        raise ValueError('%s: rows of %d elements for %d inputs' % (what, x.shape[-1], I))
    _check_bias(what, bias, M, O)
    _same_device(what, x, weight, bias)
    _sizes(what, M, x.shape[-2], O, I)
    number = _products(what, products, x.dtype)
    if not torch.is_grad_enabled() and not _lib.recorded():      # nothing is kept for a backward pass
        w = _quantize_weight(weight, transposed=False)
        return _product(_quantize(x)[0], w.codes, w.scales, M, O, I, _bias_rows(bias), float(scale), float(bias_scale), x.dtype, number)
    return _Linear8.apply(x, weight, _bias_rows(bias), float(scale), float(bias_scale), number)
