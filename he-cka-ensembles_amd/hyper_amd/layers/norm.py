"""Batched BatchNorm (hyper/layers/norm.py:12-46 `_NormAffine` / `_NormBuffers`, :49-127 `_NormBase`, :129-224
`_BatchNorm.forward`, BatchNorm1d / BatchNorm2d).  The reference loops F.batch_norm over the ensemble members and stacks;
here all members go through ONE launch (libhecka hecka_batchnorm_fwd_f32 / _bwd_f32: a workgroup per (member, channel)).
On the fused path (hecka_batchnorm_act_*_packed_f32) the kernels read weight | bias from the layer's flat parameter row
and return their gradients as one tensor, and the forward kernel updates the running statistics itself when every member
is selected in order; otherwise the selected members' statistics are updated with a handful of [members, C] tensor ops."""
import torch
import torch.nn as nn

from .. import _lib
from ..config import knobs
from .module import GenModule, ParametersGroup, register_gen_module


class _NormAffine(ParametersGroup):
    def __init__(self, num_features):
        super().__init__(shapes=[('weight', (num_features,)), ('bias', (num_features,))])

    def gen_initialized_params(self, dtype=None, device=None, gain=1):
        params = self.gen_empty_params(dtype=dtype, device=device, requires_grad=True)
        with torch.no_grad():
            nn.init.ones_(params['weight'])
            nn.init.zeros_(params['bias'])
        return params


class _NormBuffers(ParametersGroup):
    def __init__(self, num_features):
        super().__init__(shapes=[('mean', (num_features,)), ('var', (num_features,)), ('num_batches_tracked', (1,))])

    def gen_initialized_params(self, dtype=None, device=None, gain=1):
        params = self.gen_empty_params(dtype=dtype, device=device, requires_grad=False)
        nn.init.zeros_(params['mean'])
        nn.init.ones_(params['var'])
        nn.init.zeros_(params['num_batches_tracked'])
        return params


class BatchedBatchNorm(torch.autograd.Function):
    """y[m] = batch_norm(x[m], weight[m], bias[m]);  x [M,N,C,*], weight / bias [M,C] | None.  Returns (y, batch mean,
    biased batch variance) - the statistics are by-products for the running averages and carry no gradient."""

    @staticmethod
    def forward(ctx, x, weight, bias, run_mean, run_var, training, eps):
        if not x.is_cuda or x.dtype != torch.float32:
            raise RuntimeError('hyper_amd BatchNorm needs fp32 GPU tensors; there is no CPU path')
        x = x.contiguous()
        M, N, C = x.shape[:3]
        S = int(x[0, 0, 0].numel())
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        y = torch.empty_like(x)
        mean = torch.empty((M, C), device=x.device, dtype=torch.float32)
        rstd = torch.empty_like(mean)
        var = torch.empty_like(mean) if training else None
        ptr = lambda t: t.data_ptr() if t is not None else None   # noqa: E731
        _lib.check(_lib.lib().hecka_batchnorm_fwd_f32(
            x.data_ptr(), M, N, C, S, ptr(w), ptr(b), ptr(run_mean), ptr(run_var), int(training), float(eps),
            y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), ptr(var), torch.cuda.current_stream().cuda_stream),
            'batchnorm_fwd')
        ctx.save_for_backward(x, mean, rstd, w)
        ctx.cfg = (training, S, weight is not None, bias is not None)
        if var is None:
            var = mean.new_zeros(())
        ctx.mark_non_differentiable(mean, var)
        return y, mean, var

    @staticmethod
    def backward(ctx, dy, _dm, _dv):
        x, mean, rstd, w = ctx.saved_tensors
        training, S, has_w, has_b = ctx.cfg
        M, N, C = x.shape[:3]
        dy = dy.contiguous()
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(mean) if has_w and ctx.needs_input_grad[1] else None
        db = torch.empty_like(mean) if has_b and ctx.needs_input_grad[2] else None
        ptr = lambda t: t.data_ptr() if t is not None else None   # noqa: E731
        _lib.check(_lib.lib().hecka_batchnorm_bwd_f32(
            dy.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), ptr(w), M, N, C, S, int(training),
            ptr(dx), ptr(dw), ptr(db), torch.cuda.current_stream().cuda_stream), 'batchnorm_bwd')
        return dx, dw, db, None, None, None, None


def tag_absmax(t, amax):
    """Remember max |t[g]| (a kernel by-product, [G] on the device) on the tensor object; `cached_absmax` gives it to the next
    consumer as long as the tensor has not been written since."""
    t._hecka_absmax = (amax, t._version)


def cached_absmax(t, rows):
    tag = getattr(t, '_hecka_absmax', None)
    if tag is not None and tag[1] == t._version and tag[0].shape[0] == rows and t.shape[0] == rows:
        return tag[0]
    return None


class BatchedBatchNormAct(torch.autograd.Function):
    """y[m] = [relu](batch_norm(x[m], weight[m], bias[m]) [+ res[m]]) in one launch each way (hecka_batchnorm_act_*): the
    two tails of a ResNet block, norm -> relu and norm -> + shortcut -> relu.  Same by-products as BatchedBatchNorm.
    packed: `weight` is the layer's flat parameter row [M, 2 C] (weight | bias) as the batched layers keep it - read in
    place, its gradient returned as one tensor (no slice copies either way); upd = (running mean store, running var
    store, factor): the kernel updates the running statistics itself (then the returned statistics are not needed)."""

    @staticmethod
    def forward(ctx, x, res, weight, bias, run_mean, run_var, training, eps, relu, packed=False, upd=None):
        if not x.is_cuda or x.dtype != torch.float32:
            raise RuntimeError('hyper_amd BatchNorm needs fp32 GPU tensors; there is no CPU path')
        x = x.contiguous()
        res = res.contiguous() if res is not None else None
        M, N, C = x.shape[:3]
        S = int(x[0, 0, 0].numel())
        ptr = lambda t: t.data_ptr() if t is not None else None   # noqa: E731
        if packed:
            w = weight.contiguous()
            assert bias is None and tuple(w.shape) == (M, 2 * C) and w.dtype == torch.float32
            w_ptr, b_ptr, wstride = w.data_ptr(), w.data_ptr() + 4 * C, 2 * C
        else:
            w = weight.contiguous() if weight is not None else None
            b = bias.contiguous() if bias is not None else None
            w_ptr, b_ptr, wstride = ptr(w), ptr(b), C
        y = torch.empty_like(x)
        ymax = torch.empty((M,), device=x.device, dtype=torch.float32)
        mean = torch.empty((M, C), device=x.device, dtype=torch.float32)
        rstd = torch.empty_like(mean)
        var = torch.empty_like(mean) if training and upd is None else None
        # all the backward needs of y is the relu's sign: one byte per four outputs instead of y in both of its sweeps
        mask = (torch.empty((x.numel() // 4,), device=x.device, dtype=torch.uint8)
                if relu and knobs.bn_mask and any(ctx.needs_input_grad[:4]) else None)
        _lib.check(_lib.lib().hecka_batchnorm_act_fwd_packed_f32(
            x.data_ptr(), ptr(res), M, N, C, S, w_ptr, b_ptr, wstride, ptr(run_mean), ptr(run_var), int(training), float(eps),
            int(bool(relu)), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), ptr(var), ymax.data_ptr(),
            upd[0].data_ptr() if upd is not None else None, upd[1].data_ptr() if upd is not None else None,
            float(upd[2]) if upd is not None else 0.0, ptr(mask), torch.cuda.current_stream().cuda_stream), 'batchnorm_act_fwd')
        tag_absmax(y, ymax)      # the convolution that reads y next takes its operand scale from here
        ctx.save_for_backward(x, mean, rstd, w, y if relu and mask is None else None, mask)
        ctx.cfg = (training, S, weight is not None, bias is not None or packed, res is not None, packed, bool(relu))
        if var is None:
            var = mean if upd is not None else mean.new_zeros(())
        ctx.mark_non_differentiable(mean, var)
        return y, mean, var

    @staticmethod
    def backward(ctx, dy, _dm, _dv):
        x, mean, rstd, w, y, mask = ctx.saved_tensors
        training, S, has_w, has_b, has_res, packed, relu = ctx.cfg
        M, N, C = x.shape[:3]
        dy = dy.contiguous()
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dxmax = torch.empty((M,), device=x.device, dtype=torch.float32) if dx is not None else None
        dres = None
        if has_res and ctx.needs_input_grad[1]:
            dres = torch.empty_like(x) if relu else dy      # no relu: the residual's gradient is dy itself
        ptr = lambda t: t.data_ptr() if t is not None else None   # noqa: E731
        if packed:
            dw = torch.empty((M, 2 * C), device=x.device, dtype=torch.float32) if ctx.needs_input_grad[2] else None
            db = None
            dw_ptr, db_ptr, wstride = ptr(dw), (dw.data_ptr() + 4 * C if dw is not None else None), 2 * C
        else:
            dw = torch.empty_like(mean) if has_w and ctx.needs_input_grad[2] else None
            db = torch.empty_like(mean) if has_b and ctx.needs_input_grad[3] else None
            dw_ptr, db_ptr, wstride = ptr(dw), ptr(db), C
        _lib.check(_lib.lib().hecka_batchnorm_act_bwd_packed_f32(
            dy.data_ptr(), x.data_ptr(), ptr(y), mean.data_ptr(), rstd.data_ptr(), ptr(w), wstride, M, N, C, S, int(training),
            ptr(dx), ptr(dres) if relu else None, dw_ptr, db_ptr, ptr(dxmax), ptr(mask),
            torch.cuda.current_stream().cuda_stream), 'batchnorm_act_bwd')
        if dx is not None:
            tag_absmax(dx, dxmax)    # dx is the output gradient of the convolution in front of this norm
        return dx, dres, dw, db, None, None, None, None, None, None, None


def fused_act_eligible(x):
    """The fused norm (+ residual) + relu launch takes fp32 GPU tensors with a multiple of four positions per channel."""
    return (knobs.bn_fuse and x.is_cuda and x.dtype == torch.float32 and x.dim() >= 3
            and int(x[0, 0, 0].numel()) % 4 == 0)


class _NormBase(GenModule):
    def __init__(self, num_features, eps=1e-5, momentum=0.1, affine=True, track_running_stats=True, track=True):
        super().__init__(track=track)
        self.num_features, self.eps, self.momentum = num_features, eps, momentum
        self.affine, self.track_running_stats = affine, track_running_stats
        self.affine_module = _NormAffine(num_features) if affine else None
        self.buffer_module = _NormBuffers(num_features) if track_running_stats else None

    def is_generated(self):
        return False

    def define_generated_modules(self):
        mod = super().define_generated_modules()
        if self.affine:
            mod['affine'] = self.affine_module.define_generated_modules()
        if self.track_running_stats:      # fixed ensembles only (as in the reference)
            mod['norm_buffer'] = self.buffer_module.define_generated_modules()
        return mod

    def _check_input_dim(self, input):
        raise NotImplementedError

    def extra_repr(self):
        return '{num_features}, eps={eps}, momentum={momentum}, affine={affine}, ' \
               'track_running_stats={track_running_stats}'.format(**self.__dict__)


class _BatchNorm(_NormBase):
    def forward(self, params, input, residual=None, relu=False):
        """`residual` / `relu` (not in the reference's signature): y = [relu](norm(input) [+ residual]) as ONE launch when
        the shape allows (fused_act_eligible), else the same thing with torch ops behind the plain norm."""
        self._check_input_dim(input)
        fused = fused_act_eligible(input) and (relu or residual is not None or self.affine)
        weight = bias = None
        bufs = params['norm_buffer']['self'] if self.track_running_stats else None
        bn_training = self.training or not self.track_running_stats
        run_mean = run_var = None
        if bufs is not None and not bn_training:
            run_mean, run_var = bufs.gather('mean'), bufs.gather('var')
        # the running statistics updated inside the forward kernel: every member in order, a fixed momentum
        upd = None
        if fused and self.training and bufs is not None and self.momentum is not None and bufs.whole('mean') and bufs.whole('var'):
            upd = (bufs.store('mean'), bufs.store('var'), float(self.momentum))
        flat = params['affine']['self'] if self.affine else None
        packed = (fused and flat is not None and flat.is_cuda and flat.dtype == torch.float32 and flat.dim() == 2
                  and flat.shape[1] == 2 * self.num_features)
        if self.affine and not packed:
            viewed = self.affine_module.from_flat(flat)
            weight, bias = viewed['weight'], viewed['bias']
        if fused:
            y, mean, var = BatchedBatchNormAct.apply(input, residual, flat if packed else weight, None if packed else bias,
                                                     run_mean, run_var, bn_training, self.eps, bool(relu), packed, upd)
        else:
            y, mean, var = BatchedBatchNorm.apply(input, weight, bias, run_mean, run_var, bn_training, self.eps)
            if residual is not None:
                y = y + residual
            if relu:
                y = torch.relu(y)
        if self.training and bufs is not None and upd is None:
            cnt = input.shape[1] * int(input[0, 0, 0].numel())
            with torch.no_grad():
                if self.momentum is None:   # cumulative average (num_batches_tracked is never advanced by the reference)
                    factor = 1.0 / bufs.gather('num_batches_tracked')
                else:
                    factor = self.momentum
                bufs.update('mean', mean, factor)
                bufs.update('var', var * (cnt / max(cnt - 1, 1)), factor)
        return self.track_feature(y), y


_NORM_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _ptr(t):
    return t.data_ptr() if t is not None else None


class _LayerNorm(torch.autograd.Function):
    """Layer norm of x [..., D] as G groups of rows (libhecka hecka_layernorm_*).  weight / bias fp32 [G, D], [D] where G = 1;
    packed: `weight` is the flat parameter row [G, 2 D] (weight | bias), read in place, its gradient returned as one tensor.
    Reshapes happen in here: outside they would be nodes of the graph."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, packed, G):
        x = x.contiguous()
        D = x.shape[-1]
        R = x.numel() // (G * D) if G else 0
        y = torch.empty_like(x)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        mean = rstd = None
        if ctx is not None and any(ctx.needs_input_grad):
            mean, rstd = torch.empty((2, G, R), device=x.device, dtype=torch.float32).unbind(0)
        if R:
            w_ptr = _ptr(w)
            _lib.call('hecka_layernorm_fwd', x.device, x.data_ptr(), _NORM_DTYPES[x.dtype], G, R, D, w_ptr,
                      w_ptr + 4 * D if packed else _ptr(b), 2 * D if packed else D, eps, y.data_ptr(), _ptr(mean), _ptr(rstd))
        if ctx is not None:
            ctx.save_for_backward(x, mean, rstd, w)
            ctx.cfg = (packed, bias is not None, G, R)
        return y

    @staticmethod
    def run(*args):
        """apply, without a graph's node where nothing will ask for one (a third of a small call's time)."""
        if _lib.recorded() or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:3])):
            return _LayerNorm.apply(*args)
        return _LayerNorm.forward(None, *args)

    @staticmethod
    @_lib.first_order
    def backward(ctx, dy):
        x, mean, rstd, w = ctx.saved_tensors
        packed, has_bias, G, R = ctx.cfg
        D = x.shape[-1]
        need = ctx.needs_input_grad
        dx = torch.empty_like(x) if need[0] else None
        dw = torch.empty_like(w) if w is not None and need[1] else None
        db = torch.empty(w.shape, device=x.device, dtype=torch.float32) if has_bias and need[2] else None
        if R == 0:
            return dx, dw.zero_() if dw is not None else None, db.zero_() if db is not None else None, None, None, None
        nbytes, ws = 0, None
        if dw is not None or db is not None:
            nbytes = _lib.lib().hecka_layernorm_bwd_workspace_bytes(G, R, D)
            ws = torch.empty((nbytes // 4,), device=x.device, dtype=torch.float32) if nbytes else None
        dy = dy.contiguous()      # (kept: a copy has to live until the launch)
        _lib.call('hecka_layernorm_bwd', x.device, dy.data_ptr(), x.data_ptr(), _NORM_DTYPES[x.dtype], mean.data_ptr(),
                  rstd.data_ptr(), G, R, D, _ptr(w), 2 * D if packed else D, _ptr(dx), _ptr(dw),
                  dw.data_ptr() + 4 * D if packed and dw is not None else _ptr(db), 2 * D if packed else D, _ptr(ws), nbytes)
        return dx, dw, db, None, None, None


def _check_layer_norm(x, affine):
    if not torch.is_tensor(x) or not x.is_cuda:
        raise RuntimeError('hyper_amd layer norm needs GPU tensors; there is no CPU path')
    if x.dtype not in _NORM_DTYPES:
        raise TypeError('layer norm takes float32, bfloat16 or float16, got %s' % x.dtype)
    if x.dim() < 1 or not 0 < x.shape[-1] <= 16384:
        raise ValueError('layer norm takes rows of 1 to 16384 elements, got %s' % (tuple(x.shape),))
    for name, t in affine:
        if t is None:
            continue
        if t.device != x.device:
            raise RuntimeError('layer norm: x on %s, %s on %s' % (x.device, name, t.device))
        if t.dtype != torch.float32:
            raise TypeError('layer norm: %s has to be float32, got %s' % (name, t.dtype))


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last axis (1 to 16384 elements) of x, fp32 / bf16 / fp16 on the GPU; statistics in fp32.  weight / bias
    fp32: [D] shared by every row, or [M, D] with x [M, ..., D], a row for each member.  Gradients for x (its dtype), weight and
    bias (fp32; a shared one's is the sum over the members)."""
    _check_layer_norm(x, (('weight', weight), ('bias', bias)))
    D = x.shape[-1]
    given = [t for t in (weight, bias) if t is not None]
    if weight is None and bias is not None:
        raise ValueError('layer norm: a bias needs a weight')
    if any(t.shape != given[0].shape for t in given):
        raise ValueError('layer norm: weight %s and bias %s' % (tuple(weight.shape), tuple(bias.shape)))
    G = 1
    if given and weight.dim() == 2:
        if x.dim() < 2 or tuple(weight.shape) != (x.shape[0], D):
            raise ValueError('layer norm: weight has to be (%d,) or (%s, %d), got %s' % (D, x.shape[0] if x.dim() > 1 else '-', D, tuple(weight.shape)))
        G = x.shape[0]
    elif given and tuple(weight.shape) != (D,):
        raise ValueError('layer norm: weight has to be (%d,) or (members, %d), got %s' % (D, D, tuple(weight.shape)))
    if G > 65535:
        raise ValueError('layer norm: at most 65535 members, got %d' % G)
    return _LayerNorm.run(x, weight, bias, float(eps), False, G)


@register_gen_module('layer_norm')
class LayerNorm(GenModule):
    """Batched layer norm, every member with its own weight and bias (affine): x [members, samples, ..., num_features].  The
    reference has none; parameters and naming follow its batched norms (hyper/layers/norm.py:12-46)."""

    def __init__(self, num_features, eps=1e-5, affine=True, track=True):
        super().__init__(track=track)
        if not 0 < num_features <= 16384:
            raise ValueError('LayerNorm takes rows of 1 to 16384 elements, got %d' % num_features)
        self.num_features, self.eps, self.affine = num_features, eps, affine
        self.affine_module = _NormAffine(num_features) if affine else None

    def define_generated_modules(self):
        mod = super().define_generated_modules()
        if self.affine:
            mod['affine'] = self.affine_module.define_generated_modules()
        return mod

    def forward(self, params, input):
        flat = params['affine']['self'] if self.affine else None
        _check_layer_norm(input, (('params', flat),))
        if input.dim() < 2 or input.shape[-1] != self.num_features:
            raise ValueError('expected (members, ..., %d) input (got %s)' % (self.num_features, tuple(input.shape)))
        if flat is not None and tuple(flat.shape) != (input.shape[0], 2 * self.num_features):
            raise ValueError('expected parameters (%d, %d) (got %s)' % (input.shape[0], 2 * self.num_features, tuple(flat.shape)))
        y = _LayerNorm.run(input, flat, None, float(self.eps), flat is not None, input.shape[0])
        return self.track_feature(y), y

    def extra_repr(self):
        return '{num_features}, eps={eps}, affine={affine}'.format(**self.__dict__)


class BatchNorm1d(_BatchNorm):
    def _check_input_dim(self, input):
        if input.dim() != 3 and input.dim() != 4:
            raise ValueError('expected 3D or 4D input (got %dD input)' % input.dim())


class BatchNorm2d(_BatchNorm):
    def _check_input_dim(self, input):
        if input.dim() != 5:
            raise ValueError('expected 5D input (got %dD input)' % input.dim())
