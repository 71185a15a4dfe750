"""Layer norm over the last dimension, with the residual add in front of it, and its gradients.

`LayerNorm` is `nn.LayerNorm` over one dimension (same arguments, parameters and state-dict keys)
whose forward runs `sf_layer_norm` (csrc/layer_norm.hip); it is registered as the norm layer `LN`, so
`norm_cfg=dict(type='LN')` reaches it in every module that builds its norms from a config (sparse conv
blocks apply it to the (N, C) voxel features).  Rows are fp32, fp16 or bf16, parameters of the same
type or fp32; statistics and sums are fp32 and every output is rounded once.  Differentiable once (no
double backward) and backwards only: tensors with forward-mode tangents are refused, and so are
torch.jit.trace, make_fx and export.  No CPU path.

Capturing a backward pass in a HIP graph follows torch's rule for any operator: no autograd graph
over the same leaves may be alive outside the capture.
"""
import torch
from torch import nn

from . import _lib
from .registry import NORM_LAYERS


MOST_FEATURES = 1 << 29      # column numbers, twice over, stay in 31 bits


def _check(x, weight, bias):
    """-> (d, dtype code, parameters' type) of well-formed rows and parameters."""
    dtype = x.dtype
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None:
        raise RuntimeError(f'layer_norm takes fp32, fp16 or bf16, got {dtype}')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f'layer_norm needs rows of at least one element, got {tuple(x.shape)}')
    d = x.shape[-1]
    if type(d) is not int:      # torch.jit.trace hands out tensors, and would record allocations, no call
        raise RuntimeError('layer_norm cannot be traced')
    if _lib.dispatch_modes():
        _lib.refuse_tracing('layer_norm')
    if d > MOST_FEATURES:
        raise RuntimeError(f'layer_norm takes rows of up to {MOST_FEATURES} elements, got {d}')
    pdtype = None
    for name, t in (('weight', weight), ('bias', bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != d:
            raise RuntimeError(f'{name} must have shape ({d},), got {tuple(t.shape)}')
        if t.device != x.device:
            raise RuntimeError(f'{name} is on {t.device}, x on {x.device}')
        if t.dtype not in (dtype, torch.float32) or t.dtype != (pdtype or t.dtype):
            raise RuntimeError(f'weight and bias must both be {dtype} or both float32, '
                               f'{name} is {t.dtype}')
        pdtype = t.dtype
    return d, code, pdtype or dtype


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, residual=None, return_sum=False,
                       keep_stats=False):
    """-> (y, sum, mean, rstd) of s = x + residual, y = (s - mean) * rstd * weight + bias.  sum (s
    rounded) with return_sum, mean and rstd (fp32, x.shape[:-1]) with keep_stats, else None.  Not
    differentiable: see `layer_norm`."""
    if _lib.forward_ad._current_level >= 0:
        _lib.refuse_tangents('layer_norm', x, weight, bias, residual)
    d, code, pdtype = _check(x, weight, bias)
    if d == 1:
        x, weight, bias, residual = _lib.resolved(x, weight, bias, residual)
    if not eps >= 0:
        raise RuntimeError(f'eps must not be negative, got {eps}')
    if residual is not None:
        _lib.same(x, 'residual', residual)
        if residual.shape != x.shape:
            residual = residual.expand(x.shape)
        residual = residual.contiguous()
    if _lib.elsewhere(x.device):
        with torch.cuda.device(x.device):
            return layer_norm_forward(x, weight, bias, eps, residual, return_sum, keep_stats)
    x = x.contiguous()
    if weight is not None:
        weight = weight.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    y = torch.empty_like(x)
    s = torch.empty_like(x) if return_sum else None
    mean = rstd = None
    if keep_stats:
        mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
        rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rc = _lib.lib().sf_layer_norm(
        x.data_ptr(), None if residual is None else residual.data_ptr(),
        None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
        y.data_ptr(), None if s is None else s.data_ptr(), None if mean is None else mean.data_ptr(),
        None if rstd is None else rstd.data_ptr(), x.numel() // d, d, eps, code,
        _lib.DTYPE_CODES[pdtype], _lib.stream(x.device))
    if rc:
        _lib.check(rc)
    return y, s, mean, rstd


def layer_norm_backward(grad, x, mean, rstd, weight=None, grad_sum=None, needs=(True, True, True),
                        param_dtype=None):
    """Gradients (dx, dweight, dbias) of `layer_norm_forward` for the gradient `grad` of y and
    `grad_sum` of the sum (or None); x is the normalised sum, mean and rstd as it returned them.  dx is
    the gradient of x and of the residual alike.  `needs` says which are wanted, the others are None;
    the parameter gradients have weight's type (without a weight: `param_dtype`, or x's)."""
    if _lib.forward_ad._current_level >= 0:
        _lib.refuse_tangents('layer_norm_backward', grad, x, mean, rstd, weight, grad_sum)
    d, code, pdtype = _check(x, weight, None)
    if weight is None and param_dtype is not None:
        pdtype = param_dtype
        if pdtype not in (x.dtype, torch.float32):
            raise RuntimeError(f'param_dtype must be {x.dtype} or float32, got {pdtype}')
    for name, t in (('grad', grad), ('grad_sum', grad_sum)):
        if t is not None:
            _lib.same(x, name, t)
            if t.shape != x.shape:
                raise RuntimeError(f'{name} must have shape {tuple(x.shape)}, got {tuple(t.shape)}')
    m = x.numel() // d
    if d == 1 or m == 1:
        grad, x, mean, rstd, weight, grad_sum = _lib.resolved(grad, x, mean, rstd, weight, grad_sum)
    for name, t in (('mean', mean), ('rstd', rstd)):
        if t.dtype != torch.float32 or t.numel() != m or t.device != x.device:
            raise RuntimeError(f'{name} must be {m} fp32 values on {x.device}, got {tuple(t.shape)} '
                               f'{t.dtype} on {t.device}')
    if _lib.elsewhere(x.device):
        with torch.cuda.device(x.device):
            return layer_norm_backward(grad, x, mean, rstd, weight, grad_sum, needs, param_dtype)
    grad, x = grad.contiguous(), x.contiguous()
    if grad_sum is not None:
        grad_sum = grad_sum.contiguous()
    if weight is not None:
        weight = weight.contiguous()
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dx = torch.empty_like(x)
    dw = x.new_empty(d, dtype=pdtype) if needs[1] else None
    db = x.new_empty(d, dtype=pdtype) if needs[2] else None
    L = _lib.lib()
    nbytes = L.sf_layer_norm_backward_workspace(m, d, code) if needs[1] or needs[2] else 0
    ws = _lib.workspace(nbytes, x)
    rc = L.sf_layer_norm_backward(
        grad.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
        None if weight is None else weight.data_ptr(),
        None if grad_sum is None else grad_sum.data_ptr(), dx.data_ptr(),
        None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), m, d, code,
        _lib.DTYPE_CODES[pdtype], None if ws is None else ws.data_ptr(), nbytes,
        _lib.stream(x.device))
    if rc:
        _lib.check(rc)
    return dx if needs[0] else None, dw, db


class _LayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, return_sum):
        y, s, mean, rstd = layer_norm_forward(x, weight, bias, eps, residual,
                                              return_sum or residual is not None, True)
        ctx.pdtype = bias.dtype if bias is not None else None
        ctx.set_materialize_grads(False)
        # without a residual the sum is x: a returned one is x's copy, the saved one x itself
        ctx.save_for_backward(x if residual is None else s, weight, mean, rstd)
        return (y, s) if return_sum else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, grad_sum=None):
        x, weight, mean, rstd = ctx.saved_tensors
        needs = ctx.needs_input_grad
        if grad is None and grad_sum is None:
            return (None,) * 6
        if grad is None:
            grad = torch.zeros_like(x)
        dx, dw, db = layer_norm_backward(grad, x, mean, rstd, weight, grad_sum,
                                         (needs[0] or needs[4], needs[1], needs[2]), ctx.pdtype)
        return dx if needs[0] else None, dw, db, None, dx if needs[4] else None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None, return_sum=False):
    """Layer norm of x + residual over the last dimension, differentiable in all four tensors; with
    return_sum -> (y, sum), for blocks that carry the sum on.  weight and bias (D,) or None; residual
    has x's shape or expands to it (its gradient is summed back)."""
    if (x.requires_grad or (weight is not None and weight.requires_grad) or
            (bias is not None and bias.requires_grad) or
            (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
        if residual is not None and residual.shape != x.shape:
            residual = residual.expand(x.shape)
        return _LayerNorm.apply(x, weight, bias, eps, residual, return_sum)
    y, s, _, _ = layer_norm_forward(x, weight, bias, eps, residual, return_sum)
    return (y, s) if return_sum else y


class LayerNorm(nn.LayerNorm):
    """`nn.LayerNorm` over the last dimension with an optional residual added in front."""

    _abbr_ = 'ln'

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None,
                 dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError('LayerNorm over more than the last dimension')

    def forward(self, x, residual=None, return_sum=False):
        if tuple(x.shape[-1:]) != self.normalized_shape:
            raise RuntimeError(f'expected rows of {self.normalized_shape[0]} elements, got '
                               f'{tuple(x.shape)}')
        return layer_norm(x, self.weight, self.bias, self.eps, residual, return_sum)


if NORM_LAYERS.get('LN') is None:
    NORM_LAYERS.register_module('LN', module=LayerNorm)
