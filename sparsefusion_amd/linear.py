"""Linear layer with its bias, activation and residual in one launch, and its gradients.

`Linear` is `nn.Linear` (same arguments, parameters and state-dict keys) whose forward runs
`sf_linear` (csrc/linear.hip, csrc/gemm_tile.h); `FeedForward` is the two-layer block of the decoders
that read the BEV map.  fp32, fp16 and bf16, all tensors of a call of one type; products and sums are
fp32 and every output is rounded once.  Differentiable once (no double backward) and backwards only: tensors
with forward-mode tangents are refused, and so are torch.jit.trace, make_fx and export.  No CPU path.

With an activation the gradient ahead of it, dz, is rounded to the storage type as well, being an operand of
both products (the bias gradient sums it unrounded): in bf16 dx and dw of 32400 x 512 -> 2048 are 2.3e-3 off, of
which their own rounding is 1.7e-3.  Two operands for dz, high and low part, would double the products.

Capturing a backward pass in a HIP graph follows torch's rule for any operator: no autograd graph
over the same leaves may be alive outside the capture.
"""
import functools

import torch
from torch import nn

from . import _lib
from .registry import LINEAR_LAYERS

MOST_FEATURES = 1 << 20      # in or out: a tile's rows stay in reach of 31-bit offsets
ACTIVATIONS = {None: 0, 'none': 0, 'relu': 1, 'gelu': 2}


def _act_code(activation):
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise RuntimeError(f"activation must be None, 'none', 'relu' or 'gelu' (erf), got {activation!r}")
    return code


def _check(x, weight, device):
    """-> (n, k, dtype code) of a well-formed pair."""
    dtype = x.dtype
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None:
        raise RuntimeError(f'linear takes fp32, fp16 or bf16, got {dtype}')
    if weight.dim() != 2:
        raise RuntimeError(f'weight must be (out_features, in_features), got {tuple(weight.shape)}')
    n, k = weight.shape
    if type(n) is not int:      # torch.jit.trace hands out tensors, and would record allocations, no call
        raise RuntimeError('linear cannot be traced')
    if _lib.dispatch_modes():
        _lib.refuse_tracing('linear')
    if x.dim() < 1 or x.shape[-1] != k:
        raise RuntimeError(f'expected rows of {k} elements, got {tuple(x.shape)}')
    if n > MOST_FEATURES or k > MOST_FEATURES:
        raise RuntimeError(f'linear takes up to {MOST_FEATURES} features, got {k} -> {n}')
    if weight.dtype != dtype or weight.device != device:
        _lib.same(x, 'weight', weight)
    return n, k, code


# Scratch bytes by sizes and by where in 16 bytes the operands start, on which alone the plans depend: asked once.
@functools.lru_cache(maxsize=4096)
def _forward_scratch(x_at, ldx, weight_at, m, k, n, code, residual):
    return _lib.lib().sf_linear_workspace(x_at, ldx, weight_at, m, k, n, code, residual)


@functools.lru_cache(maxsize=4096)
def _backward_scratch(grad_at, x_at, ldx, weight_at, m, k, n, code, act):
    return _lib.lib().sf_linear_backward_workspace(grad_at, x_at, ldx, weight_at, m, k, n, code, act)


def linear_forward(x, weight, bias=None, activation=None, residual=None, keep_pre=False):
    """-> (y, pre): y = act(x @ weight.T + bias) + residual and, with keep_pre, the values before
    the activation (None otherwise).  x (..., K), weight (N, K), bias (N,), residual (..., N) or
    anything that expands to it.  Not differentiable: see `linear`."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        act = _act_code(activation)
    if _lib.forward_ad._current_level >= 0:
        _lib.refuse_tangents('linear', x, weight, bias, residual)
    device = x.device
    n, k, code = _check(x, weight, device)
    if k == 1 or n == 1:
        x, weight, bias, residual = _lib.resolved(x, weight, bias, residual)
    shape = (x.shape[0], n) if x.dim() == 2 else (*x.shape[:-1], n)
    pb = pr = pp = None
    if bias is not None:
        _lib.same(x, 'bias', bias)
        if bias.dim() != 1 or bias.shape[0] != n:
            raise RuntimeError(f'bias must have shape ({n},), got {tuple(bias.shape)}')
        bias = bias.contiguous()
        pb = bias.data_ptr()
    if residual is not None:
        _lib.same(x, 'residual', residual)
        if residual.shape != shape:
            residual = residual.expand(shape)
        residual = residual.contiguous()
        pr = residual.data_ptr()
    if _lib.elsewhere(device):
        with torch.cuda.device(device):
            return linear_forward(x, weight, bias, activation, residual, keep_pre)
    rows, ldx = _lib.rows(x)
    weight = weight.contiguous()
    y = x.new_empty(shape)
    pre = None
    if keep_pre:
        pre = x.new_empty(shape)
        pp = pre.data_ptr()
    m, px, pw, py, stream = rows.shape[0], rows.data_ptr(), weight.data_ptr(), y.data_ptr(), _lib.stream(device)
    nbytes = _forward_scratch(px & 15, ldx, pw & 15, m, k, n, code, pr is not None)
    ws = _lib.workspace(nbytes, x)
    rc = _lib.lib().sf_linear(px, ldx, pw, pb, pr, py, pp, m, k, n, code, act, None if ws is None else ws.data_ptr(),
                              nbytes, stream)
    if rc:
        _lib.check(rc)
    return y, pre


def linear_backward(grad, x, weight, pre=None, activation=None, needs=(True, True, True)):
    """Gradients (dx, dweight, dbias) of `linear_forward` for the gradient `grad` (..., N) of its
    output; `pre` as it returned them (not needed without an activation).  `needs` says which are
    wanted, the others are None.  The residual's gradient is `grad` itself."""
    act = _act_code(activation)
    if _lib.forward_ad._current_level >= 0:
        _lib.refuse_tangents('linear_backward', grad, x, weight, pre)
    n, k, code = _check(x, weight, x.device)
    if k == 1 or n == 1:
        grad, x, weight, pre = _lib.resolved(grad, x, weight, pre)
    shape = (*x.shape[:-1], n)
    if not act:
        pre = None
    elif pre is None:
        raise RuntimeError(f"the gradient of '{activation}' needs the values before it (pre)")
    for name, t in (('grad', grad), ('pre', pre)):
        if t is not None:
            _lib.same(x, name, t)
            if t.shape != shape:
                raise RuntimeError(f'{name} must have shape {shape}, got {tuple(t.shape)}')
    if _lib.elsewhere(x.device):
        with torch.cuda.device(x.device):
            return linear_backward(grad, x, weight, pre, activation, needs)
    rows, ldx = _lib.rows(x)
    m = rows.shape[0]
    grad, weight = grad.contiguous(), weight.contiguous()
    if pre is not None:
        pre = pre.contiguous()
    dx = x.new_empty(x.shape) if needs[0] else None
    dw = x.new_empty((n, k)) if needs[1] else None
    db = x.new_empty(n) if needs[2] else None
    pg, px, pw = grad.data_ptr(), rows.data_ptr(), weight.data_ptr()
    nbytes = _backward_scratch(pg & 15, px & 15, ldx, pw & 15, m, k, n, code, act)
    ws = _lib.workspace(nbytes, x)
    rc = _lib.lib().sf_linear_backward(
        pg, px, ldx, pw, None if pre is None else pre.data_ptr(), None if dx is None else dx.data_ptr(),
        None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), m, k, n, code, act,
        None if ws is None else ws.data_ptr(), nbytes, _lib.stream(x.device))
    if rc:
        _lib.check(rc)
    return dx, dw, db


class _Linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        act = _act_code(activation)
        # a ReLU without a residual shows its sign in the output: nothing more is kept
        own = act == 1 and residual is None
        y, pre = linear_forward(x, weight, bias, activation, residual, keep_pre=bool(act) and not own)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, y if own else pre)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, pre = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dx = dw = db = None
        if any(needs[:3]):
            dx, dw, db = linear_backward(grad, x, weight, pre, ctx.activation, needs[:3])
        return dx, dw, db, None, grad if needs[4] else None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x @ weight.T + bias) + residual, differentiable in all four tensors.  x (..., K), weight
    (N, K), bias (N,); activation None, 'relu' or 'gelu'; residual (..., N) or anything that expands
    to it (its gradient is summed back)."""
    if (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
            (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
        if residual is not None and x.dim() and residual.shape != x.shape[:-1] + weight.shape[:1]:
            residual = residual.expand(x.shape[:-1] + weight.shape[:1])
        return _Linear.apply(x, weight, bias, activation, residual)
    return linear_forward(x, weight, bias, activation, residual)[0]


@LINEAR_LAYERS.register_module()
class Linear(nn.Linear):
    """`nn.Linear` with an optional activation and residual in the same launch."""

    def __init__(self, in_features, out_features, bias=True, activation=None, device=None, dtype=None):
        _act_code(activation)
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self):
        return f'{super().extra_repr()}, activation={self.activation}'


class FeedForward(nn.Module):
    """norm(x + linear2(act(linear1(x)))): the feed-forward part of a post-norm decoder layer, or with
    pre_norm x + linear2(act(linear1(norm(x)))).  Three launches; parameters `linear1`, `linear2`,
    `norm` as nn.TransformerDecoderLayer names the first two."""

    def __init__(self, channels, hidden_channels, activation='relu', pre_norm=False,
                 norm_cfg=dict(type='LN')):
        super().__init__()
        from .registry import build_norm_layer
        self.linear1 = Linear(channels, hidden_channels, activation=activation)
        self.linear2 = Linear(hidden_channels, channels)
        self.norm = build_norm_layer(norm_cfg, channels)[1]
        self.pre_norm = pre_norm

    def forward(self, x):
        if self.pre_norm:
            return self.linear2(self.linear1(self.norm(x)), residual=x)
        return self.norm(self.linear2(self.linear1(x), residual=x))
