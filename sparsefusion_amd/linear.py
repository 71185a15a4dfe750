"""Linear layer with its bias, activation and residual in one launch, and its gradients.

`Linear` is `nn.Linear` (same arguments, parameters and state-dict keys) whose forward runs
`sf_linear` (csrc/linear.hip, csrc/gemm_tile.h); `FeedForward` is the two-layer block of the decoders
that read the BEV map.  fp32, fp16 and bf16, all tensors of a call of one type; products and sums are
fp32 and every output is rounded once.  Differentiable once (no double backward).  No CPU path.

Capturing a backward pass in a HIP graph follows torch's rule for any operator: no autograd graph
over the same leaves may be alive outside the capture.
"""
import torch
from torch import nn

from . import _lib
from .registry import LINEAR_LAYERS

ACTIVATIONS = {None: 0, 'none': 0, 'relu': 1, 'gelu': 2}


def _act_code(activation):
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"activation must be None, 'none', 'relu' or 'gelu' (erf), got {activation!r}")
    return ACTIVATIONS[activation]


def _check(x, weight, bias):
    if x.dtype not in _lib.DTYPE_CODES:
        raise RuntimeError(f'linear takes fp32, fp16 or bf16, got {x.dtype}')
    if weight.dim() != 2:
        raise RuntimeError(f'weight must be (out_features, in_features), got {tuple(weight.shape)}')
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise RuntimeError(f'expected rows of {k} elements, got {tuple(x.shape)}')
    _lib.same(x, weight=weight, bias=bias)
    if bias is not None and tuple(bias.shape) != (n,):
        raise RuntimeError(f'bias must have shape ({n},), got {tuple(bias.shape)}')


def linear_forward(x, weight, bias=None, activation=None, residual=None, keep_pre=False):
    """-> (y, pre): y = act(x @ weight.T + bias) + residual and, with keep_pre, the values before
    the activation (None otherwise).  x (..., K), weight (N, K), bias (N,), residual (..., N) or
    anything that expands to it.  Not differentiable: see `linear`."""
    act = _act_code(activation)
    _check(x, weight, bias)
    n, k = weight.shape
    shape = x.shape[:-1] + (n,)
    rows, ldx = _lib.rows(x)
    m = rows.shape[0]
    if residual is not None:
        _lib.same(x, residual=residual)
        if residual.shape != shape:
            residual = residual.expand(shape)
        residual = residual.contiguous()
    w = weight.contiguous()
    with _lib.on(x.device):
        y = torch.empty(shape, dtype=x.dtype, device=x.device)
        pre = torch.empty(shape, dtype=x.dtype, device=x.device) if keep_pre else None
        dtype = _lib.DTYPE_CODES[x.dtype]
        L = _lib.lib()
        ws, nbytes = _lib.workspace(L.sf_linear_workspace(m, k, n, dtype), x.device)
        _lib.check(L.sf_linear(
            _lib.dev_ptr(rows), ldx, _lib.ptr(w),
            _lib.ptr(bias.contiguous()) if bias is not None else None, _lib.ptr(residual),
            y.data_ptr(), pre.data_ptr() if keep_pre else None, m, k, n, dtype, act, _lib.ptr(ws), nbytes,
            _lib.stream(x.device)))
    return y, pre


def linear_backward(grad, x, weight, pre=None, activation=None, needs=(True, True, True)):
    """Gradients (dx, dweight, dbias) of `linear_forward` for the gradient `grad` (..., N) of its
    output; `pre` as it returned them (not needed without an activation).  `needs` says which are
    wanted, the others are None.  The residual's gradient is `grad` itself."""
    act = _act_code(activation)
    _check(x, weight, None)
    n, k = weight.shape
    shape = x.shape[:-1] + (n,)
    _lib.same(x, grad=grad, pre=pre if act else None)
    if act and pre is None:
        raise RuntimeError(f"the gradient of '{activation}' needs the values before it (pre)")
    for name, t in (('grad', grad), ('pre', pre if act else None)):
        if t is not None and t.shape != shape:
            raise RuntimeError(f'{name} must have shape {tuple(shape)}, got {tuple(t.shape)}')
    rows, ldx = _lib.rows(x)
    m = rows.shape[0]
    grad, w = grad.contiguous(), weight.contiguous()
    pre = pre.contiguous() if act else None
    with _lib.on(x.device):
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if needs[0] else None
        dw = torch.empty((n, k), dtype=x.dtype, device=x.device) if needs[1] else None
        db = torch.empty((n,), dtype=x.dtype, device=x.device) if needs[2] else None
        dtype = _lib.DTYPE_CODES[x.dtype]
        L = _lib.lib()
        ws, nbytes = _lib.workspace(L.sf_linear_backward_workspace(m, k, n, dtype, act), x.device)
        _lib.check(L.sf_linear_backward(
            _lib.ptr(grad), _lib.dev_ptr(rows), ldx, _lib.ptr(w), _lib.ptr(pre), _lib.ptr(dx),
            _lib.ptr(dw), _lib.ptr(db), m, k, n, dtype, act, _lib.ptr(ws), nbytes, _lib.stream(x.device)))
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
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias, residual)):
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
