"""Linear layer (bias, activation and residual in one launch) and layer norm (residual add in front),
forward and backward, against the formulas in float64.

Tolerances are worst-case bounds of the arithmetic, written before any run: u = eps / 2 of the storage
type for each rounding to it, e = 2^-24 for an fp32 operation.  A sum of n fp32 terms in any order is
within (n + 2) e of the sum of the magnitudes; the matrix units may truncate where an fma rounds, so
sums are charged 2 e a term.
"""
import math

import pytest
import torch

from sparsefusion_amd import _lib
from sparsefusion_amd.layer_norm import (LayerNorm, layer_norm, layer_norm_backward,
                                         layer_norm_forward)
from sparsefusion_amd.linear import FeedForward, Linear, linear, linear_backward, linear_forward
from sparsefusion_amd.registry import build_linear_layer, build_norm_layer

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ['f32', 'f16', 'bf16']
E = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the type's subnormals: what a rounding near zero may be off by."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def rand(seed, *shape, dtype=torch.float32, dev='cpu', scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(dev)


def act64(z, act):
    if act == 'relu':
        return z.clamp(min=0)
    if act == 'gelu':
        return z * torch.special.ndtr(z)
    return z


def slope64(z, act):
    if act == 'relu':
        return (z > 0).double()
    if act == 'gelu':
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def phi_err(dtype):
    """What the kernels' normal distribution function is off by: the polynomial inside its logistic form
    is fitted to 2.9e-8 (fp32) and 1.4e-6 (16-bit storage); the logistic's argument, of size at most
    |z| P < 30, carries 6 e, which its slope (at most phi(1.2) z P < 0.45) turns into 2.7 e, exp, sum
    and reciprocal 4 e more."""
    return 2.9e-8 + 7 * E if dtype == torch.float32 else 1.4e-6 + 7 * E


def within(got, want, bound, what=''):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max().item() if got.numel() else -1.0
    assert over <= 0, (what, over, (got - want).abs().max().item())


def check_forward(x, w, b, act, r, y, pre=None):
    """Bound of y: the sum's error, grown by at most 1.13 (the steepest slope of GELU) through the
    activation, GELU's own phi_err, the residual's addition, one rounding."""
    t, k = x.dtype, x.shape[-1]
    xd, wd = x.double(), w.double()
    z, mag = xd @ wd.T, xd.abs() @ wd.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    err = 2 * (k + 4) * E * mag
    if pre is not None:
        within(pre, z, err + u(t) * (z.abs() + err) + tiny(t), 'pre')
    want = act64(z, act)
    err = 1.13 * err + ((phi_err(t) + E) * z.abs() if act == 'gelu' else 0)
    if r is not None:
        err = err + E * (want.abs() + r.double().abs() + err)
        want = want + r.double()
    within(y, want, err + u(t) * (want.abs() + err) + tiny(t), 'y')


def check_backward(dy, x, w, pre, act, dx, dw, db):
    """dz carries phi_err and 6 e (z phi(z) and its exponential) for GELU's slope and, when it is stored
    for the products (an activation), one rounding; the products are sums as above; db sums the unrounded dz."""
    t = x.dtype
    m, (n, k) = x.numel() // max(1, x.shape[-1]), w.shape
    g = dy.double().reshape(-1, n)
    slope_err = torch.zeros_like(g)
    if act in ('relu', 'gelu'):
        z = pre.double().reshape(-1, n)
        if act == 'gelu':
            slope_err = (phi_err(t) + 6 * E) * g.abs()
        g = g * slope64(z, act)
    rounded = (u(t) * g.abs() + tiny(t) if act in ('relu', 'gelu') else 0) + slope_err
    xd, wd = x.double().reshape(-1, k), w.double()
    for got, want, mag, carried, terms in (
            (dx, g @ wd, g.abs() @ wd.abs(), rounded @ wd.abs() if torch.is_tensor(rounded) else 0, n),
            (dw, g.T @ xd, g.abs().T @ xd.abs(), rounded.T @ xd.abs(), m),
            (db, g.sum(0), g.abs().sum(0), slope_err.sum(0), m)):
        if got is None:
            continue
        err = 2 * (terms + 4) * E * mag + carried
        within(got.reshape(want.shape), want, err + u(t) * (want.abs() + err) + tiny(t),
               f'gradient of {tuple(want.shape)}')


# ---------------------------------------------------------------------------------- host side

def test_modules_mirror_torch():
    lin, ref = Linear(12, 7, activation='gelu'), torch.nn.Linear(12, 7)
    assert lin.state_dict().keys() == ref.state_dict().keys()
    lin.load_state_dict(ref.state_dict())
    assert Linear(4, 4, bias=False).bias is None and 'gelu' in repr(lin)
    ln, ref = LayerNorm(12, eps=1e-3), torch.nn.LayerNorm(12)
    assert ln.state_dict().keys() == ref.state_dict().keys() and ln.eps == 1e-3
    name, layer = build_norm_layer(dict(type='LN', eps=1e-4), 16, postfix=2)
    assert name == 'ln2' and isinstance(layer, LayerNorm) and layer.eps == 1e-4
    name, layer = build_norm_layer(dict(type='BN1d'), 16, postfix=1)
    assert name == 'bn1' and isinstance(layer, torch.nn.BatchNorm1d)
    layer = build_linear_layer(dict(type='Linear', activation='relu'), 8, 16)
    assert isinstance(layer, Linear) and layer.activation == 'relu'
    with pytest.raises(KeyError):
        build_linear_layer(dict(type='Nope'), 8, 16)
    assert set(FeedForward(8, 32).state_dict()) == {
        'linear1.weight', 'linear1.bias', 'linear2.weight', 'linear2.bias', 'norm.weight', 'norm.bias'}


def test_refusals_need_no_device():
    x, w, b = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(6)
    for call in (lambda: linear(x, w, b), lambda: layer_norm(x),
                 lambda: linear_backward(torch.zeros(4, 6), x, w),
                 lambda: layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4))):
        with pytest.raises(RuntimeError, match='HIP device'):
            call()
    for call, text in (
            (lambda: linear(x.double(), w.double()), 'fp32, fp16 or bf16'),
            (lambda: linear(x.half(), w), 'weight must be'),
            (lambda: linear(x, w, b.half()), 'bias must be'),
            (lambda: linear(x, w, b, residual=torch.zeros(4, 6).half()), 'residual must be'),
            (lambda: linear(x[:, :7], w), 'rows of 8'),
            (lambda: linear(torch.zeros(()), w), 'rows of 8'),
            (lambda: linear(x, w, torch.zeros(5)), r'shape \(6,\)'),
            (lambda: linear(x, w[0]), 'out_features'),
            (lambda: linear(torch.zeros(1, 1), torch.zeros((1 << 20) + 1, 1)), 'features'),
            (lambda: linear(x, w, activation='tanh'), 'activation'),
            (lambda: Linear(4, 4, activation='swish'), 'activation'),
            (lambda: linear(x, w, residual=torch.zeros(3, 6)), 'expand'),
            (lambda: linear_backward(torch.zeros(4, 5), x, w), 'grad must have shape'),
            (lambda: linear_backward(torch.zeros(4, 6), x, w, activation='relu'), 'pre'),
            (lambda: linear_backward(torch.zeros(4, 6), x, w, b, activation='relu'), 'pre must have'),
            (lambda: layer_norm(x.long()), 'fp32, fp16 or bf16'),
            (lambda: layer_norm(torch.zeros(4, 0)), 'at least one element'),
            (lambda: layer_norm(torch.zeros(1).expand((1 << 32) + 8)), 'rows of up to'),
            (lambda: layer_norm(x, torch.zeros(7)), r'shape \(8,\)'),
            (lambda: layer_norm(x, torch.zeros(8).half()), 'weight and bias'),
            (lambda: layer_norm(x.half(), torch.zeros(8), torch.zeros(8).half()), 'weight and bias'),
            (lambda: layer_norm(x, eps=-1.0), 'eps'),
            (lambda: layer_norm(x, residual=x.half()), 'residual must be'),
            (lambda: layer_norm(x, residual=x[:3]), 'expand'),
            (lambda: layer_norm_backward(x[:3], x, torch.zeros(4), torch.zeros(4)), 'grad must have'),
            (lambda: layer_norm_backward(x, x, torch.zeros(3), torch.zeros(4)), 'mean must be'),
            (lambda: layer_norm_backward(x, x, torch.zeros(4), torch.zeros(4).half()), 'rstd must be'),
            (lambda: LayerNorm(8)(torch.zeros(4, 7)), 'rows of 8')):
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises(NotImplementedError):
        LayerNorm((4, 8))
    from sparsefusion_amd.voxel_encoder import HardVFE
    with pytest.raises(NotImplementedError, match='BatchNorm'):
        HardVFE(in_channels=5, feat_channels=[64], norm_cfg=dict(type='LN'))
    HardVFE(in_channels=5, feat_channels=[64], norm_cfg=dict(type='BN', eps=1e-3))


def test_a_callers_own_norm_layers_keep_their_names():
    from sparsefusion_amd.registry import NORM_LAYERS

    class Own(torch.nn.LayerNorm):
        pass

    old = dict(NORM_LAYERS._modules)
    try:
        NORM_LAYERS._modules.pop('LN', None)
        NORM_LAYERS.register_module('LN', module=Own)
        for _ in range(2):
            name, layer = build_norm_layer(dict(type='LN'), 8, postfix=1)
            assert name == 'bn1' and type(layer) is Own
    finally:
        NORM_LAYERS._modules.clear()
        NORM_LAYERS._modules.update(old)
    assert isinstance(build_norm_layer(dict(type='LN'), 8)[1], LayerNorm)


def test_c_entry_points_refuse_bad_arguments():
    L = _lib.lib()
    one = 64      # never dereferenced: every call below is refused or empty
    assert L.sf_linear(one, 8, one, None, None, one, None, 4, 8, 4, 7, 0, None, 0, None) == -1
    assert L.sf_linear(one, 8, one, None, None, one, None, 4, 8, 4, 0, 3, None, 0, None) == -1
    assert L.sf_linear(one, 7, one, None, None, one, None, 4, 8, 4, 0, 0, None, 0, None) == -1
    assert b'apart' in L.sf_last_error()
    assert L.sf_linear(None, 8, one, None, None, one, None, 4, 8, 4, 0, 0, None, 0, None) == -1
    assert L.sf_linear(one, 8, one, None, None, one, None, -1, 8, 4, 0, 0, None, 0, None) == -1
    assert L.sf_linear(None, 8, None, None, None, None, None, 0, 8, 4, 0, 0, None, 0, None) == 0
    need = L.sf_linear_workspace(one, 8192, one, 80, 8192, 64, 0, 0)      # a contraction in parts
    assert need > 0
    assert L.sf_linear(one, 8192, one, None, None, one, None, 80, 8192, 64, 0, 0, one, need - 1, None) == -2
    assert b'workspace' in L.sf_last_error()
    assert L.sf_linear_workspace(one, 64, one, 80, 64, 64, 0, 0) == 0
    assert L.sf_linear_workspace(one + 4, 67, one, 80, 64, 64, 0, 0) == 0
    need = L.sf_linear_workspace(one, 65, one, 80, 64, 64, 1, 0)      # a copy of x
    assert need >= 80 * 64 * 2
    assert L.sf_linear(one, 65, one, None, None, one, None, 80, 64, 64, 1, 0, one, need - 1, None) == -2
    assert L.sf_linear(one, 65, one, None, None, one, None, 80, 64, 64, 1, 0, one + 4, need, None) == -1
    assert b'aligned' in L.sf_last_error()
    assert L.sf_linear_backward(one, one, 8, one, None, one, one, one, 4, 8, 4, 0, 2, None, 0, None) == -1
    need = L.sf_linear_backward_workspace(one, one, 32, one, 6400, 32, 32, 2, 2)
    assert need >= 6400 * 32 * 2
    assert L.sf_linear_backward(one, one, 32, one, one, one, one, one, 6400, 32, 32, 2, 2, one, need - 1,
                                None) == -2
    assert L.sf_linear_workspace(one, 4, one, -1, 4, 4, 0, 0) == 0
    assert L.sf_linear_backward_workspace(one, one, 4, one, 4, 4, 4, 9, 0) == 0
    assert L.sf_layer_norm(one, None, None, None, one, None, None, None, 4, 0, 1e-5, 0, 0, None) == -1
    assert L.sf_layer_norm(one, None, None, None, one, None, None, None, 4, 8, 1e-5, 1, 2, None) == -1
    assert L.sf_layer_norm(one, None, None, None, None, None, None, None, 4, 8, 1e-5, 0, 0, None) == -1
    assert L.sf_layer_norm(None, None, None, None, None, None, None, None, 0, 8, 1e-5, 0, 0, None) == 0
    for m, d in ((4, (1 << 29) + 1), (4, -1), (-1, 8)):
        assert L.sf_layer_norm(one, None, None, None, one, None, None, None, m, d, 1e-5, 0, 0, None) == -1
        assert L.sf_layer_norm_backward(one, one, one, one, None, None, one, None, None, m, d, 0, 0, None,
                                        0, None) == -1
    need = L.sf_layer_norm_backward_workspace(100, 32, 0)
    assert need >= 2 * 32 * 4
    assert L.sf_layer_norm_backward(one, one, one, one, None, None, one, one, one, 100, 32, 0, 0, one,
                                    need - 1, None) == -2
    assert L.sf_layer_norm_backward(one, one, None, one, None, None, one, None, None, 100, 32, 0, 0,
                                    None, 0, None) == -1


def test_rows_are_viewed_where_strides_allow():
    x = torch.arange(60.0).reshape(3, 4, 5)
    assert _lib.rows(x)[0].data_ptr() == x.data_ptr() and _lib.rows(x)[1] == 5
    flat, ld = _lib.rows(x[:, 1, 1:4])
    assert flat.data_ptr() == x[:, 1, 1:].data_ptr() and ld == 20
    for t in (x.transpose(1, 2), x[:1, :1].expand(2, 4, 5), x[..., ::2], x[:, :, :1].expand(3, 4, 5)):
        flat, ld = _lib.rows(t)
        assert torch.equal(flat, t.reshape(-1, t.shape[-1])) and ld >= t.shape[-1]
        assert flat.stride(1) == 1 or flat.shape[1] == 1
    assert _lib.rows(x[0, 0])[0].shape == (1, 5) and _lib.rows(torch.zeros(3, 0))[0].shape == (3, 0)
    assert _lib.rows(torch.zeros(0, 7))[1] == 7


# ---------------------------------------------------------------------------------- linear

# rows, in, out: one row, fewer than a tile, tile borders +- 1, odd everything, long contractions
# (cut into parts), wide outputs
SIZES = [(1, 64, 64), (1, 1, 1), (3, 7, 5), (64, 64, 64), (65, 127, 63), (129, 128, 130),
         (200, 128, 256), (127, 451, 333), (257, 96, 129), (5, 8192, 40), (1, 4100, 1000),
         (1500, 200, 520), (2100, 64, 1024),
         (16, 72, 48), (17, 33, 31), (64, 1023, 65), (65, 3, 2)]
# enough tiles for the larger shapes, whole, split and cut at the edges
LARGE = [(4000, 512, 1024), (9000, 1024, 1000), (16300, 800, 1016), (2000, 4096, 4096)]
# rows that end inside a 16-byte chunk: one step of k and many, whole and in parts, each shape of tile
CUT = [(20001, 30, 514), (7002, 90, 1030), (300, 4098, 70), (3000, 2050, 202), (9001, 1027, 1001),
       (40, 66, 2050), (6, 4098, 34), (500, 62, 62)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,k,n', SIZES + LARGE + CUT)
def test_linear_matches_float64(dev, dtype, m, k, n):
    x, w = rand(1, m, k, dtype=dtype, dev=dev), rand(2, n, k, dtype=dtype, dev=dev, scale=k ** -0.5)
    b, r = rand(3, n, dtype=dtype, dev=dev), rand(4, m, n, dtype=dtype, dev=dev)
    for act, bias, res, keep in ((None, None, None, False), ('relu', b, None, True),
                                 ('gelu', b, r, True), ('none', b, r, False), ('gelu', None, None, False)):
        y, pre = linear_forward(x, w, bias, act, res, keep)
        assert y.dtype == dtype and (pre is not None) == keep
        check_forward(x, w, bias, act, res, y, pre)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,k,n', SIZES + LARGE + CUT + [(40000, 72, 48), (33, 300, 1111), (40000, 64, 1024)])
def test_linear_backward_matches_float64(dev, dtype, m, k, n):
    x, w = rand(1, m, k, dtype=dtype, dev=dev), rand(2, n, k, dtype=dtype, dev=dev, scale=k ** -0.5)
    dy, z = rand(3, m, n, dtype=dtype, dev=dev), rand(4, m, n, dtype=dtype, dev=dev)
    for act in (None, 'relu', 'gelu'):
        dx, dw, db = linear_backward(dy, x, w, z, act)
        check_backward(dy, x, w, z, act, dx, dw, db)
    only = linear_backward(dy, x, w, z, 'gelu', needs=(False, True, False))
    assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
    only = linear_backward(dy, x, w, z, 'gelu', needs=(True, False, True))
    assert torch.equal(only[0], dx) and only[1] is None and torch.equal(only[2], db)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_linear_strides_alignment_and_shapes(dev, dtype):
    w, b = rand(2, 96, 64, dtype=dtype, dev=dev, scale=0.125), rand(3, 96, dtype=dtype, dev=dev)
    wide = rand(1, 50, 200, dtype=dtype, dev=dev)
    for x in (wide[:, :64], wide[:, 3:67], wide[:, 8:72], wide[::2, 16:80], wide[:, :128:2],
              wide[7, 5:69], wide[:, :64].reshape(5, 10, 64), wide[:, :64].reshape(5, 10, 64).transpose(0, 1),
              rand(5, 64, 70, dtype=dtype, dev=dev).t(), wide[:1, :64].expand(9, 64)):
        y = linear(x, w, b, 'gelu')
        assert y.shape == x.shape[:-1] + (96,) and y.is_contiguous()
        check_forward(x, w, b, 'gelu', None, y)
        dy = rand(6, *y.shape, dtype=dtype, dev=dev)
        check_backward(dy, x, w, None, None, *linear_backward(dy, x, w))
    # parameters that are views of a larger block, off the 16-byte grid
    block = rand(7, 300, 64, dtype=dtype, dev=dev)
    x = wide[:, :64]
    flat = block.reshape(-1)
    for wv in (block[96:192], flat[1:1 + 96 * 64].view(96, 64), block[:96, :].flip(0),
               rand(8, 64, 96, dtype=dtype, dev=dev).t()):
        check_forward(x, wv, flat[5:101], 'relu', None, linear(x, wv, flat[5:101], 'relu'))
    # residuals that expand or are strided
    for r in (rand(9, 96, dtype=dtype, dev=dev), rand(9, 50, 1, dtype=dtype, dev=dev),
              rand(9, 50, 200, dtype=dtype, dev=dev)[:, 1:97]):
        check_forward(x, w, b, None, r.expand(50, 96), linear(x, w, b, residual=r))
    # nothing behind or between the rows that are read
    guard = torch.full((50, 200), float('nan'), dtype=dtype, device=dev)
    guard[:, 8:72] = x
    assert torch.isfinite(linear(guard[:, 8:72], w, b)).all()
    guard = torch.full((50, 71), float('nan'), dtype=dtype, device=dev)
    guard[:, 3:67] = x
    assert torch.isfinite(linear(guard[:, 3:67], w, b)).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_linear_empty_sizes(dev, dtype):
    z = lambda *s: torch.zeros(s, dtype=dtype, device=dev)
    b, r = rand(3, 5, dtype=dtype, dev=dev), rand(4, 6, 5, dtype=dtype, dev=dev)
    assert linear(z(0, 8), z(5, 8), b).shape == (0, 5)
    assert linear(z(2, 0, 8), z(5, 8), b).shape == (2, 0, 5)
    assert linear(z(6, 8), z(0, 8)).shape == (6, 0)
    y = linear(z(6, 0), z(5, 0), b, 'relu', r)      # a sum of nothing
    assert torch.equal(y, (b.float().clamp(min=0) + r.float()).to(dtype))
    dx, dw, db = linear_backward(z(0, 5), z(0, 8), z(5, 8))
    assert dx.shape == (0, 8) and not dw.any() and dw.shape == (5, 8) and not db.any()
    dx, dw, db = linear_backward(z(6, 0), z(6, 8) + 1, z(0, 8))
    assert not dx.any() and dx.shape == (6, 8) and dw.shape == (0, 8) and db.shape == (0,)
    dx, dw, db = linear_backward(r, z(6, 0), z(5, 0), r, 'relu')
    assert dx.shape == (6, 0) and dw.shape == (5, 0)
    within(db, r.double().clamp(min=0).sum(0), 0.05)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_linear_infinities_and_nan_stay_in_their_rows(dev, dtype):
    x, w = rand(1, 130, 64, dtype=dtype, dev=dev), rand(2, 70, 64, dtype=dtype, dev=dev).abs() + 1
    clean = linear(x, w)
    x2 = x.clone()
    x2[3, 5], x2[77, 63], x2[129, 0] = float('inf'), float('nan'), -float('inf')
    y = linear(x2, w)
    hit = torch.zeros(130, dtype=torch.bool, device=dev)
    hit[[3, 77, 129]] = True
    assert torch.equal(y[~hit], clean[~hit])
    assert (y[3] == float('inf')).all() and y[77].isnan().all() and (y[129] == -float('inf')).all()
    act = linear(x2, w, activation='relu')
    assert (act[3] == float('inf')).all() and act[77].isnan().all() and not act[129].any()
    # what ReLU blocks stays blocked, whatever it is
    for m in (130, 9000):
        x, z = rand(3, m, 64, dtype=dtype, dev=dev), rand(4, m, 70, dtype=dtype, dev=dev)
        dy = rand(5, m, 70, dtype=dtype, dev=dev)
        masked = dy.masked_fill(z <= 0, 0)
        dy[z <= 0] = torch.tensor([float('inf'), float('nan'), -float('inf')], dtype=dtype,
                                  device=dev).repeat(m * 70)[:int((z <= 0).sum())]
        got, want = linear_backward(dy, x, w, z, 'relu'), linear_backward(masked, x, w, z, 'relu')
        assert all(torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,k,n', [(130, 62, 70), (3000, 94, 602), (20001, 30, 514), (300, 4098, 70), (5, 30, 34)])
def test_linear_nothing_leaks_behind_a_cut_row(dev, dtype, m, k, n):
    """Rows that end inside a chunk lie against the next row's first values: those may be anything."""
    x, w = rand(1, m, k, dtype=dtype, dev=dev), rand(2, n, k, dtype=dtype, dev=dev)
    dy = rand(3, m, n, dtype=dtype, dev=dev)
    bad = torch.arange(m, device=dev) % 3 == 1
    x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
    x2[bad, 0], dy2[bad, 0] = float('nan'), float('inf')
    y, y2 = linear(x, w), linear(x2, w)
    assert torch.equal(y2[~bad], y[~bad]) and y2[bad].isnan().all()
    odd = torch.arange(n, device=dev) % 3 == 1
    w2[odd, :1] = float('nan')
    y2 = linear(x, w2)
    assert torch.equal(y2[:, ~odd], y[:, ~odd]) and y2[:, odd].isnan().all()
    dx, dx2 = linear_backward(dy, x, w)[0], linear_backward(dy2, x, w)[0]
    assert torch.equal(dx2[~bad], dx[~bad]) and not torch.isfinite(dx2[bad]).any()
    # behind the last row: a view of a larger tensor whose rest is not finite
    room = torch.full((m * k + 64,), float('nan'), dtype=dtype, device=dev)
    room[:m * k] = x.flatten()
    assert torch.equal(linear(room[:m * k].view(m, k), w), y)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_linear_autograd_and_differences(dev, dtype):
    """Gradients through autograd are linear_backward's on what the forward kept; in fp32 they also
    follow central differences of the kernel itself (loss = <y, c>; the quotient is off by the third
    derivative times h^2 and by the forward's own error over h)."""
    x, w = rand(1, 2, 33, 40, dtype=dtype, dev=dev), rand(2, 24, 40, dtype=dtype, dev=dev, scale=0.16)
    b, r = rand(3, 24, dtype=dtype, dev=dev), rand(4, 33, 24, dtype=dtype, dev=dev)
    c = rand(5, 2, 33, 24, dtype=dtype, dev=dev)
    for act in (None, 'relu', 'gelu'):
        for res in (None, r):
            leaves = [t.clone().requires_grad_() for t in (x, w, b)]
            rl = res.clone().requires_grad_() if res is not None else None
            y = linear(*leaves, act, rl)
            y.backward(c)
            pre = linear_forward(x, w, b, act, res, True)[1]
            check_backward(c, x, w, pre, act, *(t.grad for t in leaves))
            if rl is not None:      # broadcast over the first axis: summed back
                assert torch.equal(rl.grad, c.sum(0))
    if dtype == torch.float32:
        h = 2.0 ** -7
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        linear(*leaves, 'gelu').backward(c)
        for i, t in enumerate(leaves):
            d = rand(6 + i, *t.shape, dev=dev)
            with torch.no_grad():
                f = []
                for s in (h, -h):
                    args = [a + s * d if a is t else a for a in leaves]
                    f.append((linear(*args, 'gelu').double() * c.double()).sum().item())
            want = (f[0] - f[1]) / (2 * h)
            got = (t.grad.double() * d.double()).sum().item()
            # |gelu'''| <= 1.6 on |dz|^3 of at most 8^3 an element; 1584 outputs of error 1e-5 over h
            assert abs(got - want) <= 1584 * (1.6 / 6 * 16 * h * h + 1e-5 / h), (i, got, want)


@pytest.mark.gpu
def test_linear_gradients_only_where_asked_and_no_double_backward(dev):
    x, w = rand(1, 9, 16, dev=dev), rand(2, 8, 16, dev=dev)
    wl = w.clone().requires_grad_()
    y = linear(x, wl, activation='relu')
    g, = torch.autograd.grad(y.sum(), wl, create_graph=False)
    check_backward(torch.ones_like(y), x, w, y.detach(), 'relu', None, g, None)
    xl = x.clone().requires_grad_()
    g, = torch.autograd.grad(linear(xl, wl, activation='gelu').sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.no_grad():
        assert not linear(xl, wl).requires_grad
    y = linear(xl, wl, activation='relu')
    y.add_(1)      # the kept output was changed: torch refuses, no silent wrong gradient
    with pytest.raises(RuntimeError, match='modified'):
        y.sum().backward()


# ---------------------------------------------------------------------------------- layer norm

NORM_SIZES = [(1, 1), (1, 64), (3, 7), (200, 128), (33, 256), (50, 333), (17, 512), (9, 1000),
              (21, 2048), (6, 4097), (5, 8192), (3, 16384), (2, 20001), (5000, 96), (70000, 40), (110000, 333), (70000, 512)]


def norm64(x, w, b, eps, r=None):
    s = x.double() + (r.double() if r is not None else 0)
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((s - mean).square().mean(-1, keepdim=True) + eps)
    xh = (s - mean) * rstd
    y = xh * (w.double() if w is not None else 1) + (b.double() if b is not None else 0)
    return s, mean, rstd, xh, y


def check_norm(x, w, b, eps, r, out, mean, rstd, y):
    """A lane adds at most D / 64 + 16 terms, then 6 steps across a wave and 16 across waves: a sum's
    error is (D / 64 + 48) e of the magnitudes.  The mean's error shifts xh by that times rstd (once
    in s - mean, and it cancels in the variance to second order); rstd carries half the variance's
    relative error, its own square root and division; the rest are single operations."""
    t, d = x.dtype, x.shape[-1]
    s64, m64, r64, xh, y64 = norm64(x, w, b, eps, r)
    ge = (d / 64 + 48) * E
    mag = s64.abs()
    add = E * (x.double().abs() + r.double().abs()) if r is not None else 0 * mag
    dm = ge * mag.mean(-1, keepdim=True) + add.mean(-1, keepdim=True) + E * m64.abs()
    dc = dm + add + E * (s64 - m64).abs()                       # error of the centred value
    spread = ((s64 - m64).square().mean(-1, keepdim=True) + 1e-300).sqrt()
    dv = 2 * spread * dc.square().mean(-1, keepdim=True).sqrt() + dc.square().mean(-1, keepdim=True) \
        + ge * spread.square()
    dr = r64 * (0.5 * dv * r64.square() * (1 + dv * r64.square()) + 4 * E)
    dxh = dc * (r64 + dr) + (s64 - m64).abs() * dr + 2 * E * xh.abs()
    wa = w.double().abs() if w is not None else 1
    err = dxh * wa + 2 * E * (xh.abs() * wa) + E * y64.abs()
    if out is not None:
        within(out, s64, add + u(t) * (mag + add) + tiny(t), 'sum')
    if mean is not None:
        within(mean, m64[..., 0], dm[..., 0], 'mean')
        within(rstd, r64[..., 0], dr[..., 0] + E * r64[..., 0], 'rstd')
    within(y, y64, err + u(t) * (y64.abs() + err) + tiny(t), 'y')


def check_norm_backward(dy, x, mean, rstd, w, ds, dx, dw, db):
    """From the statistics handed over: xh carries 2 e; the two row sums (D / 64 + 48) e of their
    magnitudes, columns (rows + 64) e of theirs."""
    t, d = x.dtype, x.shape[-1]
    m = x.numel() // d
    g, xd = dy.double().reshape(m, d), x.double().reshape(m, d)
    mu, rs = mean.double().reshape(m, 1), rstd.double().reshape(m, 1)
    xh = (xd - mu) * rs
    xe = E * (2 * xh.abs() + (xd.abs() + mu.abs()) * rs)
    wd = w.double() if w is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    gw = g * wd
    ge = (d / 64 + 52) * E
    s1, s2 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    e1 = ge * gw.abs().mean(1, keepdim=True)
    e2 = ge * (gw * xh).abs().mean(1, keepdim=True) + (gw.abs() * xe).mean(1, keepdim=True)
    want = rs * (gw - s1 - xh * s2)
    err = rs * (4 * E * (gw.abs() + s1.abs() + (xh * s2).abs()) + e1 + xh.abs() * e2 + xe * s2.abs())
    if ds is not None:
        want = want + ds.double().reshape(m, d)
        err = err + E * (ds.double().reshape(m, d).abs() + want.abs())
    if dx is not None:
        within(dx.reshape(m, d), want, err + u(t) * (want.abs() + err) + tiny(t), 'dx')
    for got, cols, ce in ((dw, g * xh, g.abs() * xe), (db, g, 0 * g)):
        if got is not None:
            want = cols.sum(0)
            err = (m + 64) * E * cols.abs().sum(0) + ce.sum(0)
            within(got, want, err + u(got.dtype) * (want.abs() + err) + tiny(got.dtype), 'columns')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,d', NORM_SIZES)
def test_layer_norm_matches_float64(dev, dtype, m, d):
    x, r = rand(1, m, d, dtype=dtype, dev=dev, shift=0.5), rand(2, m, d, dtype=dtype, dev=dev)
    for pd in {dtype, torch.float32}:
        w, b = rand(3, d, dtype=pd, dev=dev, shift=1.0), rand(4, d, dtype=pd, dev=dev)
        for wi, bi, ri, total in ((w, b, r, True), (None, None, None, False), (w, None, None, True),
                                  (None, b, r, False)):
            y, s, mean, rstd = layer_norm_forward(x, wi, bi, 1e-5, ri, total, keep_stats=True)
            assert (s is not None) == total and y.dtype == dtype
            check_norm(x, wi, bi, 1e-5, ri, s, mean, rstd, y)
    y2 = layer_norm(x, None, b, residual=r)
    assert torch.equal(y2, y)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,d', NORM_SIZES)
def test_layer_norm_backward_matches_float64(dev, dtype, m, d):
    x, dy = rand(1, m, d, dtype=dtype, dev=dev, shift=0.5), rand(2, m, d, dtype=dtype, dev=dev)
    ds = rand(5, m, d, dtype=dtype, dev=dev)
    _, _, mean, rstd = layer_norm_forward(x, keep_stats=True)
    for pd in {dtype, torch.float32}:
        w = rand(3, d, dtype=pd, dev=dev, shift=1.0)
        for wi, si in ((w, ds), (w, None), (None, ds)):
            dx, dw, db = layer_norm_backward(dy, x, mean, rstd, wi, si, param_dtype=pd)
            assert dw.dtype == pd == db.dtype
            check_norm_backward(dy, x, mean, rstd, wi, si, dx, dw, db)
    one = layer_norm_backward(dy, x, mean, rstd, None, ds, needs=(True, False, False))
    assert torch.equal(one[0], dx) and one[1] is None and one[2] is None


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_layer_norm_hard_rows(dev, dtype):
    """Rows without spread, a large common offset, infinities and NaN."""
    w, b = rand(3, 320, dtype=dtype, dev=dev), rand(4, 320, dtype=dtype, dev=dev)
    x = rand(1, 40, 320, dtype=dtype, dev=dev)
    x[0] = 0
    x[1] = 100
    x[2] = 100
    x[2, 7] += 1
    x[3] = rand(6, 320, dtype=dtype, dev=dev) + 250
    y, _, mean, rstd = layer_norm_forward(x, w, b, 1e-5, keep_stats=True)
    check_norm(x, w, b, 1e-5, None, None, mean, rstd, y)
    assert torch.equal(y[0], b)
    bad = x.clone()
    bad[5, 9], bad[6, 319] = float('inf'), float('nan')
    y2 = layer_norm(bad, w, b)
    assert y2[5].isnan().all() and y2[6].isnan().all()
    keep = [i for i in range(40) if i not in (5, 6)]
    assert torch.equal(y2[keep], y[keep])
    for d in (333, 40):      # the columns behind a row's end never enter it
        wide = torch.full((8, d + 3), float('nan'), dtype=dtype, device=dev)
        wide[:, :d] = rand(7, 8, d, dtype=dtype, dev=dev)
        assert torch.isfinite(layer_norm(wide[:, :d])).all()
        flat = torch.full((d + 64,), float('inf'), dtype=dtype, device=dev)
        flat[1:1 + d] = wide[0, :d]
        check_norm(flat[1:1 + d], None, None, 1e-5, None, None, None, None, layer_norm(flat[1:1 + d]))
    big = torch.full((4, 64), torch.finfo(dtype).max / 4, dtype=dtype, device=dev)
    assert not layer_norm(big).any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_layer_norm_strides_and_empty(dev, dtype):
    base = rand(1, 6, 90, 70, dtype=dtype, dev=dev)
    w, b = rand(3, 90, dtype=dtype, dev=dev), rand(4, 90, dtype=dtype, dev=dev)
    tokens = base.permute(0, 2, 1)      # cells of a (B, C, H W) map
    check_norm(tokens, w, b, 1e-5, None, None, None, None, layer_norm(tokens, w, b))
    r = rand(5, 70, 90, dtype=dtype, dev=dev)      # expands over the batch
    y, s = layer_norm(tokens, w, b, residual=r, return_sum=True)
    check_norm(tokens, w, b, 1e-5, r.expand(tokens.shape), s, None, None, y)
    odd = rand(6, 12, 91, dtype=dtype, dev=dev)[:, 1:]
    check_norm(odd, w, b, 1e-5, None, None, None, None, layer_norm(odd, w, b))
    e = torch.zeros((0, 90), dtype=dtype, device=dev)
    y, s = layer_norm(e, w, b, residual=e, return_sum=True)
    assert y.shape == s.shape == (0, 90)
    z = torch.zeros(0, device=dev)
    dx, dw, db = layer_norm_backward(e, e, z, z, w)
    assert dx.shape == (0, 90) and dw.shape == (90,) and not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_layer_norm_autograd_and_differences(dev, dtype):
    x, r = rand(1, 2, 30, 72, dtype=dtype, dev=dev), rand(2, 30, 72, dtype=dtype, dev=dev)
    w, b = rand(3, 72, dtype=dtype, dev=dev, shift=1.0), rand(4, 72, dtype=dtype, dev=dev)
    c, cs = rand(5, 2, 30, 72, dtype=dtype, dev=dev), rand(6, 2, 30, 72, dtype=dtype, dev=dev)
    for res, total in ((None, False), (r, False), (r, True), (None, True)):
        lx, lw, lb = (t.clone().requires_grad_() for t in (x, w, b))
        lr = res.clone().requires_grad_() if res is not None else None
        out = layer_norm(lx, lw, lb, residual=lr, return_sum=total)
        torch.autograd.backward(out if total else [out], [c, cs] if total else [c])
        re = res.expand(x.shape) if res is not None else None
        _, s, mean, rstd = layer_norm_forward(x, w, b, 1e-5, re, True, True)
        dx, dw, db = layer_norm_backward(c, x if res is None else s, mean, rstd, w, cs if total else None)
        check_norm_backward(c, x if res is None else s, mean, rstd, w, cs if total else None, dx, dw, db)
        assert torch.equal(lx.grad, dx) and torch.equal(lw.grad, dw) and torch.equal(lb.grad, db)
        if lr is not None:
            assert torch.equal(lr.grad, dx.sum(0))
    lx = x.clone().requires_grad_()      # only the sum is used further on
    _, s = layer_norm(lx, w, b, residual=r, return_sum=True)
    s.backward(cs)
    want = norm64(x, w, b, 1e-5, r)
    assert torch.equal(lx.grad, cs) and want[0].shape == s.shape
    if dtype == torch.float32:
        h = 2.0 ** -7
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        layer_norm(*leaves).backward(c)
        for i, t in enumerate(leaves):
            d = rand(7 + i, *t.shape, dev=dev)
            with torch.no_grad():
                f = [(layer_norm(*[a + k * d if a is t else a for a in leaves]).double()
                      * c.double()).sum().item() for k in (h, -h)]
            want = (f[0] - f[1]) / (2 * h)
            got = (t.grad.double() * d.double()).sum().item()
            # 4320 outputs: third derivative of order 10 |d|^3 / 6, forward error 2e-6 over h
            assert abs(got - want) <= 4320 * (10 * h * h + 2e-6 / h), (i, got, want)


# ---------------------------------------------------------------------------------- together

def feed_forward64(ff, x):
    p = {k: v.detach().double() for k, v in ff.state_dict().items()}
    norm = lambda t: torch.nn.functional.layer_norm(t, t.shape[-1:], p['norm.weight'], p['norm.bias'])
    h = norm(x) if ff.pre_norm else x
    h = act64(h @ p['linear1.weight'].T + p['linear1.bias'], ff.linear1.activation)
    t = x + h @ p['linear2.weight'].T + p['linear2.bias']
    return t if ff.pre_norm else norm(t)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('pre_norm', [False, True])
def test_feed_forward_block(dev, dtype, pre_norm):
    """The run as a decoder makes it: three launches forward, gradients of every parameter back.  Three
    roundings to the storage type forward and as many back, each u of values of order one, behind
    layers whose gain is below 4: 16 u of the largest value (plus fp32 sums, far below)."""
    torch.manual_seed(0)
    ff = FeedForward(128, 256, 'gelu', pre_norm).to(dev).to(dtype)
    x = rand(1, 2, 200, 128, dtype=dtype, dev=dev).requires_grad_()
    c = rand(2, 2, 200, 128, dtype=dtype, dev=dev)
    y = ff(x)
    y.backward(c)
    ref = FeedForward(128, 256, 'gelu', pre_norm).to(dev).double()
    ref.load_state_dict({k: v.double() for k, v in ff.state_dict().items()})
    xd = x.detach().double().requires_grad_()
    leaves = dict(ref.named_parameters())

    def run64(xx, p):
        norm = lambda t: torch.nn.functional.layer_norm(t, (128,), p['norm.weight'], p['norm.bias'])
        h = norm(xx) if pre_norm else xx
        z = h @ p['linear1.weight'].T + p['linear1.bias']
        t = xx + (z * torch.special.ndtr(z)) @ p['linear2.weight'].T + p['linear2.bias']
        return t if pre_norm else norm(t)

    yd = run64(xd, leaves)
    yd.backward(c.double())
    tol = 16 * u(dtype) + 2000 * E
    within(y.detach(), yd.detach(), tol * yd.abs().max().item() * torch.ones_like(yd), 'y')
    within(x.grad, xd.grad, tol * xd.grad.abs().max().item() * torch.ones_like(xd), 'dx')
    for name, p in ff.named_parameters():
        want = leaves[name].grad
        within(p.grad, want, tol * want.abs().max().item() * torch.ones_like(want), name)
    within(feed_forward64(ff, xd.detach()), yd.detach(), 1e-9 + 0 * yd.detach())


@pytest.mark.gpu
def test_layer_norm_inside_a_sparse_block(dev):
    """norm_cfg type LN in the sparse convolution path: SubM conv -> LN -> ReLU on the voxel features."""
    from sparsefusion_amd.sparse_block import SparseBasicBlock, make_sparse_convmodule
    from sparsefusion_amd.spconv import SparseConvTensor
    torch.manual_seed(1)
    idx = torch.unique(torch.randint(0, 12, (400, 3), generator=torch.Generator().manual_seed(2)), dim=0)
    idx = torch.cat([torch.zeros(len(idx), 1, dtype=idx.dtype), idx], 1).int().to(dev)
    feats = rand(3, idx.shape[0], 16, dev=dev)
    x = SparseConvTensor(feats, idx, [12, 12, 12], 1)
    mod = make_sparse_convmodule(16, 32, 3, 'k', padding=1, norm_cfg=dict(type='LN')).to(dev).eval()
    with torch.no_grad():
        bare = mod[0](x).features
        y = mod(x).features
    assert isinstance(mod[1], LayerNorm)
    want = norm64(bare, mod[1].weight, mod[1].bias, 1e-5)[4].clamp(min=0)
    within(y, want, 1e-5 * (1 + want.abs()))
    block = SparseBasicBlock(16, 16, norm_cfg=dict(type='LN')).to(dev).eval()
    assert hasattr(block, 'ln1') and block.norm2 is block.ln2
    with torch.no_grad():
        assert torch.isfinite(block(x).features).all()


@pytest.mark.gpu
def test_two_streams_and_replayed_graphs(dev):
    """Calls on side streams, and forward + backward captured once and replayed on new contents with
    eager calls between the replays: every replay equals the eager result bit for bit."""
    dtype = torch.bfloat16
    w, b = rand(2, 96, 4096, dtype=dtype, dev=dev, scale=0.02), rand(3, 96, dtype=dtype, dev=dev)
    nw, nb = rand(4, 96, dtype=dtype, dev=dev), rand(5, 96, dtype=dtype, dev=dev)

    def step(x, dy):
        y, pre = linear_forward(x, w, b, 'gelu', None, True)      # cut along k: uses scratch memory
        o, s, mean, rstd = layer_norm_forward(y, nw, nb, 1e-5, dy, True, True)
        dn, dnw, dnb = layer_norm_backward(dy, s, mean, rstd, nw, dy)
        dx, dw, db = linear_backward(dn, x, w, pre, 'gelu')
        return y, o, s, dn, dnw, dnb, dx, dw, db

    xs = [rand(10 + i, 70, 4096, dtype=dtype, dev=dev) for i in range(3)]
    ds = [rand(20 + i, 70, 96, dtype=dtype, dev=dev) for i in range(3)]
    want = [step(x, d) for x, d in zip(xs, ds)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for rep in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = step(xs[i], ds[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))
    graphs, ins, outs = [], [], []
    for i in range(2):
        x, d = xs[i].clone(), ds[i].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, d)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(x, d)
        graphs.append(g), ins.append((x, d)), outs.append(o)
    for rep in range(4):
        for i in range(2):
            j = (rep + i) % 3
            ins[i][0].copy_(xs[j]), ins[i][1].copy_(ds[j])
            graphs[i].replay()
        eager = step(xs[2], ds[2])      # the program's own work between the replays
        torch.cuda.synchronize()
        for i in range(2):
            j = (rep + i) % 3
            assert all(torch.equal(p, q) for p, q in zip(outs[i], want[j])), (rep, i)
        assert all(torch.equal(p, q) for p, q in zip(eager, want[2]))


@pytest.mark.gpu
def test_captured_training_step(dev):
    """A whole step through autograd (forward, backward, accumulated gradients) in one graph."""
    torch.manual_seed(0)
    ff = FeedForward(64, 128, 'relu').to(dev)
    x = torch.zeros(300, 64, device=dev)
    c = rand(2, 300, 64, dev=dev)

    def grads():
        return torch.autograd.grad(ff(x), list(ff.parameters()), c)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = grads()
    for i in range(3):
        x.copy_(rand(30 + i, 300, 64, dev=dev))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, grads())), i


@pytest.mark.gpu
def test_same_inputs_same_bits_and_inputs_untouched(dev):
    for dtype in DTYPES:
        x, w = rand(1, 3000, 200, dtype=dtype, dev=dev), rand(2, 130, 200, dtype=dtype, dev=dev)
        dy = rand(3, 3000, 130, dtype=dtype, dev=dev)
        z = rand(4, 3000, 130, dtype=dtype, dev=dev)
        keep = [t.clone() for t in (x, w, dy, z)]
        a = linear_backward(dy, x, w, z, 'gelu')
        _, _, mean, rstd = layer_norm_forward(x, keep_stats=True)
        n = layer_norm_backward(x, x, mean, rstd)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(a, linear_backward(dy, x, w, z, 'gelu')))
            assert all(torch.equal(p, q) for p, q in zip(n, layer_norm_backward(x, x, mean, rstd)))
        assert all(torch.equal(p, q) for p, q in zip(keep, (x, w, dy, z)))


@pytest.mark.gpu
def test_offsets_past_31_bits(dev):
    """Tensors of more than 2^31 elements, zero but for their last rows, those against 64 bits (zero rows
    add nothing to the sums over rows); rows far apart."""
    m, d, dtype = 8_400_100, 256, torch.bfloat16
    last = slice(m - 300, m)
    x = torch.zeros(m, d, dtype=dtype, device=dev)
    x[last] = rand(1, 300, d, dtype=dtype, dev=dev)
    w, b = rand(2, d, dtype=dtype, dev=dev), rand(3, d, dtype=dtype, dev=dev)
    y, _, mean, rstd = layer_norm_forward(x, w, b, keep_stats=True)
    small = layer_norm_forward(x[last], w, b, keep_stats=True)
    assert torch.equal(y[last], small[0]) and torch.equal(mean[last], small[2])
    assert torch.equal(y[0], b) and torch.equal(y[m // 2], b)      # rows of zeros
    dx, dw, db = layer_norm_backward(x, x, mean, rstd, w)      # zero gradients ahead of the last rows
    check_norm_backward(x[last], x[last], mean[last], rstd[last], w, None, dx[last], dw, db)
    assert not dx[:m - 300].any()
    del y, dx
    wl, bl = rand(4, d, d, dtype=dtype, dev=dev, scale=d ** -0.5), rand(5, d, dtype=dtype, dev=dev)
    y, _ = linear_forward(x, wl, bl)
    check_forward(x[last], wl, bl, None, None, y[last])
    assert torch.equal(y[0], bl) and torch.equal(y[m // 2], bl)
    del y
    dx, dw, db = linear_backward(x, x, wl)
    check_backward(x[last], x[last], wl, None, None, dx[last], dw, db)
    assert not dx[:m - 300].any()
    del dx
    wide = x.view(-1)[:64 << 25].view(64, 1 << 25)[:, -64:]      # rows 2^25 elements apart
    wide.copy_(rand(6, 64, 64, dtype=dtype, dev=dev))
    check_forward(wide, wl[:, :64], bl, 'gelu', None, linear(wide, wl[:, :64], bl, 'gelu'))
