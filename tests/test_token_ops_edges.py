"""Token operators where a bound on the average case sees nothing: digits of small values, sums whose
parts can be told apart, inputs that are not plain memory, calls that cannot be served.

Tolerances count half steps of the storage type (u), E = 2^-24 for an fp32 operation, and what the
kernels' own approximations state; each is derived where it stands.
"""
import math
import os
import subprocess
import sys

import pytest
import torch

from sparsefusion_amd import _lib
from sparsefusion_amd.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
from sparsefusion_amd.linear import Linear, linear, linear_backward, linear_forward

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ['f32', 'f16', 'bf16']
E = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def rand(seed, *shape, dtype=torch.float32, dev='cpu', scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(dev)


# ---------------------------------------------------------------------------------- digits of GELU

def gelu_inputs(dtype, dev):
    """Every 16-bit number of [-20, 20] that is not subnormal; for fp32 a grid of 2^-11, and powers of two
    around zero."""
    if dtype == torch.float32:
        z = torch.arange(-20 * 2048, 20 * 2048 + 1, device=dev).float() / 2048
        small = 2.0 ** torch.arange(-120, 0, device=dev).float()
        z = torch.cat([z, small, -small])
    else:
        z = torch.arange(-32768, 32768, dtype=torch.int32, device=dev).to(torch.int16).view(dtype)
    z = z[(z.abs() <= 20) & ((z.abs() >= torch.finfo(dtype).smallest_normal) | (z == 0))]
    return torch.cat([z, z.new_zeros(-z.numel() % 64)]).view(-1, 64)


def gelu_bounds(z, dtype):
    """-> gelu, its slope and what each may be off by before it is rounded to dtype.  Phi(-a), a = |z|, is
    off by `fit` of itself; exp(-a^2 / 2) by 2.5 a^2 E (the constant and the two products in its exponent)
    and 2 E; the reciprocal 2 E, seven steps of a Horner scheme whose terms add up to twice its value 28 E,
    products 4 E.  Results below the smallest normal fp32 number may be flushed."""
    zd = z.double()
    a = zd.abs()
    tail = torch.special.erfc(a / math.sqrt(2)) / 2      # (ndtr loses its digits for arguments far below 0)
    density = torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    if dtype == torch.float32:
        fit = 5.2e-8 * (1 + (a - 1).clamp(min=0) ** 3)
    else:
        fit = torch.where(a <= 4, 6e-5, 4e-4)
    rel = fit + (2.5 * a * a + 36) * E
    flush = 20 * torch.finfo(torch.float32).smallest_normal
    y = torch.where(zd < 0, -a * tail, zd - a * tail)
    s = tail - a * density
    slope = torch.where(zd < 0, s, 1 - s)
    return (y, a * tail * rel + E * y.abs() + flush,
            slope, tail * rel + a * density * (2.5 * a * a + 8) * E + 2 * E * slope.abs() + flush)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('rows,width', [(8, 64), (None, 64), (20000, 512)])
def test_gelu_keeps_the_digits_of_its_type(dev, dtype, rows, width):
    """Through an identity weight (its products and sums are exact): few rows, tiny and large layers."""
    z = gelu_inputs(dtype, dev)
    if width > 64:
        z = z.reshape(-1)[torch.arange(rows * width, device=dev) % z.numel()].view(rows, width)
    eye = torch.eye(width, dtype=dtype, device=dev)
    dy = torch.where(torch.arange(z.numel(), device=dev).view_as(z) % 3 == 1, -1.5, 1.0).to(dtype)
    for part in ((z,) if width > 64 or rows is None else z.split(rows)):
        y, ey, slope, es = gelu_bounds(part, dtype)
        got, pre = linear_forward(part, eye, None, 'gelu', None, True)
        assert torch.equal(pre, part)
        over = (got.double() - y).abs() - (ey + u(dtype) * (y.abs() + ey) + tiny(dtype))
        worst = over.argmax()
        assert over.max() <= 0, (part.flatten()[worst].item(), got.flatten()[worst].item(), y.flatten()[worst].item())
        if rows == 8 and width == 64:
            continue
        g = dy.double()
        dx, _, _ = linear_backward(dy, part, eye, part, 'gelu', (True, False, False))
        want, err = g * slope, g.abs() * (es + E * slope.abs())
        over = (dx.double() - want).abs() - (err + u(dtype) * (want.abs() + err) + tiny(dtype))
        worst = over.argmax()
        assert over.max() <= 0, (part.flatten()[worst].item(), dx.flatten()[worst].item(), want.flatten()[worst].item())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_gelu_of_infinities_and_nan(dev, dtype):
    inf = float('inf')
    big = torch.finfo(dtype).max
    z = torch.tensor([inf, -inf, float('nan'), big, -big, 0.0], dtype=dtype, device=dev)[:, None]
    for m in (6, 600):
        x = z.repeat(m // 6, 1)
        one = torch.ones(1, 1, dtype=dtype, device=dev)
        y = linear(x, one, activation='gelu').view(-1, 6)
        assert (y[:, 0] == inf).all() and not y[:, 1].any() and y[:, 2].isnan().all()
        assert (y[:, 3] == big).all() and not y[:, 4].any() and not y[:, 5].any()
        dy = torch.ones_like(x)
        dx = linear_backward(dy, x, one, x, 'gelu', (True, False, False))[0].view(-1, 6)
        want = torch.tensor([1, 0, float('nan'), 1, 0, 0.5], dtype=dtype, device=dev)
        assert torch.equal(dx.isnan(), want.isnan().expand_as(dx))
        assert torch.equal(dx.nan_to_num(), want.nan_to_num().expand_as(dx))


# ---------------------------------------------------------------------------------- digits of layer norm

@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('d', [1, 7, 40, 128, 320, 333, 700, 1000, 1500, 3000, 5000, 16000, 20001])
def test_a_common_offset_costs_no_digits(dev, dtype, d):
    """Rows far from zero, with little spread or none.  A sum's error is ge = (d / 64 + 48) E of the magnitudes;
    the first mean's, dm, is that of the offset; what is left of a value, at most |s - m| + dm, is centred by
    the mean of all that is left, off by ge of those magnitudes, with two roundings of E.  The variance carries
    twice that error times the spread, its square, and ge; rstd half of its relative error and 4 E."""
    rows = [torch.full((d,), c) for c in (0.0, 0.1, 100.0, 1000.7, -12345.6, 3.0e4)]
    rows += [c + spread * rand(i, d) for i, (c, spread) in enumerate(
        [(1000.0, 1e-3), (250.0, 1.0), (-3000.0, 0.01), (2.0e4, 30.0), (1.0, 1e-3), (0.0, 1.0)])]
    x = torch.stack(rows).to(dtype).to(dev)
    w, b = rand(20, d, dtype=dtype, dev=dev, shift=1.0), rand(21, d, dtype=dtype, dev=dev)
    ge = (d / 64 + 48) * E
    s = x.double()
    m = s.mean(1, keepdim=True)
    dm = ge * s.abs().mean(1, keepdim=True)
    left = (s - m).abs() + dm
    dc = ge * left.mean(1, keepdim=True) + 2 * E * left
    for eps in (1e-5, 1e-3):
        y, _, mean, rstd = layer_norm_forward(x, w, b, eps, keep_stats=True)
        var = (s - m).square().mean(1, keepdim=True)
        r = 1 / torch.sqrt(var + eps)
        # squares of what is left: ge and its own roundings of them, the offset's share cancels to as much
        dv = 2 * var.sqrt() * dc.square().mean(1, keepdim=True).sqrt() + dc.square().mean(1, keepdim=True) \
            + (ge + 4 * E) * left.square().mean(1, keepdim=True) + 2 * dm * ge * left.mean(1, keepdim=True)
        dr = r * (0.5 * dv * r * r * (1 + dv * r * r) + 4 * E)
        xh = (s - m) * r
        dxh = dc * (r + dr) + (s - m).abs() * dr + 2 * E * xh.abs()
        want = xh * w.double() + b.double()
        err = dxh * w.double().abs() + 2 * E * (xh * w.double()).abs() + E * want.abs()
        bound = err + u(dtype) * (want.abs() + err) + tiny(dtype)
        over = (y.double() - want).abs() - bound
        assert over.max() <= 0, (divmod(over.argmax().item(), d), (y.double() - want).abs().max(1).values)
        assert ((mean.double() - m[:, 0]).abs() <= (dc.mean(1) + 2 * E * m[:, 0].abs() + 1e-45)).all()
        assert ((rstd.double() - r[:, 0]).abs() <= (dr + 2 * E * r)[:, 0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 320, 3000, 20001])
def test_a_constant_row_normalises_to_its_bias(dev, d):
    """To a part in 1e5 (fp32, eps 1e-5): what is left of the offset is within ge^2 rstd of it."""
    ge = (d / 64 + 48) * E
    b = rand(1, d, dev=dev)
    for c in (1000.7, -77.3, 0.1):
        y = layer_norm(torch.full((3, d), c, device=dev), None, b)
        assert (y - b).abs().max() <= 2 * ge * ge * abs(c) * 317 + 1e-6


# ---------------------------------------------------------------------------------- sums, exactly

def whole(seed, *shape, dtype=torch.float32, dev='cpu'):
    """-2, -1, 1 or 2: products and their sums are exact in fp32, in any order, as long as they stay below 2^24,
    and no term is 0, so that none can be left out without a trace."""
    g = torch.Generator().manual_seed(seed)
    return torch.tensor([-2.0, -1.0, 1.0, 2.0])[torch.randint(0, 4, shape, generator=g)].to(dtype).to(dev)


def assert_sum(got, want, what):
    """want (float64) is exact: got is it, rounded once."""
    want = want.to(got.dtype)
    wrong = (got != want).nonzero()
    assert not len(wrong), (what, len(wrong), wrong[0].tolist(), got[tuple(wrong[0])].item(), want[tuple(wrong[0])].item())


def linear_sums(dy, x, w, keep=slice(None)):
    """dx, dw and db in 64 bits; `keep`: of these rows alone (dx: all)."""
    dy, x, w = dy.double(), x.double(), w.double()
    return dy @ w, dy[keep].T @ x[keep], dy[keep].sum(0)


def norm_sums(dy, x, mean, rstd, keep=slice(None)):
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    return (dy.double() * xh)[keep].sum(0), dy.double()[keep].sum(0)


def test_exact_sums_show_what_is_left_out():
    """The comparisons below turn down sums without the last row, a run of rows or a share of them."""
    assert set(whole(1, 4000).tolist()) == {-2.0, -1.0, 1.0, 2.0}
    m = 70000
    dy, x, y, w = whole(1, m, 5), whole(2, m, 6), whole(6, m, 5), whole(3, 5, 6)
    mean, rstd = whole(4, m), 2.0 ** whole(5, m)
    rows = torch.arange(m)
    for left in (rows == m - 1, rows == 0, rows >= m - 128, rows % 97 == 5, (rows >= 640) & (rows < 704)):
        for name, full, part in (*zip(('dw', 'db'), linear_sums(dy, x, w)[1:], linear_sums(dy, x, w, ~left)[1:]),
                                 *zip(('dw', 'db'), norm_sums(dy, y, mean, rstd), norm_sums(dy, y, mean, rstd, ~left))):
            assert_sum(full.float(), full, name)
            with pytest.raises(AssertionError):
                assert_sum(part.float(), full, name)


SUM_SIZES = [(1, 64, 64), (7, 5, 3), (65, 127, 63), (200, 128, 256), (1000, 512, 512), (4000, 512, 1024),
             (2000, 4096, 96), (16300, 800, 1016), (20001, 30, 514), (40000, 72, 48), (9001, 1027, 1001),
             (33, 300, 1111), (32400, 256, 256), (70001, 64, 40), (110000, 33, 37), (259200, 64, 64), (6, 8192, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,k,n', SUM_SIZES)
def test_linear_sums_are_complete(dev, dtype, m, k, n):
    x, w, b = whole(1, m, k, dtype=dtype, dev=dev), whole(2, n, k, dtype=dtype, dev=dev), whole(3, n, dtype=dtype, dev=dev)
    dy, z = whole(4, m, n, dtype=dtype, dev=dev), whole(5, m, n, dtype=dtype, dev=dev)
    assert_sum(linear(x, w, b), x.double() @ w.double().T + b.double(), 'y')
    for act, g in ((None, dy), ('relu', dy * (z > 0))):
        for needs in ((True, True, True), (False, True, False), (False, False, True)):
            for name, got, want in zip(('dx', 'dw', 'db'), linear_backward(dy, x, w, z, act, needs), linear_sums(g, x, w)):
                if got is not None:
                    assert_sum(got, want, (name, act, needs))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('m,d', [(1, 64), (3, 7), (200, 128), (5003, 333), (5000, 96), (1537, 2048), (515, 4097), (64, 16384),
                                 (100, 20001), (70000, 40), (110000, 333), (70000, 512), (259200, 64)])
def test_layer_norm_sums_are_complete(dev, dtype, m, d):
    """Statistics handed over that keep (x - mean) * rstd exact."""
    x, dy = whole(1, m, d, dtype=dtype, dev=dev), whole(2, m, d, dtype=dtype, dev=dev)
    mean, rstd = whole(3, m, dev=dev), 2.0 ** whole(4, m, dev=dev)
    for pd in {dtype, torch.float32}:
        w = whole(5, d, dtype=pd, dev=dev)
        _, dw, db = layer_norm_backward(dy, x, mean, rstd, w, dy)
        assert dw.dtype == db.dtype == pd
        for name, got, want in zip(('dw', 'db'), (dw, db), norm_sums(dy, x, mean, rstd)):
            assert_sum(got, want, name)


# ---------------------------------------------------------------------------------- inputs that are no plain memory

def negated(t):
    """t as a lazily negated view: the imaginary part of a conjugate, 2 elements apart."""
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg() and torch.equal(view, t)
    return view


def test_lazily_negated_views_are_resolved():
    """Contiguous, or rows of one element that rows() hands on as they are: only these need a look."""
    for shape in ((1, 1), (5, 1), (1, 3), (3, 4), (1,), (2, 2, 1), (2, 2, 3)):
        t = negated(rand(1, *shape))
        assert t.is_contiguous() == (t.numel() == 1)
        assert _lib.rows(t)[0].is_neg() == (shape[-1] == 1)
        out, none, same = _lib.resolved(t, None, rand(2, 3))
        assert not out.is_neg() and torch.equal(out, t) and none is None and torch.equal(same, rand(2, 3))


@pytest.mark.gpu
def test_lazily_negated_tensors(dev):
    """Sizes at which such a view keeps the strides that the kernels read in place (fp32: complex numbers)."""
    for m, k, n in ((5, 1, 7), (1, 1, 1), (300, 1, 64), (6, 8, 1)):
        x, w, b, r = (rand(i, *s, dev=dev) for i, s in enumerate(((m, k), (n, k), (n,), (m, n))))
        dy, z = rand(5, m, n, dev=dev), rand(6, m, n, dev=dev)
        y = linear(x, w, b, 'gelu', r)
        assert torch.equal(linear(*map(negated, (x, w, b)), 'gelu', negated(r)), y)
        want = linear_backward(dy, x, w, z, 'gelu')
        got = linear_backward(*map(negated, (dy, x, w, z)), 'gelu')
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        if n == 1:      # a gradient that autograd hands over in this form
            xl = x.clone().requires_grad_()
            out = linear(xl, w, b)
            torch.complex(torch.zeros_like(out), out).conj().imag.backward(dy)
            assert torch.equal(xl.grad, linear_backward(-dy, x, w)[0])
    for m, d in ((4, 1), (1, 1), (3, 8)):
        x, r, dy, ds = (rand(i, m, d, dev=dev, shift=0.5) for i in range(4))
        w, b = rand(7, d, dev=dev), rand(8, d, dev=dev)
        y, s, mean, rstd = layer_norm_forward(x, w, b, 1e-5, r, True, True)
        got = layer_norm_forward(*map(negated, (x, w, b)), 1e-5, negated(r), True, True)
        assert all(torch.equal(p, q) for p, q in zip(got, (y, s, mean, rstd)))
        want = layer_norm_backward(dy, s, mean, rstd, w, ds)
        got = layer_norm_backward(*map(negated, (dy, s, mean, rstd, w, ds)))
        assert all(torch.equal(p, q) for p, q in zip(got, want))


# ---------------------------------------------------------------------------------- calls that cannot be served

def test_forward_mode_tangents_are_refused():
    """Without a HIP device: the refusal comes before the device is looked at, plain tensors get that far."""
    from torch.autograd import forward_ad
    x, w, b = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8)
    stats = torch.zeros(4)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: linear(dual(x), w, b), lambda: linear(x, dual(w), b), lambda: linear(x, w, dual(b)),
                     lambda: linear(x, w, b, residual=dual(x)), lambda: linear_forward(dual(x), w),
                     lambda: linear_backward(dual(x), x, w), lambda: linear_backward(x, dual(x), w),
                     lambda: linear_backward(x, x, w, dual(x), 'relu'),
                     lambda: layer_norm(dual(x)), lambda: layer_norm(x, dual(b)), lambda: layer_norm(x, b, dual(b)),
                     lambda: layer_norm(x, residual=dual(x)), lambda: layer_norm_forward(dual(x)),
                     lambda: layer_norm_backward(dual(x), x, stats, stats),
                     lambda: layer_norm_backward(x, x, stats, stats, None, dual(x))):
            with torch.no_grad(), pytest.raises(RuntimeError, match='no forward-mode derivative'):
                call()
        for call in (lambda: linear(x, w, b), lambda: layer_norm(x, b)):
            with pytest.raises(RuntimeError, match='HIP device'):
                call()
        # parameters that require grad: the autograd function has no forward-mode rule either
        with pytest.raises(RuntimeError):
            Linear(8, 8)(dual(x))


def test_traces_are_refused():
    x, w, b = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8)
    for call in (lambda t: linear(t, w, b), lambda t: linear_backward(t, x, w)[0], lambda t: layer_norm(t, b),
                 lambda t: layer_norm_backward(t, x, b[:4], b[:4])[0], Linear(8, 8)):
        with pytest.raises(RuntimeError, match='cannot be traced'):
            torch.jit.trace(call, x)


def test_recorded_operators_are_refused():
    """make_fx in each of its modes, and fake tensors; a mode that only watches is none of them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    x, w, b, stats = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8), torch.zeros(4)
    calls = (lambda t: linear(t, w, b), lambda t: linear_backward(t, t, w)[0], lambda t: layer_norm(t, b),
             lambda t: layer_norm_backward(t, t, stats, stats)[0], Linear(8, 8))
    for call in calls:
        for mode in ('real', 'fake', 'symbolic'):
            with pytest.raises(RuntimeError, match='cannot be traced'):
                make_fx(call, tracing_mode=mode)(x)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        for call in calls[:4]:
            with pytest.raises(RuntimeError, match='cannot be traced'):
                call(mode.from_tensor(x))

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    for call in calls:
        with Watch(), pytest.raises(RuntimeError, match='HIP device'):
            call(x)


# ---------------------------------------------------------------------------------- the package around them

def test_import_needs_no_device_functions():
    """A torch built without devices lacks the bindings that the stream and device lookups use."""
    code = """
import torch
for name in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import sparsefusion_amd
from sparsefusion_amd import _lib, layer_norm, linear, pipeline, sparse_encoder, voxelize
try:
    linear.linear(torch.zeros(2, 3), torch.zeros(4, 3))
except RuntimeError as e:
    assert 'HIP device' in str(e), e
else:
    raise SystemExit('served')
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


@pytest.mark.gpu
def test_stream_of_any_form_of_device(dev):
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for device in (dev, torch.device('cuda', 0), torch.device('cuda'), 0, 'cuda:0', 'cuda', None):
            assert _lib.stream(device) == side.cuda_stream
    assert _lib.stream(0) == torch.cuda.current_stream().cuda_stream


def test_scratch_depends_on_sizes_and_places_alone():
    """What the Python layer looks up by sizes and by the operands' place in 16 bytes is what the library asks
    for at the addresses themselves."""
    L = _lib.lib()
    for code in (0, 1, 2):
        for m, k, n in ((1, 64, 64), (80, 8192, 64), (80, 65, 64), (6400, 32, 33), (3001, 451, 333), (40000, 256, 256)):
            for place in (0, 2, 4, 8, 14):
                at = [0x7f0000000000 + 4096 * i + place for i in range(3)]
                low = [a & 15 for a in at]
                for res in (0, 1):
                    assert (L.sf_linear_workspace(at[0], k, at[1], m, k, n, code, res) ==
                            L.sf_linear_workspace(low[0], k, low[1], m, k, n, code, res))
                    assert (L.sf_linear_backward_workspace(at[0], at[1], k, at[2], m, k, n, code, res) ==
                            L.sf_linear_backward_workspace(low[0], low[1], k, low[2], m, k, n, code, res))


@pytest.mark.gpu
def test_calls_are_made_once(dev, monkeypatch):
    """No call is refused on the way to its result, and a message that a caller has yet to read stays."""
    L = _lib.lib()
    assert L.sf_linear(64, 8, 64, None, None, 64, None, 4, 8, 4, 7, 0, None, 0, None) == -1
    told = L.sf_last_error()
    calls = []

    class Counted:
        def __getattr__(self, name):
            calls.append(name)
            return getattr(L, name)

    monkeypatch.setattr(_lib, 'lib', Counted)
    for m, k, n in ((4, 8, 6), (80, 8192, 64), (81, 65, 33), (6400, 32, 32), (2000, 1024, 1024)):
        for dtype in DTYPES:
            x, w = rand(1, m, k, dtype=dtype, dev=dev), rand(2, n, k, dtype=dtype, dev=dev)
            dy = rand(3, m, n, dtype=dtype, dev=dev)
            for _ in range(2):
                calls.clear()
                linear(x, w, activation='relu')
                linear_backward(dy, x, w, dy, 'gelu')
                assert calls.count('sf_linear') == 1 and calls.count('sf_linear_backward') == 1
            assert len(calls) == 2      # known sizes ask for nothing more
    assert L.sf_last_error() == told
