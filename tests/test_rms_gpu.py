"""RMS norms on the GPU against float64, with and without the residual's addition,
their gradients, and the form written in 8 bits.

Bounds, in units of u = 2^-24 (half a step of fp32). A row's sum of squares is a chain
of at most 32 (a thread's) + 6 (a wave's exchanges) + 8 (waves) additions after one
rounding each of the squares folded into them: 46 u, which the square root halves; the
division, the addition of eps and the hardware's root add 4 u: rstd is off by 27 u at
most. y = s * rstd * gamma has two more roundings: 29 u, then half a step of its type.
dx = rstd (g - xh m) + ds: g has 1 u, xh 28 u, m (a chain of 46 again, over terms of 30 u)
76 u of mean |g xh|; with the products and sums behind them 110 u of
A = rstd (|g| + |xh| mean |g xh|) + |ds| bounds it. dgamma adds terms of 29 u in chains of
at most rows / 1024 (a workgroup's rows; 1 at least) + 16 (its row groups) + 16 + 20 (the
partial rows' strips): 120 u of sum |dy xh| up to 20000 rows.
"""
import numpy as np
import pytest

from oracle import distill_fp8 as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"bfloat16": 2.0 ** -8, "float32": U}
TINY = 2.0 ** -149
EPS = 1e-5

# rows of 16 lanes, of a wave (1, 2 and 4 vectors a lane), of 256 and of 512 threads; their ends and odd sizes
SHAPES = [(1, 1), (3, 7), (40, 64), (17, 128), (33, 129), (200, 512), (5, 513), (129, 1001), (64, 2048), (9, 2049),
          (30, 4096), (7, 5000), (12, 8192), (3, 8193), (5, 16384), (1500, 333)]


def _rng(*key):
    return np.random.default_rng(list(key))


def _matrix(rng, rows, cols):
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-6, 7, (rows, 1))
    return (x * np.where(rng.random((rows, cols)) < 0.01, 64.0, 1.0)).astype(np.float32)


def _device(x, dtype, dev, stride=None, shift=0):
    """x on the GPU with a row stride and a shift (elements) from an aligned base, NaN around it."""
    import torch

    rows, cols = x.shape
    buf = torch.full((rows * (stride or cols) + shift + 8,), float("nan"), dtype=dtype, device=dev)
    t = torch.as_strided(buf, (rows, cols), (stride or cols, 1), shift)
    t.copy_(torch.from_numpy(x).to(dev))
    return t


def _np(t):
    return t.detach().double().cpu().numpy()


def _norm64(s, eps=EPS):
    return 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)


def _close(got, want, bound, what):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3])


def _check(x, r, gamma, dy, ds, dtype):
    """Forward and gradients of both forms against float64."""
    import torch
    from nlearn_amd.kernels.fused import add_rms_norm, rms_norm

    dt = getattr(torch, dtype)
    leaf = lambda t: None if t is None else t.detach().requires_grad_(True)  # noqa: E731  (keeps strides)
    x, r, gamma = leaf(x), leaf(r), leaf(gamma)
    s = x.detach()
    if r is None:
        y = rms_norm(x, gamma, EPS)
        dx, dg = torch.autograd.grad(y, (x, gamma), dy)
    else:
        y, t = add_rms_norm(x, r, gamma, EPS)
        s = (x.detach().double() + r.detach().double()).to(dt)
        assert t.dtype is dt and torch.equal(t, s)
        dx, dr, dg = torch.autograd.grad((y, t), (x, r, gamma), (dy, ds))
        assert torch.equal(dx, dr)
    assert y.dtype is dt and dx.dtype is dt and dg.dtype is gamma.dtype and y.is_contiguous()
    s64, g64, d64 = _np(s), _np(gamma), _np(dy)
    rstd = _norm64(s64)
    xh = s64 * rstd
    want = xh * g64
    _close(_np(y), want, np.abs(want) * (HALF[dtype] + 30 * U) + TINY, "y")
    g = d64 * g64
    res = _np(ds) if r is not None else np.zeros_like(g)
    want = rstd * (g - xh * (g * xh).mean(1, keepdims=True)) + res
    size = rstd * (np.abs(g) + np.abs(xh) * np.abs(g * xh).mean(1, keepdims=True)) + np.abs(res)
    _close(_np(dx), want, np.abs(want) * HALF[dtype] + 110 * U * size + TINY, "dx")
    want, size = (d64 * xh).sum(0), np.abs(d64 * xh).sum(0)
    half = U if gamma.dtype is torch.float32 else 2.0 ** -8
    _close(_np(dg), want, np.abs(want) * half + 120 * U * size + TINY, "dgamma")


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm_and_gradients(dev, rows, cols, dtype, add):
    import torch

    rng, dt = _rng(rows, cols), getattr(torch, dtype)
    x = _device(_matrix(rng, rows, cols), dt, dev)
    r = _device(_matrix(rng, rows, cols), dt, dev) if add else None
    dy, ds = (_device(_matrix(rng, rows, cols) * 1e-3, dt, dev) for _ in range(2))
    gamma = torch.from_numpy(1 + 0.2 * rng.standard_normal(cols).astype(np.float32)).to(dev)
    _check(x, r, gamma, dy, ds, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("cols,stride,shift", [(259, 264, 0), (259, 261, 1), (128, 131, 3), (2048, 2056, 5), (5000, 5001, 7)])
def test_norm_strided_and_unaligned(dev, dtype, cols, stride, shift):
    import torch

    rng, dt = _rng(cols, stride, shift), getattr(torch, dtype)
    x, r, dy, ds = (_device(_matrix(rng, 37, cols), dt, dev, stride, shift) for _ in range(4))
    buf = torch.full((cols + 9,), float("nan"), device=dev)
    gamma = buf[shift:shift + cols].copy_(torch.from_numpy(1 + rng.random(cols).astype(np.float32)))
    _check(x, r, gamma, dy, ds, dtype)
    _check(x, None, gamma.bfloat16(), dy, None, dtype)  # a bf16 gamma gets a bf16 gradient


def test_norm_leading_dimensions_and_broadcast_cotangents(dev):
    import torch
    from nlearn_amd.kernels.fused import add_rms_norm, rms_norm

    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn((2, 3, 4, 96), generator=g, device=dev, dtype=torch.bfloat16)
    gamma = torch.ones(96, device=dev, requires_grad=True)
    flat = rms_norm(x.view(24, 96), gamma)
    assert torch.equal(rms_norm(x, gamma).view(24, 96), flat)
    # heads on the second axis: rows of a permuted view have no single stride
    assert torch.equal(rms_norm(x.permute(0, 2, 1, 3), gamma), rms_norm(x, gamma).permute(0, 2, 1, 3))
    assert rms_norm(x[0, 0, 0], gamma).shape == (96,)
    # y.sum() hands back a cotangent of stride 0
    a = x.clone().requires_grad_(True)
    rms_norm(a, gamma).sum().backward()
    b = x.clone().requires_grad_(True)
    want = gamma.grad.clone()
    gamma.grad = None
    rms_norm(b, gamma).backward(torch.ones_like(b))
    assert torch.equal(a.grad, b.grad) and torch.equal(gamma.grad, want)
    # one of the two outputs alone, and inputs that are the same tensor
    c = x.clone().requires_grad_(True)
    y, s = add_rms_norm(c, c, gamma)
    (ds,) = torch.autograd.grad(s, c, torch.ones_like(s), retain_graph=True)
    assert torch.equal(ds, torch.full_like(ds, 2))
    (dy,) = torch.autograd.grad(y, c, torch.ones_like(y))
    e = (x + x).requires_grad_(True)
    (want,) = torch.autograd.grad(rms_norm(e, gamma), e, torch.ones_like(y))
    assert torch.equal(dy, want + want)


def test_norm_without_gradients_of_one_input(dev):
    import torch
    from nlearn_amd.kernels.fused import rms_norm

    g = torch.Generator(device=dev).manual_seed(6)
    x = torch.randn((50, 300), generator=g, device=dev)
    gamma = torch.randn((300,), generator=g, device=dev)
    dy = torch.randn((50, 300), generator=g, device=dev)
    both = [x.clone().requires_grad_(True), gamma.clone().requires_grad_(True)]
    dx, dg = torch.autograd.grad(rms_norm(*both), both, dy)
    assert torch.equal(torch.autograd.grad(rms_norm(both[0], gamma), both[0], dy)[0], dx)
    assert torch.equal(torch.autograd.grad(rms_norm(x, both[1]), both[1], dy)[0], dg)
    assert not rms_norm(x, gamma).requires_grad
    # a gradient buffer takes dgamma, twice the same
    both[1].main_grad = torch.full((300,), 7.0, device=dev)
    for _ in range(2):
        rms_norm(*both).backward(dy)
        assert torch.equal(both[1].main_grad, dg) and both[1].grad is None
    both[1].main_grad = torch.zeros((301,), device=dev)
    with pytest.raises(ValueError, match="main_grad"):
        rms_norm(*both).backward(dy)


def test_norm_gradient_against_differences(dev):
    """Central differences in float64 of the definition, and of the fp32 kernel itself along one direction."""
    import torch
    from nlearn_amd.kernels.fused import rms_norm

    g = torch.Generator(device=dev).manual_seed(8)
    x = torch.randn((6, 200), generator=g, device=dev)
    gamma = 1 + 0.1 * torch.randn((200,), generator=g, device=dev)
    dy = torch.randn((6, 200), generator=g, device=dev)
    v = torch.randn((6, 200), generator=g, device=dev)
    a = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(rms_norm(a, gamma), a, dy)
    h = 2.0 ** -6
    up, down = (rms_norm(x + k * v, gamma).double() for k in (h, -h))
    slope = float(((up - down) * dy.double()).sum() / (2 * h))
    # the kernel's roundings: 31 u of |y| a value over 2h; the third derivative's term: y is homogeneous of degree 0
    # in x, so h^2 |v|^3 / rms^3 scales it: below 10 h^2 of sum |dy| |v|
    y = rms_norm(x, gamma).double().abs()
    bound = float((y * dy.double().abs()).sum()) * 31 * U / h + 10 * h * h * float((dy.double() * v.double()).abs().sum())
    assert abs(slope - float((dx.double() * v.double()).sum())) <= bound


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("cols", [100, 1000, 5000])
def test_norm_rows_of_zeros_of_large_values_and_not_finite(dev, cols, dtype):
    import torch
    from nlearn_amd.kernels.fused import rms_norm

    rng, dt = _rng(cols), getattr(torch, dtype)
    x = _matrix(rng, 12, cols)
    x[0] = 0
    x[1] *= 1e-30
    x[2] = np.sign(x[2]) * 2.0 ** 127     # squares pass fp32
    x[3] *= 2.0 ** 70
    x[4, cols // 2] = 3e38
    x[5] = 1.5 * 2.0 ** 63                # the squares' sum passes fp32
    t = _device(x, dt, dev)
    gamma = torch.from_numpy(1 + rng.random(cols).astype(np.float32)).to(dev)
    y = _np(rms_norm(t, gamma, EPS))
    s = _np(t)
    want = s * _norm64(s) * _np(gamma)
    # an rstd below 2^-126 keeps 23 bits less its distance from there: 2^-23 of it at 2^-127, where 2^127 lies;
    # a value below 2^-126 is off by half a step of the subnormals of its type
    step = 2.0 ** -133 if dtype == "bfloat16" else TINY
    _close(y, want, np.abs(want) * (HALF[dtype] + 34 * U) + step, "y")
    assert (y[0] == 0).all()
    t[6, 3] = float("inf")
    t[7, 3] = float("nan")
    t[8, 0], t[8, 1] = float("inf"), float("-inf")
    z = _np(rms_norm(t, gamma, EPS))
    assert (np.delete(z[6], 3) == 0).all() and np.isnan(z[6, 3])
    assert np.isnan(z[7]).all()
    assert (z[8, 2:] == 0).all() and np.isnan(z[8, :2]).all()
    rest = [i for i in range(12) if i not in (6, 7, 8)]
    np.testing.assert_array_equal(z[rest], y[rest])


def test_norm_is_the_same_every_time_and_over_many_rows(dev):
    """More rows than a launch's workgroups take at once, and a fixed order of dgamma's sum."""
    import torch
    from nlearn_amd.kernels.fused import rms_norm

    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn((20000, 72), generator=g, device=dev, dtype=torch.bfloat16)
    dy = torch.randn((20000, 72), generator=g, device=dev, dtype=torch.bfloat16)
    gamma = torch.ones(72, device=dev)
    _check(x, None, gamma, dy, None, "bfloat16")
    a, b = x.requires_grad_(True), gamma.requires_grad_(True)
    first = torch.autograd.grad(rms_norm(a, b), (a, b), dy)
    for _ in range(3):
        again = torch.autograd.grad(rms_norm(a, b), (a, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_norm_of_no_rows(dev):
    import torch
    from nlearn_amd.kernels.fp8 import add_rms_norm_fp8
    from nlearn_amd.kernels.fused import add_rms_norm, rms_norm

    x = torch.empty((0, 96), device=dev, requires_grad=True)
    gamma = torch.ones(96, device=dev, requires_grad=True)
    y = rms_norm(x, gamma)
    assert y.shape == (0, 96)
    y.sum().backward()
    assert x.grad.shape == (0, 96) and (gamma.grad == 0).all()
    assert add_rms_norm(x, x, gamma)[1].shape == (0, 96)
    q, s = add_rms_norm_fp8(x, x, gamma)
    assert q.shape == (0, 96) and q.q.shape == (0, 128) and s.shape == (0, 96)


def _check_8_bits(b, y64, delta):
    """Each byte and scale is that of a value within delta of the definition's."""
    import torch

    got, scale = (t.contiguous().view(torch.uint8).cpu().numpy() for t in (b.q, b.scale))
    assert b.shape == y64.shape and b.group == 1
    lo, hi = orc.quantize(y64 * (1 - delta), 1)[1], orc.quantize(y64 * (1 + delta), 1)[1]
    assert ((scale == lo) | (scale == hi)).all()
    rows, cols = y64.shape
    p = np.zeros(got.shape)
    p[:, :cols] = y64
    u = p / np.repeat(2.0 ** (scale.astype(float) - 127), 128, 1)
    near = [orc.e4m3_bytes(np.clip(u * (1 + k * delta), -448, 448)) for k in (-1, 1)]
    got = np.where(got == 0xff, 0x7f, got)
    bad = (got != near[0]) & (got != near[1])
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), u[bad][:3], got[bad][:3])
    assert (got[:, cols:] == 0).all()


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_norm_in_8_bits(dev, rows, cols, dtype, add):
    import torch
    from nlearn_amd.kernels.fp8 import add_rms_norm_fp8, rms_norm_fp8

    rng, dt = _rng(rows, cols, 8), getattr(torch, dtype)
    x, r = (_device(_matrix(rng, rows, cols), dt, dev, cols + 3, 1) for _ in range(2))
    gamma = torch.from_numpy(1 + 0.2 * rng.standard_normal(cols).astype(np.float32)).to(dev)
    s = x
    if add:
        b, s = add_rms_norm_fp8(x, r, gamma, EPS)
        assert torch.equal(s, (x.double() + r.double()).to(dt))
    else:
        b = rms_norm_fp8(x, gamma, EPS)
    s64 = _np(s)
    _check_8_bits(b, s64 * _norm64(s64) * _np(gamma), 30 * U)


def test_norm_in_8_bits_of_rows_that_are_not_finite(dev):
    import torch
    from nlearn_amd.kernels.fp8 import rms_norm_fp8

    x = torch.ones((4, 300), device=dev)
    x[1, 5] = float("inf")
    x[2, 290] = float("nan")
    x[3] = 0
    v = rms_norm_fp8(x, torch.ones(300, device=dev)).dequantize().cpu().numpy()
    np.testing.assert_allclose(v[0], 1.0, rtol=2.0 ** -4)
    assert np.isnan(v[1, 5]) and (np.delete(v[1], 5) == 0).all()
    assert np.isnan(v[2]).all() and (v[3] == 0).all()


@pytest.mark.parametrize("rows,cols", [(0, 40), (1, 7), (300, 129), (90, 5000)])
def test_gradient_added_to_what_is_there(dev, rows, cols):
    """The library's accumulate: dgamma + what it held, by one addition."""
    import torch
    from nlearn_amd import _lib

    g = torch.Generator(device=dev).manual_seed(rows + cols)
    x, dy = (torch.randn((rows, cols), generator=g, device=dev) for _ in range(2))
    gamma, held = (torch.randn((cols,), generator=g, device=dev) for _ in range(2))
    rstd = torch.rand((rows,), generator=g, device=dev) + 0.5
    wsb = _lib.load().nl_rms_norm_bwd_ws_bytes(rows, cols)
    ws = torch.empty(max(wsb, 16), dtype=torch.uint8, device=dev)
    got = []
    for acc in (0, 1):
        dx, dg = torch.empty_like(x), held.clone()
        _lib.call_on(gamma, "nl_rms_norm_bwd", rows, cols, 0, dy.data_ptr(), cols, x.data_ptr(), cols, rstd.data_ptr(),
                     gamma.data_ptr(), None, 0, dx.data_ptr(), cols, dg.data_ptr(), acc, ws.data_ptr(), wsb)
        got.append((dx, dg))
    assert torch.equal(got[0][0], got[1][0])
    assert torch.equal(got[1][1], held + got[0][1])
    if rows == 0:
        assert (got[0][1] == 0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("cols", [9, 101, 333, 1001, 4099])
def test_rows_keep_to_themselves(dev, cols, dtype):
    """Rows that end inside a vector, beside rows of NaN and infinities: the bits that finite neighbours leave."""
    import torch
    from nlearn_amd.kernels.fp8 import add_rms_norm_fp8, linear_fp8, quantize_fp8, quantize_fp8_both
    from nlearn_amd.kernels.fused import add_rms_norm

    dt = getattr(torch, dtype)
    rng = _rng(cols, 77)
    clean = [torch.from_numpy(_matrix(rng, 140, cols)).to(dev).to(dt) for _ in range(4)]
    bad = [t.clone() for t in clean]
    for t in bad:
        t[1::2] = float("nan")
        t[3::4] = float("inf")
    gamma = torch.from_numpy(1 + 0.1 * rng.standard_normal(cols).astype(np.float32)).to(dev)
    W = torch.from_numpy(rng.standard_normal((16, cols)).astype(np.float32)).to(dev)
    bits = lambda b: (b.q.view(torch.uint8), b.scale.contiguous().view(torch.uint8))  # noqa: E731

    def everything(x, r, dy, ds):
        x, r = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
        y, s = add_rms_norm(x, r, gamma, EPS)
        (dx,) = torch.autograd.grad((y, s), x, (dy, ds))
        b, t = add_rms_norm_fp8(x.detach(), r.detach(), gamma, EPS)
        h = torch.ones((140, 16), device=dev, dtype=dt).requires_grad_(True)
        outs = [y, s, dx, t, *bits(b), *bits(quantize_fp8(dy)), *bits(quantize_fp8_both(dy)[0])]
        for name in ("gelu", "silu", "relu"):
            z = linear_fp8(h, W, activation=name, residual=r.detach())
            outs += [z, torch.autograd.grad(z, h, dy)[0]]
        return outs

    for a, b in zip(everything(*clean), everything(*bad)):
        assert torch.equal(a[0::2], b[0::2])
