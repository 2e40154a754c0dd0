"""8-bit products with bias, activation and residual in their epilogue, on the GPU against
float64, and the layer's gradients.

Bounds, u = 2^-24. The sum's are those of the product alone (test_fp8_gpu.py): K u sum |a b| for fp32
results, 7 * 2^-13 sum |a b| more where the 8-bit instruction sums. The bias adds a rounding. An
activation passes an error of its argument on by at most its largest slope (1.13 for gelu, 1.1 for
silu) and adds its own: a logistic 1 / (1 + 2^t) of hardware exp2 and reciprocal (each within a unit of
its last place, 2 u) at an argument t with 4 roundings (u |t| ln 2 each), then a product:
(3 |t| + 8) u of the value. The residual adds a rounding, then comes half a step of the result's type.
"""
import numpy as np
import pytest

from oracle import distill_fp8 as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"bfloat16": 2.0 ** -8, "float32": U}
C = np.sqrt(8 / np.pi)


def _rng(*key):
    return np.random.default_rng(list(key))


def _act(z, name):
    """(act(z), act'(z), t) in float64, t the logistic's argument in powers of two."""
    if name == "relu":
        return np.where(z < 0, 0, z), (z > 0) * 1.0, 0 * z
    if name is None:
        return z, np.ones_like(z), 0 * z
    w, dw = (z, 1.0) if name == "silu" else (C * (z + 0.044715 * z ** 3), C * (1 + 3 * 0.044715 * z * z))
    with np.errstate(over="ignore"):
        s = np.where(w > 0, 1 / (1 + np.exp(-np.abs(w))), np.exp(-np.abs(w)) / (1 + np.exp(-np.abs(w))))
    return z * s, s * (1 + z * (1 - s) * dw), np.minimum(np.abs(w) / np.log(2), 150)


def _np(t):
    return t.detach().double().cpu().numpy()


def _slope_error(z, name):
    """The bound of the error of act'(z) = s (1 + z q (1 - s)), q the slope of the logistic's argument: s is off by
    r = (3 |t| (1 - s) + 8) u of itself (its power of two by 3 |t| u, less the nearer s is to 1), 1 - s by s r + 2 u,
    and six roundings follow."""
    if name not in ("gelu", "silu"):
        return 0 * z
    q = C * (1 + 3 * 0.044715 * z * z) if name == "gelu" else 1.0
    w = C * (z + 0.044715 * z ** 3) if name == "gelu" else z
    s = np.where(w > 0, 1 / (1 + np.exp(-np.abs(w))), np.exp(-np.abs(w)) / (1 + np.exp(-np.abs(w))))
    r = (3 * _act(z, name)[2] * (1 - s) + 8) * U
    return s * (r * np.abs(1 + z * q * (1 - s)) + np.abs(z * q) * (s * r + 2 * U) + 6 * U * (1 + np.abs(z * q) * (1 - s)))


def _blocks(rng, rows, K, group, dev, spread=True):
    import torch
    from nlearn_amd.kernels.fp8 import quantize_fp8

    x = rng.standard_normal((rows, K))
    if spread:
        x *= 2.0 ** rng.integers(-2, 3, (rows, 1))
    b = quantize_fp8(torch.from_numpy(x.astype(np.float32)).to(dev), group)
    return b, _np(b.dequantize())


def _sums(A, B, wide):
    """(A B^T, the bound of its error)."""
    size = np.abs(A) @ np.abs(B).T
    return A @ B.T, size * (A.shape[1] * U + (0 if wide else 7 * 2.0 ** -13))


def _finish(z, e, bias, name, res, rounded=0.0):
    """(y, the bound of its error before the result's rounding) from the sum and its bound."""
    if bias is not None:
        z = z + bias
        e = e + U * np.abs(z)
    e = e + rounded * np.abs(z)
    y, _, t = _act(z, name)
    if name is not None:
        e = (1.13 if name == "gelu" else 1.1 if name == "silu" else 1.0) * e + np.abs(y) * (3 * t + 8) * U
    if res is not None:
        y = y + res
        e = e + U * (np.abs(y) + np.abs(res))
    return y, e


def _check_8_bits(b, y, e):
    """Every byte is that of a value within e of y, under a scale that such values have."""
    import torch

    got, scale = (t.contiguous().view(torch.uint8).cpu().numpy() for t in (b.q, b.scale))
    M, N = y.shape
    kb = -(-N // 128)
    pad = lambda v: np.pad(v, ((0, 0), (0, kb * 128 - N)))  # noqa: E731
    assert b.shape == (M, N) and b.group == 1 and got.shape == (M, kb * 128) and scale.shape == (M, kb)
    y, e = pad(y), pad(e)
    hi = np.abs(y) + e
    lo = np.maximum(np.abs(y) - e, 0)
    smin, smax = orc.quantize(lo, 1)[1], orc.quantize(hi, 1)[1]
    # A block whose values may all be 0 within e may have any largest value in [0, max hi]: a scale up to that
    # one's, or 127, that of zeros alone (smin, formed from zeros, would be 127 there and not the least).
    nothing = lo.reshape(M, kb, 128).max(2) == 0
    ok = (scale <= smax) & (nothing | (scale >= smin)) | (nothing & (scale == 127))
    assert ok.all(), np.argwhere(~ok)[:3].tolist()
    f = np.repeat(2.0 ** (scale.astype(float) - 127), 128, 1)
    table = orc.e4m3_table()
    v = table[got]
    least, most = (table[orc.e4m3_bytes(np.clip((y + k * e) / f, -448, 448))] for k in (-1, 1))
    bad = ~((v >= least) & (v <= most))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist())
    assert (got[:, N:] == 0).all()


# 256 x 256 tiles and 128 x 128 ones, split over K or not, their edges, one row, lengths of a few
SHAPES = [(1, 128, 512), (1, 2048, 512), (5, 333, 1000), (64, 512, 4096), (128, 128, 128), (130, 260, 77), (257, 131, 300),
          (777, 1000, 333), (4200, 4100, 200), (4096, 4096, 384), (3, 1, 5), (200, 8, 640)]
FORMS = [("gelu", True, False), ("silu", True, True), ("relu", False, True), (None, True, True), (None, False, True)]


@pytest.mark.parametrize("out", ["bfloat16", "float32", "float8_e4m3fn"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_with_epilogue(dev, M, N, K, out):
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    rng = _rng(M, N, K)
    a, A = _blocks(rng, M, K, 1, dev)
    b, B = _blocks(rng, N, K, 1 if N % 2 else 128, dev, spread=False)
    B /= 1.0
    dt = getattr(torch, out)
    rt = torch.bfloat16 if out == "float8_e4m3fn" else dt
    bias = torch.from_numpy((3 * rng.standard_normal(N)).astype(np.float32)).to(dev)
    res = torch.from_numpy((5 * rng.standard_normal((M, N))).astype(np.float32)).to(dev).to(rt)
    z, e = _sums(A, B, out == "float32")
    for name, with_bias, with_res in FORMS if M * N < 1 << 22 else FORMS[:2]:
        got = gemm_fp8(a, b, out_dtype=dt, bias=bias if with_bias else None, activation=name,
                       residual=res if with_res else None)
        y, bound = _finish(z, e, _np(bias) if with_bias else None, name, _np(res) if with_res else None)
        if out == "float8_e4m3fn":
            _check_8_bits(got, y, bound)
            continue
        assert got.dtype is dt and got.shape == (M, N)
        bad = ~(np.abs(_np(got) - y) <= bound * (1 + HALF[out]) + HALF[out] * np.abs(y) + 2.0 ** -133)
        assert not bad.any(), (name, int(bad.sum()), np.argwhere(bad)[:3].tolist())
    if out == "float8_e4m3fn":  # nothing but the change of type
        _check_8_bits(gemm_fp8(a, b, out_dtype=dt), z, e)


@pytest.mark.parametrize("M,N,K", [(300, 136, 200), (64, 512, 2048), (300, 133, 200), (5, 3, 130), (4096, 4104, 128)])
def test_product_into_rows_of_the_callers(dev, M, N, K):
    """out and residual as slices of wider matrices, out over the residual: nothing else is written."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    rng = _rng(M, N, K, 1)
    a, _ = _blocks(rng, M, K, 1, dev)
    b, _ = _blocks(rng, N, K, 128, dev)
    bias = torch.from_numpy(rng.standard_normal(N).astype(np.float32)).to(dev)
    for dt in (torch.bfloat16, torch.float32):
        r = torch.from_numpy(rng.standard_normal((M, N)).astype(np.float32)).to(dev).to(dt)
        want = gemm_fp8(a, b, out_dtype=dt, bias=bias, activation="silu", residual=r)
        ld = (N + 7) // 8 * 8 + 16
        wide = torch.full((M, ld), 7.0, dtype=dt, device=dev)
        into = wide[:, 8:8 + N]
        odd = torch.empty((M, N + 3), dtype=dt, device=dev)[:, 1:1 + N]  # rows off 16 bytes
        odd.copy_(r)
        assert gemm_fp8(a, b, out=into, bias=bias, activation="silu", residual=odd) is into
        assert torch.equal(into, want) and (wide[:, :8] == 7).all() and (wide[:, 8 + N:] == 7).all()
        into.copy_(r)
        gemm_fp8(a, b, out=into, bias=bias, activation="silu", residual=into)
        assert torch.equal(into, want) and (wide[:, :8] == 7).all() and (wide[:, 8 + N:] == 7).all()
        # a bf16 bias is the fp32 one that it stands for; without a workspace K is one sum
        short = gemm_fp8(a, b, out_dtype=dt, bias=bias.bfloat16(), ws=torch.empty(1, device=dev))
        assert torch.equal(short, gemm_fp8(a, b, out_dtype=dt, bias=bias.bfloat16().float(), ws=torch.empty(1, device=dev)))


def test_product_keeps_what_the_plain_one_gives(dev):
    """A residual of zeros and no activation: the plain product bit for bit, on every tile and split."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    for M, N, K in SHAPES:
        rng = _rng(M, N, K, 2)
        a, _ = _blocks(rng, M, K, 1, dev)
        b, _ = _blocks(rng, N, K, 128, dev)
        for dt in (torch.bfloat16, torch.float32):
            want = gemm_fp8(a, b, out_dtype=dt)
            got = gemm_fp8(a, b, out_dtype=dt, residual=torch.zeros((M, N), dtype=dt, device=dev))
            assert torch.equal(got, want), (M, N, K, dt)
            assert torch.equal(gemm_fp8(a, b, out_dtype=dt, residual=torch.zeros((M, N), dtype=dt, device=dev)), got)


def test_product_of_nothing_and_not_finite(dev):
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks, gemm_fp8

    bias = torch.linspace(-3, 3, 200, device=dev)
    res = torch.ones((50, 200), dtype=torch.bfloat16, device=dev)
    a, b = Fp8Blocks.empty(50, 0, 1, dev), Fp8Blocks.empty(200, 0, 1, dev)
    y = gemm_fp8(a, b, out_dtype=torch.bfloat16, bias=bias, activation="relu", residual=res)
    assert torch.equal(y, (bias.clamp(min=0) + 1).bfloat16().expand(50, 200))
    q = gemm_fp8(a, b, out_dtype=torch.float8_e4m3fn, bias=bias)
    np.testing.assert_allclose(_np(q.dequantize()), np.broadcast_to(_np(bias), (50, 200)), rtol=2.0 ** -4, atol=2.0 ** -15)
    for M, N in ((0, 5), (5, 0)):
        e = [Fp8Blocks.empty(r, 100, 1, dev) for r in (M, N)]
        assert gemm_fp8(*e, activation="gelu").shape == (M, N)
        assert gemm_fp8(*e, out_dtype=torch.float8_e4m3fn).shape == (M, N)
    rng = _rng(3)
    for M, K in ((200, 256), (40, 4096)):  # in one piece and split
        a, A = _blocks(rng, M, K, 1, dev)
        b, B = _blocks(rng, 200, K, 128, dev)
        res = torch.zeros((M, 200), device=dev)
        res[3, 7], res[4, 8], res[5, 9] = float("nan"), float("inf"), float("-inf")
        bias2 = bias.clone()
        bias2[11] = float("nan")
        for act in ("relu", "gelu", "silu", None):
            clean = gemm_fp8(a, b, out_dtype=torch.float32, bias=bias, activation=act)
            y = gemm_fp8(a, b, out_dtype=torch.float32, bias=bias2, activation=act, residual=res)
            assert torch.isnan(y[:, 11]).all() and torch.isnan(y[3, 7])
            assert y[4, 8] == float("inf") and y[5, 9] == float("-inf")
            keep = torch.isfinite(res)
            keep[:, 11] = False
            assert torch.equal(y[keep], clean[keep])
            e = gemm_fp8(a, b, out_dtype=torch.float8_e4m3fn, bias=bias2, activation=act, residual=res.bfloat16())
            v = _np(e.dequantize())
            assert np.isnan(v[:, 11]).all() and np.isnan([v[3, 7], v[4, 8], v[5, 9]]).all()
            v[:, 11] = v[3, 7] = v[4, 8] = v[5, 9] = 0
            assert np.isfinite(v).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols,ld", [(1, 1, 1), (130, 259, 264), (257, 128, 129), (40, 1000, 1000), (1000, 72, 80)])
def test_output_gradient_behind_an_activation(dev, rows, cols, ld, dtype):
    """d = dy act'(u) quantised both ways, and its column sums."""
    import ctypes

    import torch
    from nlearn_amd import _lib
    from nlearn_amd.kernels.fp8 import ACTIVATIONS, Fp8Blocks

    rng, dt = _rng(rows, cols), getattr(torch, dtype)
    make = lambda s: torch.as_strided(torch.full((rows * ld + 8,), float("nan"), dtype=dt, device=dev), (rows, cols),  # noqa: E731
                                      (ld, 1)).copy_(torch.from_numpy((s * rng.standard_normal((rows, cols))).astype(np.float32)))
    dy, u = make(1.0), make(3.0)
    code = 0 if dt is torch.float32 else 1
    for name, act in ACTIVATIONS.items():
        q, t = Fp8Blocks.empty(rows, cols, 1, dev), Fp8Blocks.empty(cols, rows, 1, dev)
        db = torch.empty(cols, device=dev)
        wsb = _lib.load().nl_quantize_fp8_dact_ws_bytes(rows, cols)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
        args = [dy.data_ptr(), code, ld, u.data_ptr(), ld, act]
        _lib.call_on(dy, "nl_quantize_fp8_dact", rows, cols, *args, *q._abi(), *t._abi(), db.data_ptr(), 0, ws.data_ptr(), wsb)
        z = _np(u)
        d = _np(dy) * _act(z, name)[1]
        e = np.abs(_np(dy)) * _slope_error(z, name)
        _check_8_bits(q, d, e)
        _check_8_bits(t, d.T, e.T)
        bound = e.sum(0) + U * (rows / 64 + 20) * np.abs(d).sum(0)
        assert (np.abs(_np(db) - d.sum(0)) <= bound).all()
        # one output at a time: the same
        q2, t2 = Fp8Blocks.empty(rows, cols, 1, dev), Fp8Blocks.empty(cols, rows, 1, dev)
        none = (None, 0, None, 0)
        _lib.call_on(dy, "nl_quantize_fp8_dact", rows, cols, *args, *q2._abi(), *none, None, 0, None, 0)
        _lib.call_on(dy, "nl_quantize_fp8_dact", rows, cols, *args, *none, *t2._abi(), None, 0, None, 0)
        db2 = torch.empty(cols, device=dev)
        _lib.call_on(dy, "nl_quantize_fp8_dact", rows, cols, *args, *none, *none, db2.data_ptr(), 0, ws.data_ptr(), wsb)
        for p, r in ((q, q2), (t, t2)):
            assert torch.equal(p.q.view(torch.uint8), r.q.view(torch.uint8))
            assert torch.equal(p.scale.contiguous().view(torch.uint8), r.scale.contiguous().view(torch.uint8))
        assert torch.equal(db, db2)
    nan = torch.full((1, 4), float("nan"), dtype=dt, device=dev)
    one, db = torch.ones((1, 4), dtype=dt, device=dev), torch.empty(4, device=dev)
    ws = torch.empty(64, dtype=torch.uint8, device=dev)
    for act in (1, 2, 3):
        _lib.call_on(one, "nl_quantize_fp8_dact", 1, 4, one.data_ptr(), code, 4, nan.data_ptr(), 4, act, None, 0, None, 0, None, 0,
                     None, 0, db.data_ptr(), 0, ws.data_ptr(), 64)
        assert torch.isnan(db).all()


def _grid_case(M, K, N, name):
    """x, W, bias and dY on grids where every sum before the activation is exact in bf16 and fp32 and no
    dY act'(u) stands within its error of a tie of its quantisation: one right answer, to the last bits of the sums."""
    rng = _rng(M, K, N, 5)
    x = rng.integers(-2, 3, (M, K)) / 2.0
    W = rng.integers(-2, 3, (K, N)) / 2.0 * (rng.random((K, N)) < 8.0 / K)
    bias = rng.integers(-4, 5, N) / 4.0
    u = x @ W + bias
    assert (np.abs(u) <= 32).all()  # quarters up to 32: 8 bits
    dy = 2.0 ** rng.integers(-3, 4, (M, N)) * rng.choice([-1.0, 1.0], (M, N))
    d = dy * _act(u, name)[1]
    e = np.abs(dy) * _slope_error(u, name)
    for v, w in ((d, e), (d.T, e.T)):
        near = [orc.values(*orc.quantize(v + k * w, 1), 1) for k in (-1, 0, 1)]
        np.testing.assert_array_equal(near[0], near[1])
        np.testing.assert_array_equal(near[2], near[1])
    return x, W, bias, u, dy, d


GRIDS = [(70, 32, 24), (300, 96, 200), (33, 130, 129), (1, 16, 40), (257, 16, 136)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("M,K,N", GRIDS)
def test_layer_and_its_gradients(dev, M, K, N, name, dtype):
    import torch
    from nlearn_amd.kernels.fp8 import fp8_weight, linear_fp8

    dt = getattr(torch, dtype)
    x, W, bias, u, dy, d = _grid_case(M, K, N, name)
    res = _rng(M, 9).standard_normal((M, N))
    dev_ = lambda v, t=dt: torch.from_numpy(v.astype(np.float32)).to(dev).to(t)  # noqa: E731
    xt, rt, dyt = dev_(x).requires_grad_(True), dev_(res).requires_grad_(True), dev_(dy)
    dq, dqt = (orc.values(*orc.quantize(v, 1), 1)[:, :v.shape[1]] for v in (d, d.T))
    wide = dtype == "float32"
    y64, _ = _finish(u, 0 * u, None, name, _np(rt))
    _, ey = _finish(u, 0 * u, None, name, _np(rt))
    dx64, edx = _sums(dq, W, wide)
    dW64, edW = _sums(x.T, dqt, True)
    db64 = d.sum(0)
    edb = np.abs(d).sum(0) * (M / 64 + 20) * U + np.abs(dy).sum(0) * 2.0 ** -20

    def near(got, want, bound, half):
        assert (np.abs(_np(got) - want) <= bound * (1 + half) + half * np.abs(want) + 1e-30).all()

    for wt in (torch.float32, torch.bfloat16):
        Wt, bt = dev_(W, wt).requires_grad_(True), dev_(bias, wt).requires_grad_(True)
        y = linear_fp8(xt, Wt, bias=bt, activation=name, residual=rt)
        assert y.dtype is dt and y.shape == (M, N)
        near(y, y64, ey, HALF[dtype])
        dx, dW, db, dr = torch.autograd.grad(y, (xt, Wt, bt, rt), dyt)
        assert dx.dtype is dt and dW.dtype is wt and db.dtype is wt and torch.equal(dr, dyt)
        hw = U if wt is torch.float32 else 2.0 ** -8
        near(dx, dx64, edx, HALF[dtype])
        near(dW, dW64, edW if wt is torch.float32 else _sums(x.T, dqt, False)[1], hw)
        near(db, db64, edb, hw)
        # each of them alone, and the forward without any
        for t, g in ((xt, dx), (Wt, dW), (bt, db), (rt, dr)):
            only = [v if v is t else v.detach() for v in (xt, Wt, bt, rt)]
            z = linear_fp8(only[0], only[1], bias=only[2], activation=name, residual=only[3])
            assert torch.equal(z, y)
            (h,) = torch.autograd.grad(z, t, dyt)
            assert torch.equal(g, h)
        with torch.no_grad():
            assert torch.equal(linear_fp8(xt, Wt, bias=bt, activation=name, residual=rt), y)
        # without a bias, without a residual
        z = linear_fp8(xt, Wt, activation=name, residual=rt) if name else linear_fp8(xt, Wt, residual=rt)
        near(z, *_finish(u - bias, 0 * u, None, name, _np(rt)), HALF[dtype])
        near(linear_fp8(xt, Wt, bias=bt, activation=name), *_finish(u, 0 * u, None, name, None), HALF[dtype])
    # buffers that an optimizer reads
    Wt, bt = dev_(W, torch.float32).requires_grad_(True), dev_(bias, torch.float32).requires_grad_(True)
    Wt.main_grad, bt.main_grad = (torch.full_like(t.detach(), 3.0) for t in (Wt, bt))
    linear_fp8(xt, Wt, bias=bt, activation=name, residual=rt).backward(dyt)
    near(Wt.main_grad, dW64, edW, U)
    near(bt.main_grad, db64, edb, U)
    assert Wt.grad is None and bt.grad is None
    # a frozen weight
    bt = dev_(bias, torch.float32).requires_grad_(True)
    y = linear_fp8(xt, fp8_weight(Wt.detach()), bias=bt, activation=name, residual=rt)
    near(y, y64, ey, HALF[dtype])
    dx, db, dr = torch.autograd.grad(y, (xt, bt, rt), dyt)
    near(dx, dx64, edx, HALF[dtype])
    near(db, db64, edb, U)
    assert torch.equal(dr, dyt)


def test_layer_leading_dimensions_strides_and_nothing(dev):
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8

    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn((3, 20, 96), generator=g, device=dev, dtype=torch.bfloat16)
    W = torch.randn((96, 52), generator=g, device=dev)
    b = torch.randn((52,), generator=g, device=dev)
    r = torch.randn((3, 20, 60), generator=g, device=dev, dtype=torch.bfloat16)[..., 3:55]
    flat = linear_fp8(x.reshape(60, 96), W, bias=b, activation="gelu", residual=r.reshape(60, 52))
    assert torch.equal(linear_fp8(x, W, bias=b, activation="gelu", residual=r).view(60, 52), flat)
    assert torch.equal(linear_fp8(x.transpose(0, 1), W, bias=b, activation="gelu", residual=r.transpose(0, 1)),
                       linear_fp8(x, W, bias=b, activation="gelu", residual=r).transpose(0, 1))
    for shape in ((0, 96), (4, 0)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        W = torch.zeros((shape[1], 10), device=dev, requires_grad=True)
        b = torch.linspace(-1, 1, 10, device=dev, requires_grad=True)
        y = linear_fp8(x, W, bias=b, activation="relu")
        assert torch.equal(y, b.detach().clamp(min=0).expand(shape[0], 10))
        y.sum().backward()
        assert x.grad.shape == shape and (W.grad == 0).all() and W.grad.shape == W.shape
        assert torch.equal(b.grad, (b.detach() > 0).float() * shape[0])


def test_layer_outputs_written_in_place_and_broadcast_residuals(dev):
    import torch
    from nlearn_amd.kernels.fp8 import fp8_weight, gemm_fp8, linear_fp8, quantize_fp8

    g = torch.Generator(device=dev).manual_seed(13)
    for N in (40, 37):
        x = torch.randn((30, 64), generator=g, device=dev, dtype=torch.bfloat16)
        W = torch.randn((64, N), generator=g, device=dev).requires_grad_(True)
        row = torch.randn((1, N), generator=g, device=dev, dtype=torch.bfloat16).requires_grad_(True)
        y = linear_fp8(x, W, activation="relu", residual=row.expand(30, N))
        want = y.detach() + 1
        y += 1
        assert torch.equal(y, want)
        dW, dr = torch.autograd.grad(y, (W, row), torch.ones_like(y))
        assert torch.equal(dr, torch.full_like(dr, 30)) and torch.isfinite(dW).all()
        # one tensor as input and residual: its gradients add up
        V = torch.randn((64, 64), generator=g, device=dev)
        z = x.clone().requires_grad_(True)
        (both,) = torch.autograd.grad(linear_fp8(z, V, residual=z), z, torch.ones_like(z))
        (one,) = torch.autograd.grad(linear_fp8(z, V, residual=x), z, torch.ones_like(z))
        assert torch.equal(both, one + 1)
        f = fp8_weight(W.detach())
        r = torch.randn((30, N), generator=g, device=dev, dtype=torch.bfloat16)
        assert torch.equal(linear_fp8(x, f, residual=r), gemm_fp8(quantize_fp8(x), f.fwd, residual=r))


def test_bias_gradient_against_differences(dev):
    """The bias is not quantised: d(sum dY y)/db against central differences of the fp32 layer itself."""
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8

    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn((40, 64), generator=g, device=dev)
    W = torch.randn((64, 48), generator=g, device=dev) / 8
    b = torch.randn((48,), generator=g, device=dev).requires_grad_(True)
    dy = torch.randn((40, 48), generator=g, device=dev)
    h = 2.0 ** -7
    for name in ("gelu", "silu", None):
        y = linear_fp8(x, W, bias=b, activation=name)
        (db,) = torch.autograd.grad(y, b, dy)
        with torch.no_grad():
            up, down = (linear_fp8(x, W, bias=b + k, activation=name).double() for k in (h, -h))
            slope = ((up - down) * dy.double()).sum(0) / (2 * h)
            # |act'''| < 3 for both: h^2 / 2 each; a value's roundings (80 u of |y| + 1) over 2 h
            bound = dy.double().abs().sum(0) * (0.5 * h * h) + (dy.double().abs() * (y.double().abs() + 1)).sum(0) * 80 * U / h
        assert ((db.double() - slope).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_relu_drops_gradients_that_are_not_finite(dev, dtype):
    """Behind relu an output gradient counts where u > 0 and nowhere else, infinities and NaN among them."""
    import torch
    from nlearn_amd import _lib

    dt = getattr(torch, dtype)
    u = torch.tensor([[-1.0, 0.0, 2.0, -0.0, 3.0, float("-inf"), float("inf"), float("nan")]], device=dev)
    u = u.repeat(130, 20).to(dt)
    dy = torch.ones_like(u)
    dy[:, 0::8], dy[:, 1::8], dy[:, 5::8] = float("inf"), float("nan"), float("-inf")
    rows, cols = u.shape
    from nlearn_amd.kernels.fp8 import Fp8Blocks

    want = torch.where(u > 0, dy, torch.zeros_like(dy))
    want[:, 7::8] = float("nan")
    q, t = Fp8Blocks.empty(rows, cols, 1, dev), Fp8Blocks.empty(cols, rows, 1, dev)
    only = Fp8Blocks.empty(rows, cols, 1, dev)
    db = torch.empty(cols, device=dev)
    wsb = _lib.load().nl_quantize_fp8_dact_ws_bytes(rows, cols)
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
    args = [dy.data_ptr(), 0 if dt is torch.float32 else 1, cols, u.data_ptr(), cols, 1]
    _lib.call_on(dy, "nl_quantize_fp8_dact", rows, cols, *args, *q._abi(), *t._abi(), db.data_ptr(), 0, ws.data_ptr(), wsb)
    _lib.call_on(dy, "nl_quantize_fp8_dact", rows, cols, *args, *only._abi(), None, 0, None, 0, None, 0, None, 0)
    for got in (q.dequantize(), t.dequantize().T, only.dequantize()):
        torch.testing.assert_close(got, want.float(), rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(db, want.float().sum(0), rtol=0, atol=0, equal_nan=True)


def test_layer_without_outputs(dev):
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8

    x = torch.ones((2, 3, 8), device=dev, requires_grad=True)
    y = linear_fp8(x, torch.zeros((8, 0), device=dev), residual=torch.zeros((2, 3, 0), device=dev))
    assert y.shape == (2, 3, 0)
    y.sum().backward()
    assert (x.grad == 0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", [(3, 20, 16), (200, 136, 24), (300, 300, 260), (40, 500, 2100), (4096, 4100, 130)])
def test_relu_passes_gradients_where_the_exact_sum_is_positive(dev, M, N, K, dtype):
    """Products of 2^16 that cancel beside small ones: the sum is a small whole number (every partial sum is one below
    2^24, exact in fp32 in any order), and its sign decides whether a gradient passes."""
    import torch
    from nlearn_amd.kernels.fp8 import fp8_weight, linear_fp8

    g = torch.Generator(device=dev).manual_seed(M + N)
    x = torch.randint(-2, 3, (M, K), generator=g, device=dev).float()
    W = torch.randint(-1, 2, (K, N), generator=g, device=dev).float()
    for k in range(0, K - 1, 16):
        x[:, k] = x[:, k + 1] = 256
        W[k], W[k + 1] = 256, -256
    u = (x.double() @ W.double()).float()
    assert u.abs().max() <= 256  # whole numbers in bf16
    x = x.to(getattr(torch, dtype))
    bias = torch.zeros((N,), device=dev).requires_grad_(True)
    for weight in (W, fp8_weight(W)):
        for res in (None, torch.ones((M, N), device=dev, dtype=x.dtype)):
            y = linear_fp8(x, weight, bias=bias, activation="relu", residual=res)
            assert torch.equal(y.float(), u.clamp(min=0) + (0 if res is None else 1))
            (db,) = torch.autograd.grad(y, bias, torch.ones_like(y))
            assert torch.equal(db, (u > 0).float().sum(0))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", [(4096, 4100, 24), (4200, 4096, 2200)])
def test_relu_on_large_tiles(dev, M, N, K, dtype):
    """The same with u kept and not, with a residual and without: whole numbers, exact in fp32, on 256 x 256 tiles too."""
    import torch
    from nlearn_amd.kernels.fp8 import fp8_weight, linear_fp8

    g = torch.Generator(device=dev).manual_seed(M + N)
    x = torch.randint(-2, 3, (M, K), generator=g, device=dev).float()
    W = torch.randint(-1, 2, (K, N), generator=g, device=dev).float()
    W *= torch.rand((K, N), generator=g, device=dev) < 0.1
    for k in range(0, K - 1, 16):
        x[:, k] = x[:, k + 1] = 256
        W[k], W[k + 1] = 256, -256
    u = (x.double() @ W.double()).float()
    assert u.abs().max() <= 255  # whole numbers in bf16, with the residual too
    x = x.to(getattr(torch, dtype))
    bias = torch.zeros((N,), device=dev)
    for res in (None, torch.ones((M, N), device=dev, dtype=x.dtype)):
        want = u.clamp(min=0) + (0 if res is None else 1)
        for weight in (W, fp8_weight(W)):
            assert torch.equal(linear_fp8(x, weight, bias=bias, activation="relu", residual=res).float(), want)
            leaf = bias.clone().requires_grad_(True)
            y = linear_fp8(x, weight, bias=leaf, activation="relu", residual=res)
            assert torch.equal(y.float(), want)
            (db,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
            assert torch.equal(db, (u > 0).float().sum(0))


@pytest.mark.parametrize("M,N,K", [(1, 300, 300), (130, 260, 77), (64, 512, 4000), (300, 133, 700), (4096, 4100, 300)])
def test_scale_rows_of_any_length(dev, M, N, K):
    """Scales whose rows are no whole dwords: the bits that padded ones give, in every form of the epilogue."""
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks, Fp8Weight, fp8_weight, gemm_fp8, linear_fp8

    def compact(b):
        kb = b.scale.shape[1]
        rows = torch.empty((b.scale.shape[0], kb + 1 - kb % 2), dtype=torch.uint8, device=dev)  # an odd stride
        rows[:, :kb] = b.scale.contiguous().view(torch.uint8)
        return Fp8Blocks(b.q, rows.view(torch.float8_e8m0fnu)[:, :kb], b.shape, b.group)

    rng = _rng(M, N, K, 9)
    a, _ = _blocks(rng, M, K, 1, dev)
    b, _ = _blocks(rng, N, K, 1, dev)
    odd = compact(a), compact(b)
    assert odd[0].scale.stride(0) % 2 == 1 or M == 1
    bias = torch.from_numpy(rng.standard_normal(N).astype(np.float32)).to(dev)
    bytes_ = lambda t: t if torch.is_tensor(t) else torch.cat([t.q.view(torch.uint8).flatten(),  # noqa: E731
                                                               t.scale.contiguous().view(torch.uint8).flatten()])
    for dt in (torch.bfloat16, torch.float32, torch.float8_e4m3fn):
        rt = torch.bfloat16 if dt is torch.float8_e4m3fn else dt
        res = torch.from_numpy(rng.standard_normal((M, N)).astype(np.float32)).to(dev).to(rt)
        for r in (None, res):
            want, got = (gemm_fp8(*ab, out_dtype=dt, bias=bias, activation="gelu", residual=r) for ab in ((a, b), odd))
            assert torch.equal(bytes_(want), bytes_(got)), (dt, r is None)
    # a frozen weight's, with u kept
    W = torch.from_numpy(rng.standard_normal((K, N)).astype(np.float32) / K ** 0.5).to(dev)
    f = fp8_weight(W)
    f2 = Fp8Weight(compact(f.fwd), compact(f.bwd))
    for dt in (torch.bfloat16, torch.float32):
        x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(dev).to(dt).requires_grad_(True)
        for name in ("gelu", "relu"):
            for r in (None, torch.ones((M, N), device=dev, dtype=dt)):
                y, y2 = (linear_fp8(x, w, bias=bias, activation=name, residual=r) for w in (f, f2))
                assert torch.equal(y, y2)
                assert torch.equal(*(torch.autograd.grad(v, x, torch.ones_like(v))[0] for v in (y, y2)))
