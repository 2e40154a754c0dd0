"""8-bit block-scaled operands and their product on the GPU, against float64.

Quantised bytes and scales are exact: a power-of-two scale and one rounding have
one right answer, so they are compared bit for bit. A product's error is bounded
per element: K products exact in fp32 summed with K roundings of half a step
(2^-24) of at most sum |a b|. A bf16 result is formed by the 8-bit matrix
instructions, which cut 8 products at a time to a grid of 2^(E - 13), E the largest
sum of two exponents among the 8 (a subnormal counts with the exponent -6, a zero
not at all). The largest product itself has 8 significant bits and stays whole, so
7 of them lose less than 2^-13 of 2^E each, and 2^E is at most the sum over the 8
of pa pb, p the power of two below a value: 7 * 2^-13 sum pa pb in all. Then one
rounding of half a step, 2^-8 of the value.
"""
import numpy as np
import pytest

from oracle import distill_fp8 as orc

pytestmark = pytest.mark.gpu


def _rng(*key):
    return np.random.default_rng(list(key))


def _matrix(rng, rows, cols):
    x = rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-6, 7, (rows, 1))
    x *= np.where(rng.random((rows, cols)) < 0.01, 64.0, 1.0)
    return x.astype(np.float32)


def _device(x, dtype, dev, stride=None, shift=0):
    """x on the GPU with a row stride and a shift (elements) from an aligned base."""
    import torch

    rows, cols = x.shape
    buf = torch.full((rows * (stride or cols) + shift + 8,), float("nan"), dtype=dtype, device=dev)
    t = torch.as_strided(buf, (rows, cols), (stride or cols, 1), shift)
    t.copy_(torch.from_numpy(x).to(dev))
    return t


def _bytes(t):
    import torch

    return t.contiguous().view(torch.uint8).cpu().numpy()


def _check_blocks(b, x64, group):
    q, s = orc.quantize(x64, group)
    assert b.shape == x64.shape and b.group == group
    np.testing.assert_array_equal(_bytes(b.scale), s)
    got = _bytes(b.q)
    # e4m3 has two NaN bytes, 0x7f and 0xff, that stand for the same
    np.testing.assert_array_equal(np.where(got == 0xff, 0x7f, got), q)


SHAPES = [(1, 1), (1, 128), (3, 7), (5, 129), (127, 128), (129, 300), (200, 1000), (513, 127), (1000, 333)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_is_exact(dev, rows, cols, dtype):
    import torch
    from nlearn_amd.kernels.fp8 import quantize_fp8, quantize_fp8_both

    dt = getattr(torch, dtype)
    x = _device(_matrix(_rng(rows, cols), rows, cols), dt, dev)
    x64 = x.double().cpu().numpy()
    for group in (1, 128):
        _check_blocks(quantize_fp8(x, group), x64, group)
        _check_blocks(quantize_fp8(x, group, transpose=True), x64.T, group)
        a, t = quantize_fp8_both(x, group)
        _check_blocks(a, x64, group)
        _check_blocks(t, x64.T, group)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("stride,shift", [(264, 0), (261, 0), (264, 1), (256 + 8, 3)])
def test_quantize_strided_and_unaligned(dev, dtype, stride, shift):
    import torch
    from nlearn_amd.kernels.fp8 import quantize_fp8_both

    x = _device(_matrix(_rng(stride, shift), 150, 259), getattr(torch, dtype), dev, stride, shift)
    x64 = x.double().cpu().numpy()
    a, t = quantize_fp8_both(x)
    _check_blocks(a, x64, 1)
    _check_blocks(t, x64.T, 1)
    # a transposed view and rows that share memory are copied first
    _check_blocks(quantize_fp8_both(x.t())[0], x64.T, 1)
    _check_blocks(quantize_fp8_both(x[:1].expand(5, 259))[1], np.repeat(x64[:1], 5, 0).T, 1)


def test_quantize_every_bf16_value(dev):
    """All 65536 bf16 patterns, with infinities and NaN, in blocks of unlike ranges."""
    import torch
    from nlearn_amd.kernels.fp8 import quantize_fp8

    bits = np.arange(65536, dtype=np.uint16)
    for order in (bits.reshape(512, 128), bits.reshape(128, 512).T.copy()):
        x = torch.from_numpy(order.view(np.int16)).to(dev).view(torch.bfloat16)
        _check_blocks(quantize_fp8(x), x.double().cpu().numpy(), 1)


def test_quantize_borders(dev):
    """Scales at their borders, values at the ties, blocks of zeros and tiny ones, no finite value at all."""
    import torch
    from nlearn_amd.kernels.fp8 import quantize_fp8, quantize_fp8_both

    x = np.zeros((12, 256), np.float32)
    x[0, 0], x[1, 0], x[2, 0] = 448, np.nextafter(np.float32(448), np.float32(449)), 447.9
    x[3, :2] = 1e-40, -1e-44               # subnormals: the least scale
    x[4, :2] = 3e38, -1
    x[5, :3] = np.inf, np.nan, 5
    x[6, :] = np.inf
    x[7, 128:] = np.nan
    x[8, :128] = 256 + np.arange(128)      # every tie between 256 and 384
    x[9, :128] = np.arange(128) * 2.0 ** -10
    x[9, 127] = 448                        # ties below the normal range
    x[10, :] = -0.0
    x[11, 255] = -448 * 2.0 ** 100
    t = torch.from_numpy(x).to(dev)
    for group in (1, 128):
        a, b = quantize_fp8_both(t, group)
        _check_blocks(a, x.astype(np.float64), group)
        _check_blocks(b, x.T.astype(np.float64), group)
    assert torch.isnan(quantize_fp8(t).dequantize()[6]).all()


def test_quantize_empty(dev):
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8, linear_fp8, quantize_fp8_both

    for rows, cols in ((0, 5), (5, 0), (0, 0)):
        a, t = quantize_fp8_both(torch.empty((rows, cols), device=dev))
        assert a.shape == (rows, cols) and t.shape == (cols, rows)
    a, _ = quantize_fp8_both(torch.empty((3, 0), device=dev))
    b, _ = quantize_fp8_both(torch.empty((4, 0), device=dev))
    assert torch.equal(gemm_fp8(a, b), torch.zeros((3, 4), dtype=torch.bfloat16, device=dev))
    W = torch.ones((16, 8), device=dev, requires_grad=True)
    y = linear_fp8(torch.empty((0, 16), dtype=torch.bfloat16, device=dev, requires_grad=True), W)
    assert y.shape == (0, 8)
    y.sum().backward()
    assert torch.count_nonzero(W.grad) == 0


def _operand(rng, rows, K, group, dev, padded=True):
    """A quantised operand from random bytes and scales, and its float64 values."""
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks

    kb = (K + 127) // 128
    q = rng.integers(0, 256, (rows, kb * 128)).astype(np.uint8)
    q[(q & 0x7f) == 0x7f] = 0x30
    q[:, K:] = 0
    s = rng.integers(120, 135, ((rows + group - 1) // group, kb)).astype(np.uint8)
    buf = torch.full((s.shape[0], (kb + 3) // 4 * 4 if padded else kb), 255, dtype=torch.uint8, device=dev)
    buf[:, :kb] = torch.from_numpy(s).to(dev)
    b = Fp8Blocks(torch.from_numpy(q).to(dev).view(torch.float8_e4m3fn),
                  buf.view(torch.float8_e8m0fnu)[:, :kb], (rows, K), group)
    return b, _values(q, s, group, K, dev)


def _values(q, s, group, K, dev):
    """Float64 values of an operand, and the powers of two below them as the matrix unit aligns products."""
    import torch

    u = np.abs(orc.e4m3_table()[q])
    p = np.where(u > 0, 2.0 ** np.floor(np.log2(np.maximum(u, 2.0 ** -6))), 0.0)
    f = np.repeat(np.repeat(2.0 ** (s.astype(float) - 127), group, 0)[:q.shape[0]], orc.BLOCK, 1)
    return tuple(torch.from_numpy((t * f)[:, :K]).to(dev) for t in (orc.e4m3_table()[q], p))


def _check_product(out, a, b, K):
    import torch

    ref, mag = a[0] @ b[0].t(), a[0].abs() @ b[0].abs().t()
    lim = (K + 2) * 2.0 ** -24 * mag
    if out.dtype == torch.bfloat16:
        lim = (lim + 7 * 2.0 ** -13 * (a[1] @ b[1].t())) * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs()
    bad = (out.double() - ref).abs() > lim
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[0].tolist())


PRODUCTS = [  # M, N, K: one of each tile, odd sizes, K inside a block, splits
    (1, 1, 1), (1, 1, 128), (2, 3, 130), (1, 333, 1000), (17, 40, 640), (64, 64, 2048), (128, 128, 128),
    (129, 257, 384), (200, 1000, 515), (8, 2048, 512), (96, 96, 16384), (512, 500, 8200),
    (4096, 4100, 300), (4000, 4096, 1152), (300, 50257, 130),
]


@pytest.mark.parametrize("ga,gb", [(1, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_gemm_against_float64(dev, M, N, K, ga, gb):
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    rng = _rng(M, N, K)
    a, a64 = _operand(rng, M, K, ga, dev)
    b, b64 = _operand(rng, N, K, gb, dev, padded=M % 2 == 0)
    for dt in (torch.float32, torch.bfloat16):
        out = gemm_fp8(a, b, dt)
        assert out.dtype == dt and out.shape == (M, N)
        _check_product(out, a64, b64, K)
        assert torch.equal(out, gemm_fp8(a, b, dt))


def test_gemm_places_every_byte(dev):
    """One-hot rows pick single elements: any wrong pairing of k, row or scale shows as a wrong value."""
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks, gemm_fp8

    rng = _rng(5)
    for N, K in ((40, 512), (513, 1408)):
        b, b64 = _operand(rng, N, K, 1, dev)
        q = torch.zeros((K, K), dtype=torch.uint8, device=dev)
        q[torch.arange(K), torch.arange(K)] = 0x38  # 1.0
        s = torch.full((K, K // 128), 127, dtype=torch.uint8, device=dev)
        eye = Fp8Blocks(q.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu), (K, K), 1)
        for dt in (torch.float32, torch.bfloat16):  # an e4m3 value times a power of two is exact in either
            assert torch.equal(gemm_fp8(eye, b, dt).double(), b64[0].t())
            assert torch.equal(gemm_fp8(b, eye, dt).double(), b64[0])


def test_gemm_extreme_scales_and_nan(dev):
    """The least and largest scales of an operand, and a NaN that stays in its row."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8, quantize_fp8

    x = torch.ones((40, 256), device=dev)
    x[0] *= 2.0 ** -126
    x[1] *= 2.0 ** 120
    x[2, 200] = float("nan")
    x[3, 5] = float("inf")
    w = torch.full((33, 256), 0.5, device=dev)
    y = gemm_fp8(quantize_fp8(x), quantize_fp8(w), torch.float32).cpu()
    assert (y[0] == 128 * 2.0 ** -126).all() and (y[1] == 128 * 2.0 ** 120).all()
    assert torch.isnan(y[2:4]).all() and (y[4:] == 128).all()


def test_gemm_into_a_strided_output(dev):
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    rng = _rng(9)
    a, a64 = _operand(rng, 70, 300, 1, dev)
    b, b64 = _operand(rng, 45, 300, 128, dev)
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.full((71, 64), 7.0, dtype=dt, device=dev)
        out = gemm_fp8(a, b, out=buf[:70, :45])
        _check_product(out, a64, b64, 300)
        assert (buf[70] == 7).all() and (buf[:, 45:] == 7).all()


def test_gemm_rows_past_32_bit_offsets(dev):
    """Operands and outputs of more than 4 GiB: the last rows are the right ones."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8, quantize_fp8

    M, K = 4_300_000, 1024
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=dev)
    x[0, 3], x[-1, 1000], x[M // 2, 512] = 2.0, -3.0, 5.0
    w = torch.zeros((520, K), dtype=torch.bfloat16, device=dev)
    w[:, 3], w[:, 512], w[:, 1000] = 1.0, 2.0, 4.0
    y = gemm_fp8(quantize_fp8(x), quantize_fp8(w))
    assert (y[0] == 2).all() and (y[-1] == -12).all() and (y[M // 2] == 10).all()
    assert int((y != 0).sum()) == 3 * 520


def _quantised(x, group=1):
    return _values(*orc.quantize(x.detach().double().cpu().numpy(), group), group, x.shape[1], x.device)


@pytest.mark.parametrize("lead,K,N", [((1,), 16, 24), ((5,), 100, 33), ((3, 77), 512, 200), ((777,), 1000, 333),
                                      ((2, 300), 130, 1024)])
@pytest.mark.parametrize("wdtype", ["float32", "bfloat16"])
def test_linear_forward_and_gradients(dev, lead, K, N, wdtype):
    """y, dX and dW are the products of the quantised operands."""
    import torch
    from nlearn_amd.kernels.fp8 import fp8_weight, linear_fp8

    rng = _rng(K, N)
    M = int(np.prod(lead))
    x = torch.from_numpy(_matrix(rng, M, K)).to(dev).to(torch.bfloat16).reshape(*lead, K).requires_grad_(True)
    W = (torch.from_numpy(_matrix(rng, K, N)).to(dev) * 0.05).to(getattr(torch, wdtype)).requires_grad_(True)
    dy = torch.from_numpy(_matrix(rng, M, N)).to(dev).to(torch.bfloat16).reshape(*lead, N)
    y = linear_fp8(x, W)
    # each gradient alone is the same as with the other
    (gx,) = torch.autograd.grad(linear_fp8(x, W.detach()), x, dy)
    (gW,) = torch.autograd.grad(linear_fp8(x.detach(), W), W, dy)
    assert torch.equal(linear_fp8(x.detach(), W.detach()), y)
    y.backward(dy)
    assert torch.equal(gx, x.grad) and torch.equal(gW, W.grad)
    assert y.dtype == torch.bfloat16 and x.grad.dtype == torch.bfloat16 and W.grad.dtype == W.dtype
    x2, dy2 = x.detach().reshape(M, K), dy.reshape(M, N)
    Wq = _quantised(W, 128)
    _check_product(y.detach().reshape(M, N), _quantised(x2), [w.t() for w in Wq], K)
    _check_product(x.grad.reshape(M, K), _quantised(dy2), Wq, N)
    _check_product(W.grad, _quantised(x2.t()), _quantised(dy2.t()), M)
    # a weight laid out beforehand gives the same output and input gradient, and no gradient of its own
    x1 = x.detach().clone().requires_grad_(True)
    y1 = linear_fp8(x1, fp8_weight(W.detach()))
    y1.backward(dy)
    assert torch.equal(y1, y) and torch.equal(x1.grad, x.grad)


def test_linear_gradient_against_differences(dev):
    """On values that e4m3 holds exactly the product is linear and differences are exact."""
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8

    rng = _rng(21)
    M, K, N = 6, 20, 10
    x = torch.from_numpy(rng.integers(-4, 5, (M, K)).astype(np.float32)).to(dev)
    W = torch.from_numpy(rng.integers(-4, 5, (K, N)).astype(np.float32)).to(dev)
    dy = torch.from_numpy(rng.integers(-4, 5, (M, N)).astype(np.float32)).to(dev)
    xg, Wg = x.clone().requires_grad_(True), W.clone().requires_grad_(True)
    (linear_fp8(xg, Wg) * dy).sum().backward()
    f = lambda x_, W_: float((linear_fp8(x_, W_).double() * dy.double()).sum())  # noqa: E731
    for (i, j) in ((0, 0), (3, 7), (5, 9)):
        for leaf, grad in ((0, xg.grad), (1, Wg.grad)):
            hi, lo = [x.clone(), W.clone()], [x.clone(), W.clone()]
            hi[leaf][i, j] += 1
            lo[leaf][i, j] -= 1
            assert float(grad[i, j]) == (f(*hi) - f(*lo)) / 2


def test_linear_main_grad_broadcast_cotangent_and_reuse(dev):
    """main_grad takes dW (with the side stream too), a broadcast dY is read as what it stands for, and a
    double backward or a wrong call is refused."""
    import torch
    from nlearn_amd.kernels import wgrad
    from nlearn_amd.kernels.fp8 import linear_fp8

    rng = _rng(22)
    x = torch.from_numpy(_matrix(rng, 300, 128)).to(dev).to(torch.bfloat16).requires_grad_(True)
    W = torch.from_numpy(_matrix(rng, 128, 40)).to(dev).requires_grad_(True)
    linear_fp8(x, W).sum().backward()           # dY: one element seen (300, 40) times
    gx, gW = x.grad.clone(), W.grad.clone()
    dy = torch.ones((300, 40), dtype=torch.bfloat16, device=dev)
    W.main_grad = torch.full((128, 40), float("nan"), device=dev)
    x.grad = W.grad = None
    with wgrad.overlap_weight_grads():
        linear_fp8(x, W).backward(dy)
    assert W.grad is None and torch.equal(W.main_grad, gW) and torch.equal(x.grad, gx)
    del W.main_grad
    y = linear_fp8(x, W)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_product_in_a_graph_and_on_two_streams(dev):
    """Captured and replayed with new inputs, beside eager calls of the same shapes; two streams at once."""
    import torch
    from nlearn_amd.kernels.fp8 import fp8_weight, linear_fp8

    rng = _rng(31)
    W = torch.from_numpy(_matrix(rng, 2048, 96)).to(dev)
    w = fp8_weight(W)
    xs = [torch.from_numpy(_matrix(rng, 50, 2048)).to(dev).to(torch.bfloat16) for _ in range(4)]
    want = [linear_fp8(x, w) for x in xs]
    side = torch.cuda.Stream(dev)
    buf = xs[0].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        linear_fp8(buf, w)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs over one input buffer
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(linear_fp8(buf, w))
        graphs.append(g)
    for x, ref in zip(xs, want):
        buf.copy_(x)
        for g, out in zip(graphs, outs):
            out.zero_()
            g.replay()
            linear_fp8(xs[1], w)
            torch.cuda.synchronize()
            assert torch.equal(out, ref)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(linear_fp8(xs[i % 4], w))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4])


@pytest.mark.parametrize("K,N", [(64, 50), (130, 7)])
def test_linear_main_grad_of_odd_rows(dev, K, N):
    """A main_grad laid out like a contiguous weight has rows off 16 bytes: it gets the same gradient, and
    its neighbours in the flat buffer nothing."""
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8

    rng = _rng(31, K, N)
    x = torch.from_numpy(_matrix(rng, 200, K)).to(dev).to(torch.bfloat16)
    dy = torch.from_numpy(_matrix(rng, 200, N)).to(dev).to(torch.bfloat16)
    W = torch.from_numpy(_matrix(rng, K, N)).to(dev).requires_grad_(True)
    linear_fp8(x, W).backward(dy)
    want, W.grad = W.grad.clone(), None
    for lead in (0, 3):
        flat = torch.full((lead + K * N + 5,), float("nan"), device=dev)
        W.main_grad = flat[lead:lead + K * N].view(K, N)
        linear_fp8(x, W).backward(dy)
        assert W.grad is None and torch.equal(W.main_grad, want)
        assert torch.isnan(flat[:lead]).all() and torch.isnan(flat[lead + K * N:]).all()


def test_gemm_workspace_elsewhere_is_refused(dev):
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8, quantize_fp8

    a = quantize_fp8(torch.ones((8, 4096), device=dev))
    b = quantize_fp8(torch.ones((64, 4096), device=dev))
    for ws in (torch.empty(1 << 16), torch.empty((256, 512), device=dev)[:, :256]):
        with pytest.raises(ValueError, match="workspace"):
            gemm_fp8(a, b, ws=ws)
    assert torch.equal(gemm_fp8(a, b, ws=torch.empty(4, device=dev)), gemm_fp8(a, b))


@pytest.mark.parametrize("wdtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("xdtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,K,N", [(1, 130, 5), (300, 257, 129), (128, 128, 128)])
def test_linear_is_its_parts(dev, M, K, N, xdtype, wdtype):
    """linear_fp8 quantises x and W in one launch: bit for bit what the operators give one by one."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8, linear_fp8, quantize_fp8_both

    rng = _rng(41, M, K, N)
    x = torch.from_numpy(_matrix(rng, M, K)).to(dev).to(getattr(torch, xdtype)).requires_grad_(True)
    W = torch.from_numpy(_matrix(rng, K, N)).to(dev).to(getattr(torch, wdtype)).requires_grad_(True)
    dy = torch.from_numpy(_matrix(rng, M, N)).to(dev).to(getattr(torch, xdtype))
    y = linear_fp8(x, W)
    y.backward(dy)
    qx, qxt = quantize_fp8_both(x.detach())
    wb, wf = quantize_fp8_both(W.detach(), group=128)
    qd, qdt = quantize_fp8_both(dy)
    assert torch.equal(y, gemm_fp8(qx, wf, x.dtype))
    assert torch.equal(x.grad, gemm_fp8(qd, wb, x.dtype))
    assert torch.equal(W.grad, gemm_fp8(qxt, qdt, W.dtype))


@pytest.mark.parametrize("M,N", [(1, 1), (5, 300), (300, 130), (4096, 4104)])
def test_gemm_without_a_sum_reads_nothing(dev, M, N):
    """K == 0 writes zeros whatever the operands' strides are, without reading them: their pointers may be null."""
    import torch
    from nlearn_amd import _lib
    from nlearn_amd.kernels.fp8 import Fp8Blocks, gemm_fp8

    for dt, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for lds in (0, 1, 4, 8):
            for ga, gb in ((1, 1), (1, 128), (128, 128)):
                out = torch.full((M, (N + 7) // 8 * 8), 7.0, dtype=dt, device=dev)
                _lib.call("nl_gemm_fp8", _lib.stream_of(out), M, N, 0, None, 128, None, lds, ga, None, 128, None, lds, gb,
                          out.data_ptr(), code, out.stride(0), None, 0)
                assert (out[:, :N] == 0).all() and (out[:, N:] == 7).all()
        # rows of eight scale bytes of which none belongs to the operand
        blocks = [Fp8Blocks(torch.empty((rows, 128), dtype=torch.float8_e4m3fn, device=dev)[:, :0],
                            torch.empty((rows, 8), dtype=torch.float8_e8m0fnu, device=dev)[:, :0], (rows, 0))
                  for rows in (M, N)]
        assert (gemm_fp8(*blocks, dt) == 0).all()


def test_linear_main_grad_of_another_shape_is_refused(dev):
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8

    x = torch.ones((8, 128), dtype=torch.bfloat16, device=dev)
    W = torch.ones((128, 40), device=dev, requires_grad=True)
    for buf in (torch.full((40, 128), 7.0, device=dev), torch.full((5120,), 7.0, device=dev), torch.full((128, 40), 7.0)):
        W.main_grad = buf
        with pytest.raises(ValueError, match="main_grad"):
            linear_fp8(x, W).sum().backward()
        assert (buf == 7).all()


def test_linear_keeps_its_operands_with_autograd(dev):
    """What the backward reads is freed by it though the loss lives on, passes through saved-tensor hooks,
    and is not kept by a checkpoint."""
    import torch
    from torch.utils.checkpoint import checkpoint
    from nlearn_amd.kernels.fp8 import linear_fp8

    rng = _rng(51)
    M, K, N = 4096, 512, 256
    x = torch.from_numpy(_matrix(rng, M, K)).to(dev).to(torch.bfloat16).requires_grad_(True)
    W = torch.from_numpy(_matrix(rng, K, N)).to(dev).requires_grad_(True)
    dy = torch.from_numpy(_matrix(rng, M, N)).to(dev).to(torch.bfloat16)
    linear_fp8(x, W).backward(dy)
    want = x.grad.clone(), W.grad.clone()
    kept = M * K + K * N  # bytes of X^T and W in 8 bits

    def grown(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(dev)
        out = call()
        return out, torch.cuda.memory_allocated(dev) - before

    x.grad = W.grad = None
    y, more = grown(lambda: linear_fp8(x, W))
    assert more >= M * N * 2 + kept
    def back():
        y.backward(dy, retain_graph=False)
        grads, x.grad, W.grad = (x.grad, W.grad), None, None
        return [torch.equal(g, w) for g, w in zip(grads, want)]
    same, less = grown(back)
    assert all(same) and less <= -kept  # y itself is still held

    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.numel() * t.element_size()) or t.cpu(),
                                                  lambda t: t.to(dev)):
        y = linear_fp8(x, W)
    assert any(n >= kept for n in packed)
    y.backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(W.grad, want[1])

    x.grad = W.grad = None
    y, more = grown(lambda: checkpoint(linear_fp8, x, W, use_reentrant=False))
    assert more < M * N * 2 + kept
    y.backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(W.grad, want[1])
    x.grad = W.grad = None
    W.main_grad = torch.full((K, N), float("nan"), device=dev)
    checkpoint(linear_fp8, x, W, use_reentrant=False).backward(dy)
    assert W.grad is None and torch.equal(W.main_grad, want[1])
    # nothing kept where nothing is summed
    e = torch.empty((0, K), dtype=torch.bfloat16, device=dev, requires_grad=True)
    linear_fp8(e, W).sum().backward()
    assert e.grad.shape == (0, K)


@pytest.mark.parametrize("ga,gb", [(1, 1), (1, 128), (128, 128)])
@pytest.mark.parametrize("M,N,K", [(4097, 4099, 300), (4095, 4352, 1100), (4096, 4608, 128), (130, 200, 640)])
def test_gemm_with_compact_scale_rows(dev, M, N, K, ga, gb):
    """Scale rows that are no whole dwords, on large tiles (several a workgroup) and small ones: against float64,
    and bit for bit what the same scales in padded rows give."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    results = []
    for padded in ((False, False), (True, True), (False, True)):
        rng = _rng(M, N, K, 61)
        a, a64 = _operand(rng, M, K, ga, dev, padded[0])
        b, b64 = _operand(rng, N, K, gb, dev, padded[1])
        assert (a.scale.stride(0) % 4 == 0) == padded[0] or a.scale.shape[0] == 1
        results.append([gemm_fp8(a, b, dt) for dt in (torch.float32, torch.bfloat16)])
    for out in results[0]:
        _check_product(out, a64, b64, K)
    for other in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], other))


@pytest.mark.parametrize("dtype,least,largest", [("float32", 3, 246), ("bfloat16", 0, 254)])
def test_gemm_scale_bytes_of_the_whole_range(dev, dtype, least, largest):
    """Every e4m3 value at scale bytes from end to end of the range that holds for a result's type, times values
    whose scale makes the products ordinary: single products, exact in fp32 and rounded once in bf16."""
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks, gemm_fp8

    table = orc.e4m3_table()
    each = np.array([b for b in range(256) if np.isfinite(table[b])], np.uint8)

    def operand(values, byte):
        q = np.zeros((len(values), 128), np.uint8)
        q[:, 77] = values
        s = np.full((len(values), 1), byte, np.uint8)
        return Fp8Blocks(torch.from_numpy(q).to(dev).view(torch.float8_e4m3fn),
                         torch.from_numpy(s).to(dev).view(torch.float8_e8m0fnu), (len(values), 128))

    few = np.array([0x01, 0x38, 0x7e, 0xb8], np.uint8)  # 2^-9, 1, 448, -1
    want = torch.from_numpy(table[each][:, None] * table[few][None]).to(dev, getattr(torch, dtype))
    for byte in sorted({least, least + 1, least + 5, 64, 127, 190, largest - 5, largest - 1, largest}):
        against = min(max(254 - byte, least), largest)
        f = 2.0 ** (byte + against - 254)  # 1 but where the ranges' ends are not alike
        a, b = operand(each, byte), operand(few, against)
        assert torch.equal(gemm_fp8(a, b, want.dtype), want * f), byte
        assert torch.equal(gemm_fp8(b, a, want.dtype), want.t() * f), byte
    # byte 255 is e8m0's NaN
    assert torch.isnan(gemm_fp8(operand(few, 255), operand(few, 127), want.dtype)).all()


def test_gemm_of_cancelling_products(dev):
    """Large products that cancel and a small one beside them: an fp32 result is the small one, a bf16 result is
    within the cut that the header states."""
    import torch
    from nlearn_amd.kernels.fp8 import Fp8Blocks, gemm_fp8

    rng = _rng(71)
    M, N, K = 40, 24, 512
    a, b = np.zeros((M, K)), np.zeros((N, K))
    at = np.stack([rng.permutation(K)[:3] for _ in range(M)])
    for m in range(M):
        a[m, at[m]] = 256.0, -256.0, 2.0 ** rng.integers(-6, 1)
        b[:, at[m]] = 1.0
    operands = []
    for x in (a, b):
        q, s = orc.e4m3_bytes(x), np.full((x.shape[0], K // 128), 127, np.uint8)
        operands.append((Fp8Blocks(torch.from_numpy(q).to(dev).view(torch.float8_e4m3fn),
                                   torch.from_numpy(s).to(dev).view(torch.float8_e8m0fnu), x.shape), _values(q, s, 1, K, dev)))
    (qa, a64), (qb, b64) = operands
    assert torch.equal(gemm_fp8(qa, qb, torch.float32).double(), a64[0] @ b64[0].t())
    _check_product(gemm_fp8(qa, qb, torch.bfloat16), a64, b64, K)
