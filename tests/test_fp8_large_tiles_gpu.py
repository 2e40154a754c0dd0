"""The epilogues of 8-bit products on 256 x 256 tiles, which heavy ones take only behind a long K: a result
in 8 bits past K = 1024 (2048 with a residual), u kept past 2048, a residual alone past 512. Every shape here
has 256 of these tiles and more, ragged ones among them; bounds and oracles are those of test_fp8_fused_gpu.py.
"""
import numpy as np
import pytest
import test_fp8_fused_gpu as fused
from test_fp8_fused_gpu import HALF, _finish, _np, _rng, _sums

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ["bfloat16", "float32", "float8_e4m3fn"])
@pytest.mark.parametrize("M,N,K", [(4200, 4100, 1100), (4097, 4099, 2100)])
def test_product(dev, M, N, K, out):
    fused.test_product_with_epilogue(dev, M, N, K, out)


@pytest.mark.parametrize("M,N,K", [(4200, 4104, 700), (4097, 4101, 2100)])
def test_product_into_rows_of_the_callers(dev, M, N, K):
    fused.test_product_into_rows_of_the_callers(dev, M, N, K)


@pytest.mark.parametrize("M,N,K", [(4200, 4100, 1100), (4097, 4099, 2100)])
def test_scale_rows_of_any_length(dev, M, N, K):
    fused.test_scale_rows_of_any_length(dev, M, N, K)


@pytest.mark.parametrize("M,N,K", [(4200, 4100, 1100), (4097, 4104, 2100)])
def test_residual_of_zeros(dev, M, N, K):
    """The plain product bit for bit, and in 8 bits the same bytes with the residual as without."""
    import torch
    from nlearn_amd.kernels.fp8 import gemm_fp8

    rng = _rng(M, N, K, 2)
    a, _ = fused._blocks(rng, M, K, 1, dev)
    b, _ = fused._blocks(rng, N, K, 128, dev)
    for dt in (torch.bfloat16, torch.float32):
        zero = torch.zeros((M, N), dtype=dt, device=dev)
        assert torch.equal(gemm_fp8(a, b, out_dtype=dt, residual=zero), gemm_fp8(a, b, out_dtype=dt))
    bare, with_res = (gemm_fp8(a, b, out_dtype=torch.float8_e4m3fn, residual=r)
                      for r in (None, torch.zeros((M, N), dtype=torch.bfloat16, device=dev)))
    assert torch.equal(bare.q.view(torch.uint8), with_res.q.view(torch.uint8))
    assert torch.equal(bare.scale.contiguous().view(torch.uint8), with_res.scale.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", [(4200, 4100, 2100), (4097, 4352, 2200)])
def test_layer_with_u_kept(dev, M, N, K, dtype):
    """u as the layer without an activation gives it, y from it, and dx from the u that was kept."""
    import torch
    from nlearn_amd import _lib
    from nlearn_amd.kernels.fp8 import ACTIVATIONS, Fp8Blocks, fp8_weight, gemm_fp8, linear_fp8, quantize_fp8

    dt = getattr(torch, dtype)
    rng = _rng(M, N, K, 6)
    make = lambda r, c, s: torch.from_numpy((s * rng.standard_normal((r, c))).astype(np.float32)).to(dev)  # noqa: E731
    x, W, bias = make(M, K, 1.0).to(dt).requires_grad_(True), make(K, N, K ** -0.5), make(1, N, 1.0)[0]
    dy, res = make(M, N, 1.0).to(dt), make(M, N, 3.0).to(dt)
    f = fp8_weight(W)
    z, e = _sums(_np(quantize_fp8(x.detach()).dequantize()), _np(f.fwd.dequantize()), dtype == "float32")
    z, e = _finish(z, e, _np(bias), None, None)
    with torch.no_grad():
        u = linear_fp8(x, W, bias=bias)
    assert (np.abs(_np(u) - z) <= e * (1 + HALF[dtype]) + HALF[dtype] * np.abs(z)).all()
    code = _lib.NL_DTYPE_F32 if dt is torch.float32 else _lib.NL_DTYPE_BF16
    for name in ("gelu", "silu"):
        q = Fp8Blocks.empty(M, N, 1, dev)
        _lib.call_on(u, "nl_quantize_fp8_dact", M, N, dy.data_ptr(), code, N, u.data_ptr(), u.stride(0), ACTIVATIONS[name],
                     *q._abi(), None, 0, None, 0, None, 0, None, 0)
        dx = gemm_fp8(q, f.bwd, dt)
        for r in (None, res):
            want, bound = _finish(_np(u), 0 * z, None, name, None if r is None else _np(r))
            for weight in (W, f):
                y = linear_fp8(x, weight, bias=bias, activation=name, residual=r)
                assert (np.abs(_np(y) - want) <= bound * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + 2.0 ** -133).all()
                assert torch.equal(torch.autograd.grad(y, x, dy)[0], dx)
                with torch.no_grad():  # and with u rounded, but not kept
                    assert torch.equal(linear_fp8(x, weight, bias=bias, activation=name, residual=r), y)
