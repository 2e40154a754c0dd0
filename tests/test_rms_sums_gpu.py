"""The sum of squares of the RMS norm where a long chain of additions loses the most.

Each thread's first value is 1 and the squares of the others lie below half a step of 1 (u = 2^-24): added one
by one to the first square every one of them is lost. A thread's 8 squares of a vector are added by pairs (the
product that a fused multiply-add takes up, that, and two sums: 4 roundings), then its vectors one to the other, so that
with a wave's exchanges and one addition a wave

    n = 4 + (vectors - 1) + exchanges + waves

roundings stand between a square and the row's sum, and the root halves what they lose: n / 2 u. The division by
the length and the addition of eps add half a unit each, the hardware's root 2, the product with it 1.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5


# columns, threads of a row, vectors of a thread, a wave's exchanges, waves that are added up
WIDTHS = [(100, 16, 1, 4, 0), (512, 64, 1, 6, 0), (1000, 64, 2, 6, 0), (2048, 64, 4, 6, 0), (4096, 256, 2, 6, 4),
          (8192, 256, 4, 6, 4), (16384, 512, 4, 6, 8)]


@pytest.mark.parametrize("cols,threads,vectors,exchanges,waves", WIDTHS)
def test_squares_beside_a_larger_one(dev, cols, threads, vectors, exchanges, waves):
    import torch
    from nlearn_amd.kernels.fused import add_rms_norm, rms_norm

    x = np.full((3, cols), np.sqrt(0.99 * U), np.float32)
    x[:, :threads * 8:8] = 1
    x[1] *= 2.0 ** 40
    x[2] *= 2.0 ** 65  # squares past fp32: summed again, scaled
    s = x.astype(np.float64)
    want = s / np.sqrt((s * s).mean(1, keepdims=True) + EPS)
    n = 4 + (vectors - 1) + exchanges + waves
    t, gamma = torch.from_numpy(x).to(dev), torch.ones(cols, device=dev)
    for y in (rms_norm(t, gamma, EPS), add_rms_norm(t, torch.zeros_like(t), gamma, EPS)[0]):
        off = np.abs(y.double().cpu().numpy() - want) / (U * np.abs(want))
        assert off.max() <= n / 2 + 4.001, (cols, off.max(1))


@pytest.mark.parametrize("cols,threads,vectors,exchanges,waves", WIDTHS)
def test_mean_of_the_backward(dev, cols, threads, vectors, exchanges, waves):
    """dx = dy - mean(dy) of rows of ones: the same n roundings of the sum, one each of the division, of the product
    with 1 and (of dx) of the difference."""
    import torch
    from nlearn_amd import _lib

    dy = np.full((3, cols), 0.99 * U, np.float32)
    dy[:, :threads * 8:8] = 1
    dy[1] *= -3
    d = torch.from_numpy(dy).to(dev)
    one, rstd, gamma = torch.ones_like(d), torch.ones(3, device=dev), torch.ones(cols, device=dev)
    dx = torch.empty_like(d)
    _lib.call_on(d, "nl_rms_norm_bwd", 3, cols, 0, d.data_ptr(), cols, one.data_ptr(), cols, rstd.data_ptr(),
                 gamma.data_ptr(), None, 0, dx.data_ptr(), cols, None, 0, None, 0)
    mean = dy.astype(np.float64).mean(1, keepdims=True)
    want = dy - mean
    n = 4 + (vectors - 1) + exchanges + waves
    off = np.abs(dx.double().cpu().numpy() - want) / (U * ((n + 2) * np.abs(mean) + np.abs(want)))
    assert off.max() <= 1.001, (cols, off.max(1))
