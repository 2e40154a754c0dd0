"""top_logits and the distillation loss on logits of large finite values: masks of -1e4 to the type's
lowest beside ordinary logits and alone, and rows far from zero.

With e = (x - X) / T, X the row's maximum, u = 2^-24 and S = sum exp(e), the bounds are:
  S        4 roundings of an exponent (the rounded 1/T two, the difference, the product; a further one of
           each reference a partial sum moves to is part of them) cost 4 |e| u of a term, and the mean of
           |e| under the weights exp(e) / S is at most log V < 18; two roundings of each exp2, 132 of the
           sums: (72 + 4 + 132) u < 2^8 u = 2^-16.
  lse      2^-16, and u |lse| for its own rounding.
  loss     T^2 times: S_t 2^-16 for the student's sum (S_t = sum p), 2^-22 p |e| of each entry, and
           2^-21 sum p |gap| for p itself.
  dlogits  half a step of bf16 (2^-8 of the value); q is off by 2^-16 and, where exp(e) is above 2^-126,
           by 4 |e| u < 2^-15: 2^-14 of S_t q + p. An exp(e) below 2^-126 is flushed to 0: q = exp(e) / S,
           S >= 1, so 2^-126 T S_t / M of the gradient, and 1e-38 for a bf16 below its own normal range.
"""
import numpy as np
import pytest

from oracle import distill_fp8 as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
MASKS = [-1e4, -1e9, -1e10, -1e20, -1e30, -3.3895313892515355e38]  # the last: bf16's lowest
ROWS = [700, 9000, 50257, 120000]  # one wave, several, the model's, streamed


def _normal(rng, M, V):
    import torch

    return torch.from_numpy((rng.standard_normal((M, V)) * 2).astype(np.float32)).to(torch.bfloat16)


def _beside(rng, V):
    """Rows with masks over a tail, a head, a stretch within, and all but three logits."""
    x = _normal(rng, 4 * len(MASKS), V)
    for n, a in enumerate(MASKS):
        x[4 * n, V - V // 3:] = a
        x[4 * n + 1, :V // 2] = a
        x[4 * n + 2, V // 7:V // 2] = a
        keep = x[4 * n + 3, [0, V // 2, V - 1]].clone()
        x[4 * n + 3] = a
        x[4 * n + 3, [0, V // 2, V - 1]] = keep
    return x


def _entries(rng, x, k, T):
    """A teacher near the student's logits: its k largest and its logsumexp."""
    import torch

    t = x.double() + torch.from_numpy(rng.standard_normal(tuple(x.shape)))
    v, i = torch.topk(t, k, 1)
    return i.int(), v.float(), torch.logsumexp(t / T, 1).float()


def _distill(x, ids, v, lse, T, dev):
    """Losses by row and the gradient of their mean, from the C entry point."""
    import torch
    from nlearn_amd import _lib

    M, V = x.shape
    z, i, w, l = x.to(dev), ids.to(dev), v.to(dev), None if lse is None else lse.to(dev)
    loss, d = torch.empty(M, device=dev), torch.empty_like(z)
    _lib.call("nl_distill_fwd_bwd", _lib.stream_of(z), M, V, z.data_ptr(), V, ids.shape[1], i.data_ptr(), 0,
              w.data_ptr(), _lib.NL_DTYPE_F32, None if l is None else l.data_ptr(), T, loss.data_ptr(), None, 1.0 / M,
              d.data_ptr(), V)
    return loss.double().cpu().numpy(), d.double().cpu().numpy()


def _from_max(x):
    """x less the row's maximum, in float64: the loss and its gradient are the same, and no sum of a
    large value and a logarithm is formed."""
    x = x.double().numpy()
    with np.errstate(invalid="ignore"):
        return x - x.max(1, keepdims=True)


def _check_loss(got, x, ids, v, lse, T):
    z, i = _from_max(x), ids.numpy()
    want, _, mass, spread = orc.distill(z, i, v.double().numpy(), None if lse is None else lse.double().numpy(), T, 1.0)
    on = i >= 0
    with np.errstate(divide="ignore", invalid="ignore"):
        w = np.where(on, v.double().numpy() / T, -np.inf)
        p = np.exp(w - (orc.lse(w) if lse is None else lse.double().numpy())[:, None])
        p = np.where(w > -np.inf, p, 0)
    e = np.where(p > 0, np.abs(np.take_along_axis(z, np.where(on, i, 0), 1)) / T, 0)
    lim = T * T * (2.0 ** -16 * mass + 2.0 ** -22 * (p * e).sum(1) + 2.0 ** -21 * spread) + U * np.abs(want)
    assert (np.abs(got - want) <= lim).all(), (got, want, lim)


def _check_gradient(got, x, ids, v, lse, T):
    z, i = _from_max(x), ids.numpy()
    M = x.shape[0]
    _, d, mass, _ = orc.distill(z, i, v.double().numpy(), None if lse is None else lse.double().numpy(), T, 1.0 / M)
    entry = np.zeros(x.shape, bool)
    for m in range(M):
        entry[m, i[m][i[m] >= 0]] = True
    # S_t q + p <= |d| M / T, and 2 S_t more at the entries
    both = np.abs(d) + np.where(entry, 2 * mass[:, None], 0) * T / M
    bad = ~(np.abs(got - d) <= 1.01 * 2.0 ** -8 * np.abs(d) + 2.0 ** -14 * both + 2.0 ** -126 * mass[:, None] * T / M
            + 1e-38)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[0], got[bad][0], d[bad][0])


@pytest.mark.parametrize("T", [1.0, 2.0 ** -7, 1024.0])
@pytest.mark.parametrize("V", ROWS)
def test_top_logits_beside_masks(dev, V, T):
    import torch
    from nlearn_amd.kernels.distill import top_logits

    x = _beside(np.random.default_rng(V), V)
    values, ids, lse = top_logits(x.to(dev), 8, T)
    want = orc.top(x.double().numpy(), 8, T)
    np.testing.assert_array_equal(ids.cpu().numpy(), want[0])
    assert torch.equal(values.cpu(), x.gather(1, ids.cpu().long()))
    assert (np.abs(lse.double().cpu().numpy() - want[1]) <= 2.0 ** -16 + U * np.abs(want[1])).all()


@pytest.mark.parametrize("T", [1.0, 1024.0])
@pytest.mark.parametrize("V", ROWS)
def test_loss_and_gradient_beside_masks(dev, V, T):
    rng = np.random.default_rng(V + 1)
    x = _beside(rng, V)
    ids, v, lse = _entries(rng, x, 3, T)
    for l in (lse, None):
        loss, d = _distill(x, ids, v, l, T, dev)
        _check_loss(loss, x, ids, v, l, T)
        _check_gradient(d, x, ids, v, l, T)


def _far(rng, V):
    """Rows of one value (a mask that leaves nothing among them), and rows about a value far from zero."""
    import torch

    one = MASKS + [3e4, -1e6, 1e6, -1e7, 1e10, 1e30]
    about = [(1e3, 16.0), (-3e4, 512.0), (1e6, 2.0 ** 14), (-1e10, 2.0 ** 28)]  # some bf16 steps wide
    x = torch.empty((len(one) + len(about), V), dtype=torch.bfloat16)
    for m, a in enumerate(one):
        x[m] = a
    for m, (a, s) in enumerate(about):
        x[len(one) + m] = (a + s * torch.from_numpy(rng.standard_normal(V))).to(torch.bfloat16)
    return x


def _teacher(rng, M, V, k):
    """Entries of a teacher of its own: distinct ids, the largest logits among the row's and their sums."""
    import torch

    ids = np.stack([rng.permutation(V)[:k] for _ in range(M)]).astype(np.int32)
    v = rng.standard_normal((M, k))
    lse = orc.lse(v) + 0.5
    return torch.from_numpy(ids), torch.from_numpy(v.astype(np.float32)), torch.from_numpy(lse.astype(np.float32))


TEMPERATURES = [1.0, float(np.float32(1e-3)), 2.0 ** -7, 1024.0]


@pytest.mark.parametrize("T", TEMPERATURES)
@pytest.mark.parametrize("V", ROWS)
def test_gradient_far_from_zero(dev, V, T):
    rng = np.random.default_rng(V + 2)
    x = _far(rng, V)
    ids, v, lse = _teacher(rng, x.shape[0], V, 4)
    v = v * T  # p as at T = 1, whatever the temperature
    for l in (lse, None):
        _check_gradient(_distill(x, ids, v, l, T, dev)[1], x, ids, v, l, T)
    # the masks of a batch beside ordinary logits, at every temperature
    y = _beside(rng, V)
    ids, v, lse = _entries(rng, y, 3, T)
    _check_gradient(_distill(y, ids, v, lse, T, dev)[1], y, ids, v, lse, T)


@pytest.mark.parametrize("T", TEMPERATURES)
@pytest.mark.parametrize("V", ROWS)
def test_loss_far_from_zero(dev, V, T):
    import torch

    rng = np.random.default_rng(V + 3)
    x = _far(rng, V)
    ids, v, lse = _teacher(rng, x.shape[0], V, 4)
    v = v * T
    for l in (lse, None):
        _check_loss(_distill(x, ids, v, l, T, dev)[0], x, ids, v, l, T)
    y = _beside(rng, V)
    yi, yv, yl = _entries(rng, y, 3, T)
    for l in (yl, None):
        _check_loss(_distill(y, yi, yv, l, T, dev)[0], y, yi, yv, l, T)
    # a teacher far from zero too: the softmax of its entries is that of their distances
    far = torch.tensor(MASKS, dtype=torch.float64).repeat(3)[:x.shape[0], None].float()
    w = torch.where(torch.arange(4) < 3, far, far * 2)
    z = _normal(rng, x.shape[0], V)
    loss, d = _distill(z, ids, w, None, T, dev)
    shifted = (w.double() - far.double()).clamp(min=-1e38).float()
    _check_loss(loss, z, ids, shifted, None, T)
    _check_gradient(d, z, ids, shifted, None, T)


@pytest.mark.parametrize("T", TEMPERATURES)
@pytest.mark.parametrize("V", ROWS)
def test_lse_far_from_zero(dev, V, T):
    """To its own rounding: what is left of the logarithm beside a large X / T is a half step of fp32."""
    from nlearn_amd.kernels.distill import top_logits

    x = _far(np.random.default_rng(V + 4), V)
    lse = top_logits(x.to(dev), 4, T)[2]
    want = x.double().numpy().max(1) / T + orc.lse(_from_max(x) / T)
    with np.errstate(over="ignore"):
        want32 = want.astype(np.float32)
    got = lse.cpu().numpy()
    fine = np.isfinite(want32)
    np.testing.assert_array_equal(got[~fine], want32[~fine])  # X / T past fp32
    assert (np.abs(got[fine].astype(np.float64) - want[fine]) <= 2.0 ** -16 + U * np.abs(want[fine])).all()


@pytest.mark.parametrize("T", [1.0, 2.0 ** -7, 1024.0])
def test_teacher_far_from_zero(dev, T):
    """p = exp(v / T - lse) where both are large: their difference, and none of their products' roundings."""
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy, top_logits

    rng = np.random.default_rng(77)
    V, k = 700, 4
    far = [a for a in MASKS + [3e4, 1e6, 1e10, 1e20, 1e30] if abs(a / T) < 3e38]
    a = torch.tensor(far, dtype=torch.float64).to(torch.bfloat16)[:, None]
    v = a.float().expand(-1, k).contiguous()
    z = _normal(rng, len(far), V)
    ids = _teacher(rng, len(far), V, k)[0]
    lse = (a.double()[:, 0] / T).float()  # exact: T is a power of two
    loss, d = _distill(z, ids, v, lse, T, dev)
    ones, none = torch.zeros_like(v), torch.zeros_like(lse)  # every p is 1
    _check_loss(loss, z, ids, ones, none, T)
    _check_gradient(d, z, ids, ones, none, T)
    if T == 1.0:  # a teacher whose mask leaves nothing: its logsumexp rounds to the mask itself
        t = a[a[:, 0].abs().double() >= 1e9].expand(-1, V)
        values, ids, lse = top_logits(t.to(dev), k)
        y = z[:t.shape[0]].to(dev).requires_grad_(True)
        loss = distill_cross_entropy(y, ids, values, lse)
        loss.backward()
        assert torch.isfinite(loss) and torch.isfinite(y.grad).all()


@pytest.mark.parametrize("T", [1.0, 2.5])
@pytest.mark.parametrize("V", [90, 700, 9000, 60000, 120000])
def test_loss_by_row_of_padding_repeats_and_odd_values(dev, V, T):
    """Each row's loss within its own bound: padding, repeated ids, no weight, masks on either side."""
    rng = np.random.default_rng(V)
    x = _normal(rng, 12, V)
    ids, v, lse = _entries(rng, x, 9, T)
    ids[0, 4:] = -1
    ids[1] = -7
    ids[2] = -1
    x[2] = float("nan")                    # a student's row that no entry reads
    ids[3] = 5                             # one id, nine times
    ids[4, 1::2] = ids[4, 0].item()
    v[5, 3:] = float("-inf")
    v[6] = float("-inf")                   # entries without weight
    ids[7, 2:] = ids[7, :1]
    ids[7, 6:8] = -1
    x[8, 10:] = float("-inf")              # a masked vocabulary; the entries are inside
    ids[8] = _teacher(rng, 1, 10, 9)[0][0]
    x[9] = MASKS[-1]
    x[9, ids[9, 0].item()] = 0.0
    v[9, 1:] = float("-inf")
    x[10] = 3.0
    for l in (lse, None):
        loss, d = _distill(x, ids, v, l, T, dev)
        _check_loss(loss, x, ids, v, l, T)
        assert (loss[[1, 2, 6]] == 0).all() and (d[[1, 2, 6]] == 0).all()
