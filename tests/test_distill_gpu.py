"""top_logits and distill_cross_entropy on the GPU, against float64.

Picked logits and ids are compared exactly. Bounds of the computed numbers, with
n = additions of one thread and of the merges (at most 128 here):
  lse      n + 4 roundings of 2^-24 of a sum of positive terms (its log moves by as
           much), 2^-24 of the largest |x| / T from log2(e)/T held in 32 bits, and
           half a step of the result.
  loss     T^2 S times the error of the student's lse, and 2^-21 of sum p |gap| for p.
  dlogits  half a step of bf16 (2^-8 of the value), and (n + 80) 2^-24 <= 2^-16 of
           S q + p for the exponent's argument (below 64) and the sum.
"""
import numpy as np
import pytest

from oracle import distill_fp8 as orc

pytestmark = pytest.mark.gpu

N_ADD = 128


def _logits(rng, M, V, std=2.0):
    import torch

    return torch.from_numpy((rng.standard_normal((M, V)) * std).astype(np.float32)).to(torch.bfloat16)


def _lse_err(x, T):
    return (N_ADD + 4) * 2.0 ** -24 + 2.0 ** -23 * np.abs(np.where(np.isfinite(x), x, 0)).max(1) / T


def _check_top(x, k, T, dev, view=None):
    import torch
    from nlearn_amd.kernels.distill import top_logits

    t = x.to(dev) if view is None else view
    v, i, l = top_logits(t, k, T)
    assert v.dtype == torch.bfloat16 and i.dtype == torch.int32 and l.dtype == torch.float32
    x64 = x.double().numpy()
    ids, lse = orc.top(x64, k, T)
    np.testing.assert_array_equal(i.cpu().numpy(), ids)
    bits = lambda a: a.contiguous().view(torch.int16).cpu().numpy()  # noqa: E731
    np.testing.assert_array_equal(bits(v), np.take_along_axis(bits(x), ids, 1))
    l = l.double().cpu().numpy()
    fine = np.isfinite(lse)
    np.testing.assert_array_equal(np.isnan(l), np.isnan(lse))
    np.testing.assert_array_equal(l[~fine & ~np.isnan(lse)], lse[~fine & ~np.isnan(lse)])
    lim = _lse_err(x64, T) + 2.0 ** -24 * np.abs(np.where(fine, lse, 0))
    assert (np.abs(l[fine] - lse[fine]) <= lim[fine]).all()


TOP = [(1, 1, 1), (3, 2, 2), (5, 64, 64), (7, 65, 1), (9, 500, 100), (4, 519, 256), (4, 530, 200), (6, 2000, 256),
       (6, 4097, 33), (5, 8200, 64), (3, 20011, 7), (3, 33000, 128), (8, 50257, 64), (2, 53247, 256), (2, 53260, 64),
       (2, 70001, 64), (2, 106503, 200), (2, 106520, 64), (1, 131072, 256), (1, 300001, 50)]


@pytest.mark.parametrize("M,V,k", TOP)
def test_top_against_float64(dev, M, V, k):
    rng = np.random.default_rng([M, V, k])
    _check_top(_logits(rng, M, V), k, 1.0, dev)
    _check_top(_logits(rng, M, V, 8.0), min(k, 3), 2.5, dev)


@pytest.mark.parametrize("V", [100, 700, 3000, 9000, 60000, 120000])
def test_top_ties_and_odd_values(dev, V):
    """Rows of one value, of few values, of -inf but for some (a mask), zeros of both signs, NaN, infinity."""
    import torch

    rng = np.random.default_rng(V)
    x = _logits(rng, 14, V)
    x[0] = 1.5
    x[1] = torch.from_numpy(rng.integers(0, 3, V).astype(np.float32)).to(torch.bfloat16)
    x[2] = float("-inf")
    x[2, rng.integers(0, V, 5)] = 2.0
    x[3] = float("-inf")
    x[4] = torch.from_numpy(np.where(rng.random(V) < 0.5, 0.0, -0.0).astype(np.float32)).to(torch.bfloat16)
    x[5] = -1.0
    x[5, V // 2:] = -0.0
    x[6, V - 1] = float("nan")
    x[7] = float("nan")
    x[8, 3], x[8, 5] = float("inf"), float("nan")
    x[9, 0] = float("inf")
    x[10] = torch.finfo(torch.bfloat16).min
    x[11] = -x[11].abs()
    x[12, :] = torch.sort(x[12].float()).values.to(torch.bfloat16)                    # ascending
    x[13] = torch.tensor(-float("nan"), dtype=torch.float32).to(torch.bfloat16)
    x[13, 1::2] = 1.0
    for k in (1, 5, 60):
        _check_top(x, k, 1.0, dev)


@pytest.mark.parametrize("V,stride,shift", [(50257, 50264, 0), (1000, 1003, 1), (501, 512, 5), (60001, 60007, 3)])
def test_top_strides_shape_and_repeat(dev, V, stride, shift):
    import torch
    from nlearn_amd.kernels.distill import top_logits

    rng = np.random.default_rng(V)
    x = _logits(rng, 6, V)
    buf = torch.full((6 * stride + shift,), float("inf"), dtype=torch.bfloat16, device=dev)
    t = torch.as_strided(buf, (6, V), (stride, 1), shift)
    t.copy_(x.to(dev))
    _check_top(x, 17, 1.0, dev, view=t)
    a, b = top_logits(t, 17), top_logits(t, 17)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    v, i, l = top_logits(x.to(dev).reshape(2, 3, V), 4)
    assert v.shape == i.shape == (2, 3, 4) and l.shape == (2, 3)
    # rows that share memory
    _check_top(x[:1].expand(3, V).contiguous(), 4, 1.0, dev, view=t[:1].expand(3, V))
    empty = top_logits(torch.empty((0, V), dtype=torch.bfloat16, device=dev), 3)
    assert empty[0].shape == (0, 3) and empty[2].shape == (0,)


def _entries(rng, x, k, T, vdtype):
    """A teacher near the student: ids, values and lse of its k largest logits."""
    import torch

    t = x.double() + torch.from_numpy(rng.standard_normal(tuple(x.shape)))
    v, i = torch.topk(t, k, 1)
    lse = torch.logsumexp(t / T, 1)
    return i.to(torch.int32), v.to(getattr(torch, vdtype)), lse.float()


def _check_distill(x, ids, values, lse, T, dev, view=None, inplace=False, g=1.0, ids64=False):
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy

    M, V = x.shape
    z = (x.to(dev) if view is None else view).detach().requires_grad_(True)
    i = ids.to(dev).long() if ids64 else ids.to(dev)
    # a view of a leaf, so that `inplace` may write over it
    loss = distill_cross_entropy(z.view(M, V) if view is None else z, i, values.to(dev),
                                 None if lse is None else lse.to(dev), T, inplace)
    (loss * g).backward()
    loss = loss.detach()
    x64 = x.double().numpy()
    ref, d, mass, spread = orc.distill(x64, ids.numpy(), values.double().numpy(),
                                       None if lse is None else lse.double().numpy(), T, g / M)
    lim = T * T * (mass * _lse_err(x64, T) + 2.0 ** -21 * spread)
    if np.isnan(ref).any():
        assert torch.isnan(loss)
    elif np.isinf(ref).any():
        assert torch.isinf(loss)
    else:
        assert abs(float(loss) - ref.mean()) <= lim.mean() + 2.0 ** -20 * np.abs(ref).mean(), (float(loss), ref.mean())
    got = z.grad.double().cpu().numpy()
    nan = np.isnan(d)
    np.testing.assert_array_equal(np.isnan(got), nan)
    p = np.zeros((M, V))
    for m in range(M):
        on = (ids[m] >= 0) & (ids[m] < V)
        np.add.at(p[m], ids[m][on].numpy(), 1.0)
    # |S q| + p <= |d| / (scale T) + 2 mass at the entries, |d| elsewhere
    fp32 = 2.0 ** -16 * (np.abs(d) + 2 * np.where(p > 0, mass[:, None], 0) * abs(g) * T / M)
    steps = 2 if g != 1.0 else 1  # another cotangent scales the rounded gradient: one more rounding
    err = np.abs(got - d)
    bad = ~nan & (err > steps * 1.01 * 2.0 ** -8 * np.abs(d) + steps * fp32 + 1e-38)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[0], err[bad][0], d[bad][0])
    return z


DISTILL = [(1, 1, 1), (2, 3, 3), (7, 64, 5), (5, 65, 65), (9, 500, 100), (4, 519, 256), (6, 1000, 16), (6, 4097, 33),
           (5, 8200, 64), (3, 20011, 7), (3, 33000, 128), (4, 50257, 64), (2, 53260, 64), (2, 106520, 64),
           (1, 131072, 256)]


@pytest.mark.parametrize("T", [1.0, 2.5])
@pytest.mark.parametrize("M,V,k", DISTILL)
def test_distill_against_float64(dev, M, V, k, T):
    rng = np.random.default_rng([M, V, k])
    x = _logits(rng, M, V)
    for vdtype in ("float32", "bfloat16"):
        ids, v, lse = _entries(rng, x, k, T, vdtype)
        _check_distill(x, ids, v, lse, T, dev)
        _check_distill(x, ids, v, None, T, dev, ids64=True)
    _check_distill(x, ids, v, lse, T, dev, inplace=True, g=-0.37)


@pytest.mark.parametrize("V", [90, 700, 9000, 60000, 120000])
def test_distill_padding_repeats_and_odd_values(dev, V):
    """Padding, rows without entries or weight (their student's NaN has no part), ids given many times, -inf on
    either side."""
    import torch

    rng = np.random.default_rng(V)
    M, k = 12, 9
    x = _logits(rng, M, V)
    ids, v, lse = _entries(rng, x, k, 1.0, "float32")
    ids[0, 4:] = -1
    ids[1] = -7
    ids[2] = -1
    x[2] = float("nan")
    ids[3] = 5                            # one id, nine times
    ids[4, 1::2] = ids[4, 0]
    v[5, 3:] = float("-inf")
    v[6] = float("-inf")                  # entries without weight
    ids[7, :] = torch.tensor([0, V - 1, 0, V - 1, 1, V - 2, -1, -1, 0])
    x[8, 10:] = float("-inf")             # a masked vocabulary; the entries are inside
    ids[8] = torch.arange(9)
    x[9] = torch.finfo(torch.bfloat16).min
    x[9, ids[9, 0].item()] = 0.0
    v[9, 1:] = float("-inf")
    x[10] = 3.0
    for l in (lse, None):
        for inplace in (False, True):
            _check_distill(x, ids, v, l, 1.0, dev, inplace=inplace)


@pytest.mark.parametrize("V", [300, 9000, 60000, 120000])
def test_distill_infinite_and_nan_rows(dev, V):
    """A NaN or an id past the vocabulary makes its own row NaN, an entry at a student's -inf the loss infinite."""
    import torch

    rng = np.random.default_rng(V + 1)
    x = _logits(rng, 4, V)
    ids, v, lse = _entries(rng, x, 6, 1.0, "float32")
    for change in ("nan logits", "inf logits", "nan value", "far id", "masked", "all masked"):
        y, i, w = x.clone(), ids.clone(), v.clone()
        if change == "nan logits":
            y[1, 7] = float("nan")
        elif change == "inf logits":
            y[1, V - 1] = float("inf")
            i[1, 0] = V // 3
        elif change == "nan value":
            w[1, 2] = float("nan")
        elif change == "far id":
            i[1, 2] = V
        elif change == "masked":
            y[1, i[1, 3].item()] = float("-inf")
        else:
            y[1] = float("-inf")
        for l in (lse, None):
            _check_distill(y, i, w, l, 1.0, dev)


@pytest.mark.parametrize("V,stride,shift", [(50257, 50264, 0), (1000, 1003, 1), (60001, 60007, 3)])
def test_distill_strides_leave_the_padding(dev, V, stride, shift):
    import torch

    rng = np.random.default_rng(V)
    M = 5
    x = _logits(rng, M, V)
    ids, v, lse = _entries(rng, x, 8, 2.0, "bfloat16")
    for inplace in (False, True):
        buf = torch.full((M * stride + shift,), 7.0, dtype=torch.bfloat16, device=dev)
        t = torch.as_strided(buf, (M, V), (stride, 1), shift)
        t.copy_(x.to(dev))
        z = _check_distill(x, ids, v, lse, 2.0, dev, view=t, inplace=inplace)
        assert inplace == (not torch.equal(t, x.to(dev)))
        if inplace:
            assert torch.equal(t, z.grad)
        pad = torch.ones_like(buf, dtype=torch.bool)
        torch.as_strided(pad, (M, V), (stride, 1), shift).fill_(False)
        assert (buf[pad] == 7).all()


def test_distill_to_another_phase(dev):
    """The C entry point with rows of the gradient at other offsets than the logits'."""
    import torch
    from nlearn_amd import _lib

    rng = np.random.default_rng(3)
    M, V, k, T = 4, 3001, 6, 2.0
    x = _logits(rng, M, V)
    ids, v, lse = _entries(rng, x, k, T, "float32")
    z, i, w, l = x.to(dev), ids.to(dev), v.to(dev), lse.to(dev)
    d = torch.full((M * (V + 2) + 1,), 7.0, dtype=torch.bfloat16, device=dev)
    loss = torch.empty(M, device=dev)
    _lib.call("nl_distill_fwd_bwd", _lib.stream_of(z), M, V, z.data_ptr(), V, k, i.data_ptr(), 0, w.data_ptr(),
              _lib.NL_DTYPE_F32, l.data_ptr(), T, loss.data_ptr(), None, 0.25, d.data_ptr() + 2, V + 2)
    got = torch.as_strided(d, (M, V), (V + 2, 1), 1)
    want = torch.empty((M, V), dtype=torch.bfloat16, device=dev)
    loss2 = torch.empty(M, device=dev)
    _lib.call("nl_distill_fwd_bwd", _lib.stream_of(z), M, V, z.data_ptr(), V, k, i.data_ptr(), 0, w.data_ptr(),
              _lib.NL_DTYPE_F32, l.data_ptr(), T, loss2.data_ptr(), None, 0.25, want.data_ptr(), V)
    assert torch.equal(got, want) and torch.equal(loss, loss2)
    assert d[0] == 7 and (torch.as_strided(d, (M, 2), (V + 2, 1), V + 1) == 7).all()


def test_distill_gradient_against_differences(dev):
    """Central differences of the loss over single logits (steps that bf16 holds exactly)."""
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy

    rng = np.random.default_rng(17)
    M, V, k, T = 2, 40, 5, 2.0
    x = torch.from_numpy(rng.integers(-8, 9, (M, V)).astype(np.float32) / 4).to(torch.bfloat16).to(dev)
    ids, v, lse = (t.to(dev) for t in _entries(rng, x.cpu(), k, T, "float32"))
    z = x.clone().requires_grad_(True)
    distill_cross_entropy(z, ids, v, lse, T).backward()
    h = 0.25
    for m, c in ((0, int(ids[0, 0])), (0, 11), (1, int(ids[1, 2])), (1, 39)):
        hi, lo = x.clone(), x.clone()
        hi[m, c] += h
        lo[m, c] -= h
        diff = (distill_cross_entropy(hi, ids, v, lse, T) - distill_cross_entropy(lo, ids, v, lse, T)) / (2 * h)
        # third derivative of T^2 log-sum-exp(z / T) is at most S / (6 sqrt 3) / T below S <= 1: h^2 / 6 of it;
        # the loss itself, about 1, to 2^-20
        assert abs(float(diff) - float(z.grad[m, c])) <= h * h / 6 * 0.1 / T + 2 * 2.0 ** -20 / h + 2.0 ** -8 * 0.5


def test_hard_target_entry_equals_cross_entropy(dev):
    """One entry of probability one is the softmax cross-entropy."""
    import torch
    from nlearn_amd.kernels.cross_entropy import cross_entropy
    from nlearn_amd.kernels.distill import distill_cross_entropy

    rng = np.random.default_rng(8)
    x = _logits(rng, 33, 5000).to(dev)
    t = torch.from_numpy(rng.integers(0, 5000, 33)).to(dev)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    la = cross_entropy(a, t)
    lb = distill_cross_entropy(b, t[:, None], torch.zeros((33, 1), device=dev), torch.zeros(33, device=dev))
    la.backward()
    lb.backward()
    assert abs(la.item() - lb.item()) <= 1e-5 * la.item()
    assert (a.grad.float() - b.grad.float()).abs().max() <= 2.0 ** -7 / 33


def test_distill_without_gradient_and_called_twice(dev):
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy

    rng = np.random.default_rng(4)
    x = _logits(rng, 6, 1000)
    ids, v, lse = (t.to(dev) for t in _entries(rng, x, 8, 1.0, "float32"))
    z = x.to(dev)
    plain = distill_cross_entropy(z, ids, v, lse)
    assert not plain.requires_grad and torch.equal(z, x.to(dev))
    zg = z.clone().requires_grad_(True)
    loss = distill_cross_entropy(zg, ids, v, lse)
    assert torch.equal(loss.detach(), plain)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        loss.backward()


def test_distill_in_a_graph(dev):
    """Teacher's pick and student's loss captured together and replayed on new logits."""
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy, top_logits

    rng = np.random.default_rng(6)
    M, V, k = 40, 5003, 12
    sets = [(_logits(rng, M, V).to(dev), _logits(rng, M, V).to(dev)) for _ in range(3)]

    def step(s, t):
        v, i, l = top_logits(t, k, 2.0)
        z = s.detach().requires_grad_(True)
        loss = distill_cross_entropy(z, i, v, l, 2.0)
        return loss.detach(), *torch.autograd.grad(loss, z)

    want = [[o.clone() for o in step(*p)] for p in sets]
    s, t = sets[0][0].clone(), sets[0][1].clone()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s, t)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(s, t)
    for _ in range(2):
        for (a, b), ref in zip(sets, want):
            s.copy_(a)
            t.copy_(b)
            g.replay()
            step(*sets[1])
            torch.cuda.synchronize()
            assert all(torch.equal(o, r) for o, r in zip(out, ref))
