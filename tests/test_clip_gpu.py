"""The global norm of many tensors and clipping by it, on the GPU against float64.

Bounds, u = 2^-24: the squares of fp32 values are summed in fp64 (n roundings of 2^-53, below
2^-20 u for the sizes here) and the root is rounded to fp32 once: u of the norm. A clipped
value is (g / n) * m: the norm's u, a rounding each for the quotient and the product, then
half a step of its type (2^-8 for bf16): 3.01 u + half of the value; half a step of the
type's subnormals where it is below them.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _np(t):
    return t.detach().double().cpu().numpy()


def _make(dev, shapes, seed=0, scale=1.0):
    """Tensors of the given (shape, dtype, how): dense, padded rows, a transpose, a column, shifted off 16 bytes."""
    import torch

    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for shape, dtype, how in shapes:
        dt = getattr(torch, dtype)
        if how == "padded":
            base = torch.full((*shape[:-1], shape[-1] + 3), float("nan"), dtype=dt, device=dev)
            t = base[..., :shape[-1]]
        elif how == "transposed":
            t = torch.empty(shape[::-1], dtype=dt, device=dev).t()
        elif how == "column":
            t = torch.full((*shape, 5), float("nan"), dtype=dt, device=dev)[..., 2]
        else:
            n = math.prod(shape)
            off = 1 if how == "shifted" else 0
            t = torch.full((n + 8,), float("nan"), dtype=dt, device=dev)[off:off + n].view(shape)
        t.copy_(torch.randn(shape, generator=g, device=dev) * scale)
        out.append(t)
    return out


MIXED = [((1,), "float32", "dense"), ((7,), "bfloat16", "shifted"), ((300, 40), "float32", "padded"),
         ((41, 133), "bfloat16", "padded"), ((0, 5), "float32", "dense"), ((64, 50), "float32", "transposed"),
         ((2, 3, 77), "bfloat16", "padded"), ((1001,), "float32", "column"), ((5000, 3), "bfloat16", "padded"),
         ((123457,), "bfloat16", "shifted"), ((70001,), "float32", "shifted"), ((), "float32", "dense"),
         ((3, 40000), "float32", "padded"), ((9000, 1), "bfloat16", "column")]


def _want(tensors, most):
    n = math.sqrt(sum(float((_np(t) ** 2).sum()) for t in tensors))
    return n, [_np(t) * (1.0 if n < most else most / n) for t in tensors]


def _check(tensors, got, norm, most, want=None):
    import torch

    n, values = want or _want(tensors, most)
    assert abs(float(norm) - n) <= 1.001 * U * n
    assert len(got) == len(tensors)
    for t, o, w in zip(tensors, got, values):
        assert o.shape == t.shape and o.dtype is t.dtype and o.stride() == t.stride()
        half = 2.0 ** -8 if t.dtype is torch.bfloat16 else U
        tiny = 2.0 ** -134 if t.dtype is torch.bfloat16 else 2.0 ** -149
        bound = np.abs(w) * (half + 3.01 * U) + tiny if n >= most else 0.0
        assert (np.abs(_np(o) - w) <= bound).all(), (tuple(t.shape), t.dtype)


@pytest.mark.parametrize("over", [True, False])
def test_clip_of_unlike_tensors(dev, over):
    import torch
    from nlearn_amd.kernels.clip import clip_by_global_norm, global_norm

    tensors = _make(dev, MIXED)
    n = _want(tensors, 1.0)[0]
    most = n * (0.3 if over else 1.5)
    before = [t.clone() for t in tensors]
    out, norm = clip_by_global_norm(tensors, most)
    assert norm.shape == () and norm.dtype is torch.float32 and norm.device == tensors[0].device
    _check(tensors, out, norm, most)
    assert all(torch.equal(a, b) for a, b in zip(before, tensors))
    assert not {o.data_ptr() for o in out if o.numel()} & {t.data_ptr() for t in tensors}
    assert torch.equal(global_norm(tensors), norm)
    # the same every time, and over the gradients themselves; what lies between their rows stays
    again, norm2 = clip_by_global_norm(tensors, most)
    assert torch.equal(norm, norm2) and all(torch.equal(a, b) for a, b in zip(out, again))
    same, norm3 = clip_by_global_norm(tensors, most, inplace=True)
    assert torch.equal(norm, norm3) and all(a is b for a, b in zip(same, tensors))
    assert all(torch.equal(a, b) for a, b in zip(out, tensors))
    pad = tensors[2]._base[:, 40:]
    assert pad.numel() and torch.isnan(pad).all()


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 129, 700])
def test_clip_of_many_tensors(dev, n):
    """Around the number that a launch takes, and several of them."""
    from nlearn_amd.kernels.clip import clip_by_global_norm, global_norm

    rng = np.random.default_rng(n)
    tensors = _make(dev, [((int(rng.integers(1, 3000)),), "bfloat16" if i % 3 else "float32", "shifted")
                          for i in range(n)], seed=n)
    most = 0.5 * _want(tensors, 1.0)[0]
    want = _want(tensors, most)
    out, norm = clip_by_global_norm(tensors, most)
    _check(tensors, out, norm, most, want)
    assert float(global_norm(tensors)) == float(norm)
    same, norm = clip_by_global_norm(tensors, most, inplace=True)
    _check(tensors, same, norm, most, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [1, 8, 2047 * 4, 2048 * 8 + 1, (1 << 22) + 5, 40_000_003])
def test_clip_of_one_tensor(dev, size, dtype):
    """Ends of vectors and chunks, more chunks than workgroups."""
    from nlearn_amd.kernels.clip import clip_by_global_norm

    tensors = _make(dev, [((size,), dtype, "dense")])
    most = 0.7 * _want(tensors, 1.0)[0]
    _check(tensors, *clip_by_global_norm(tensors, most), most)


def test_norm_of_tiny_huge_and_not_finite_values(dev):
    import torch
    from nlearn_amd.kernels.clip import clip_by_global_norm, global_norm

    tiny = torch.full((1000,), 2.0 ** -100, device=dev)
    assert abs(float(global_norm([tiny])) - 2.0 ** -100 * math.sqrt(1000)) <= 1.001 * U * 2.0 ** -95
    huge = torch.full((1000,), 2.0 ** 100, device=dev, dtype=torch.bfloat16)
    _check([huge], *clip_by_global_norm([huge], 1.0), 1.0)
    zero = torch.zeros(50, device=dev)
    out, norm = clip_by_global_norm([zero], 1.0)
    assert float(norm) == 0 and (out[0] == 0).all()
    # an infinite norm makes finite values 0, a NaN all of them NaN
    a, b = torch.ones(100, device=dev), torch.ones(100, device=dev, dtype=torch.bfloat16)
    a[7] = float("inf")
    (x, y), norm = clip_by_global_norm([a, b], 1.0)
    assert math.isinf(float(norm)) and torch.isnan(x[7]) and (y == 0).all() and int((x == 0).sum()) == 99
    full = torch.full((10,), 3.4e38, device=dev)
    assert math.isinf(float(clip_by_global_norm([full], 1.0)[1]))  # finite values, a norm past fp32
    b[3] = float("nan")
    (x, y), norm = clip_by_global_norm([a, b], 1.0)
    assert math.isnan(float(norm)) and torch.isnan(x).all() and torch.isnan(y).all()
    # the largest norm that is let through is below max_norm; one that meets it is divided by itself
    c = torch.tensor([3.0, 4.0], device=dev)
    assert torch.equal(clip_by_global_norm([c], 5.0)[0][0], (c / 5) * 5)
    assert torch.equal(clip_by_global_norm([c], 5.000001)[0][0], c)


def test_norm_of_no_elements(dev):
    import torch
    from nlearn_amd.kernels.clip import clip_by_global_norm, global_norm

    e = torch.empty((0, 4), device=dev)
    assert float(global_norm([e, e])) == 0
    out, norm = clip_by_global_norm([e], 1.0, inplace=True)
    assert out[0] is e and float(norm) == 0


def test_clip_on_a_captured_graph(dev):
    """Replayed over new gradients, with eager calls on another stream between the replays."""
    import torch
    from nlearn_amd.kernels.clip import clip_by_global_norm

    tensors = _make(dev, MIXED)
    source = [_make(dev, MIXED, seed=s, scale=10.0 ** -s) for s in range(4)]
    clip_by_global_norm(tensors, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, norm = clip_by_global_norm(tensors, 30.0)
    side = torch.cuda.Stream()
    for s in source + source[:2]:
        for t, v in zip(tensors, s):
            t.copy_(v)
        graph.replay()
        with torch.cuda.stream(side):
            want, wnorm = clip_by_global_norm(s, 30.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, wnorm) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_adamw_clips_gradients_of_their_own(dev):
    """AdamW without gradient buffers, against the one that has them and clips on the way."""
    import torch
    from nlearn_amd.train import AdamW

    g = torch.Generator(device=dev).manual_seed(3)
    shapes = [(40, 56), (333,), (512, 128)]
    make = lambda: [torch.randn(s, generator=g, device=dev) for s in shapes]  # noqa: E731
    start = make()
    steps = [[t * f for t in make()] for f in (1.0, 1e-3, 5.0)]
    params, states = [], []
    for buffers in (False, True):
        leaves = {str(i): t.clone().requires_grad_(True) for i, t in enumerate(start)}
        opt = AdamW(lambda c: 1e-2, clip_norm=20.0, grad_buffers=buffers)
        state = opt.init(leaves)
        for grads in steps:
            for p, t in zip(leaves.values(), grads):
                if buffers:
                    p.main_grad.copy_(t)
                else:
                    # rows that share memory are clipped as what they stand for
                    p.grad = t.clone() if t.dim() == 1 else t.clone().t().contiguous().t()
            opt.update(leaves, state)
        params.append(list(leaves.values()))
        states.append(state)
    assert abs(float(states[0]["gnorm"]) - float(states[1]["gnorm"])) <= 1e-5 * float(states[1]["gnorm"])
    # m and v scale with the clipped gradient: the two norms differ by the fp32 summation (below 100 u of 67000
    # squares in 1024 partial sums of 66 terms), the updates' own roundings are the same
    for m in ("mu", "nu"):
        for a, b in zip(states[0][m], states[1][m]):
            assert (a - b).abs().max() <= 300 * U * b.abs().max()
    for a, b in zip(*params):
        # an update moves by lr times a ratio of the two, of size 1 at most some units
        assert (a - b).abs().max() <= 1e-2 * 3 * 2000 * U + 4 * U * b.abs().max()
