"""Norms, 8-bit products with their epilogues and clipping together, as a block uses them: a frozen
block in 8 bits, a training step, on two streams and in a captured graph, under hooks and checkpoints."""
import numpy as np
import pytest

from test_fp8_fused_gpu import HALF, _act, _check_8_bits, _finish, _np, _sums
from test_rms_gpu import _check_8_bits as _check_norm_8_bits
from test_rms_gpu import _norm64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _randn(g, *shape, dtype=None, scale=1.0):
    import torch

    t = torch.randn(shape, generator=g, device=g.device) * scale
    return t if dtype is None else t.to(dtype)


@pytest.mark.parametrize("tokens", [1, 7, 300, 4096])
def test_frozen_block_in_8_bits(dev, tokens):
    """norm -> product with gelu, to 8 bits -> product with the residual: each stage against float64 on what the
    stage before it wrote (the model's 512 and 2048, an odd width between them)."""
    import torch
    from nlearn_amd.kernels.fp8 import add_rms_norm_fp8, fp8_weight, gemm_fp8

    g = torch.Generator(device=dev).manual_seed(tokens)
    d, f = (512, 2048) if tokens != 7 else (200, 333)
    x, r = _randn(g, tokens, d, dtype=torch.bfloat16), _randn(g, tokens, d, dtype=torch.bfloat16)
    gamma = 1 + 0.1 * _randn(g, d)
    W1, W2 = fp8_weight(_randn(g, d, f, scale=d ** -0.5)), fp8_weight(_randn(g, f, d, scale=f ** -0.5))
    b1, b2 = _randn(g, f), _randn(g, d)
    h, s = add_rms_norm_fp8(x, r, gamma)
    a = gemm_fp8(h, W1.fwd, out_dtype=torch.float8_e4m3fn, bias=b1, activation="gelu")
    y = gemm_fp8(a, W2.fwd, bias=b2, residual=s)
    s64 = _np(s)
    assert torch.equal(s, (x.double() + r.double()).bfloat16())
    _check_norm_8_bits(h, s64 * _norm64(s64) * _np(gamma), 30 * U)
    _check_8_bits(a, *_finish(*_sums(_np(h.dequantize()), _np(W1.fwd.dequantize()), False), _np(b1), "gelu", None))
    want, e = _finish(*_sums(_np(a.dequantize()), _np(W2.fwd.dequantize()), False), _np(b2), None, s64)
    assert (np.abs(_np(y) - want) <= e * 1.01 + HALF["bfloat16"] * np.abs(want)).all()


class _Block:
    """A pre-norm feed-forward block whose products are in 8 bits, and a step of plain gradient descent on it."""

    def __init__(self, dev, seed, d=160, f=264, main_grad=False):
        import torch

        g = torch.Generator(device=dev).manual_seed(seed)
        self.p = [1 + 0.1 * _randn(g, d), _randn(g, d, f, scale=d ** -0.5), _randn(g, f), _randn(g, f, d, scale=f ** -0.5),
                  _randn(g, d)]
        self.p = [t.requires_grad_(True) for t in self.p]
        if main_grad:
            for t in self.p:
                t.main_grad = torch.empty(t.shape, device=dev)

    def forward(self, x, r):
        from nlearn_amd.kernels.fp8 import linear_fp8
        from nlearn_amd.kernels.fused import add_rms_norm

        gamma, W1, b1, W2, b2 = self.p
        h, s = add_rms_norm(x, r, gamma)
        return linear_fp8(linear_fp8(h, W1, bias=b1, activation="silu"), W2, bias=b2, residual=s)

    def step(self, x, r, dy, most=0.5):
        import torch
        from nlearn_amd.kernels.clip import clip_by_global_norm

        y = self.forward(x, r)
        if hasattr(self.p[0], "main_grad"):
            y.backward(dy)
            grads = [t.main_grad for t in self.p]
        else:
            grads = torch.autograd.grad(y, self.p, dy)
        clipped, norm = clip_by_global_norm(grads, most)
        with torch.no_grad():
            for t, c in zip(self.p, clipped):
                t.sub_(c, alpha=0.1)
        return y.detach(), norm, clipped


def _batches(dev, n, M=90, d=160):
    import torch

    g = torch.Generator(device=dev).manual_seed(77)
    return [(_randn(g, M, d, dtype=torch.bfloat16), _randn(g, M, d, dtype=torch.bfloat16),
             _randn(g, M, d, dtype=torch.bfloat16, scale=0.1 * 4.0 ** i)) for i in range(n)]


def test_training_step_runs_and_clips(dev):
    """Gradients of their own and in buffers are the same bits; steps are clipped to the norm, and deterministic."""
    import torch

    batches = _batches(dev, 4)
    runs = [_Block(dev, 3, main_grad=m) for m in (False, True, False)]
    for b in batches:
        outs = [r.step(*b) for r in runs]
        for o in outs[1:]:
            assert torch.equal(o[0], outs[0][0]) and torch.equal(o[1], outs[0][1])
            assert all(torch.equal(p, q) for p, q in zip(o[2], outs[0][2]))
        total = sum(float((_np(c) ** 2).sum()) for c in outs[0][2]) ** 0.5
        n = float(outs[0][1])
        assert n > 0.5 and abs(total - 0.5) <= 0.5 * 8 * U
    for r in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(r.p, runs[0].p))
    assert all(torch.isfinite(t).all() for t in runs[0].p)


def test_training_steps_in_a_graph(dev):
    """Captured once, replayed on new batches with eager steps of another block between the replays."""
    import torch

    batches = _batches(dev, 3)
    eager, block, other = _Block(dev, 5, main_grad=True), _Block(dev, 5, main_grad=True), _Block(dev, 6, main_grad=True)
    start = [t.detach().clone() for t in block.p]
    bufs = [t.clone() for t in batches[0]]
    block.step(*bufs)                     # what the allocator and the library look up once
    with torch.no_grad():
        for t, s in zip(block.p, start):
            t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, norm, clipped = block.step(*bufs)
    for b in batches + batches[:2]:
        for t, s in zip(bufs, b):
            t.copy_(s)
        graph.replay()
        want = eager.step(*b)
        other.step(*b)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(norm, want[1])
        assert all(torch.equal(p, q) for p, q in zip(clipped, want[2]))
        assert all(torch.equal(p, q) for p, q in zip(block.p, eager.p))


def test_frozen_block_in_a_graph_and_on_two_streams(dev):
    import torch
    from nlearn_amd.kernels.fp8 import add_rms_norm_fp8, fp8_weight, gemm_fp8

    g = torch.Generator(device=dev).manual_seed(12)
    W1, W2 = fp8_weight(_randn(g, 256, 1024, scale=1 / 16)), fp8_weight(_randn(g, 1024, 256, scale=1 / 32))
    b1, gamma = _randn(g, 1024), 1 + 0.1 * _randn(g, 256)

    def run(x, r):
        h, s = add_rms_norm_fp8(x, r, gamma)
        return gemm_fp8(gemm_fp8(h, W1.fwd, out_dtype=torch.float8_e4m3fn, bias=b1, activation="relu"), W2.fwd, residual=s), s

    for M in (1, 100, 2000):
        sets = [(_randn(g, M, 256, dtype=torch.bfloat16), _randn(g, M, 256, dtype=torch.bfloat16)) for _ in range(3)]
        want = [run(*s) for s in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(dev) for _ in sets]
        got = []
        for _ in range(3):
            for st, s in zip(streams, sets):
                with torch.cuda.stream(st):
                    got.append(run(*s))
        torch.cuda.synchronize()
        for n, o in enumerate(got):
            assert all(torch.equal(a, b) for a, b in zip(o, want[n % 3]))
        bufs = [t.clone() for t in sets[0]]
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):  # two graphs of the same calls, replayed beside each other
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = run(*bufs)
            graphs.append((graph, out))
        for s, ref in zip(sets + sets, want + want):
            for t, v in zip(bufs, s):
                t.copy_(v)
            torch.cuda.synchronize()
            for (graph, _), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, ref))
            run(*sets[1])


def test_backward_twice_under_hooks_and_in_a_checkpoint(dev):
    import torch
    from torch.utils.checkpoint import checkpoint

    block = _Block(dev, 9)
    x, r, dy = _batches(dev, 1)[0]
    x, r = x.requires_grad_(True), r.requires_grad_(True)
    leaves = [x, r, *block.p]
    y = block.forward(x, r)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert torch.equal(want[0], want[1])
    again = torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        hooked = torch.autograd.grad(block.forward(x, r), leaves, dy)
    ckpt = torch.autograd.grad(checkpoint(block.forward, x, r, use_reentrant=False), leaves, dy)
    for got in (again, hooked, ckpt):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):  # freed by the backward pass
        torch.autograd.grad(y, leaves, dy)
    # a second derivative is refused, not silently zero
    y = block.forward(x, r)
    (gx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.float().sum().backward()


def test_block_gradients_against_the_formula(dev):
    """The whole block in fp32 against autograd in float64 of the same quantised operands: dX of the first norm.

    u = x W + b of the fp32 layer is not rounded, and the second layer's input is quantised from fp32; the float64
    restatement takes those quantised values as they came out, so what differs is fp32 sums: 1e-5 of the norm."""
    import torch
    from nlearn_amd.kernels.fp8 import linear_fp8, quantize_fp8, quantize_fp8_both
    from nlearn_amd.kernels.fused import add_rms_norm

    block = _Block(dev, 21, d=96, f=128)
    gamma, W1, b1, W2, b2 = block.p
    g = torch.Generator(device=dev).manual_seed(1)
    x, r, dy = (_randn(g, 64, 96) for _ in range(3))
    x = x.requires_grad_(True)
    h, s = add_rms_norm(x, r, gamma)
    a = linear_fp8(h, W1, bias=b1, activation="silu")
    y = linear_fp8(a, W2, bias=b2, residual=s)
    mid = torch.autograd.grad(y, (a, h), dy, retain_graph=True)
    got = torch.autograd.grad(y, (x, gamma), dy)
    q = lambda t, **k: _np(quantize_fp8(t.detach(), **k).dequantize())  # noqa: E731
    w1, w2 = (_np(quantize_fp8_both(t.detach(), group=128)[0].dequantize()) for t in (W1, W2))
    da = q(dy) @ w2.T
    near = lambda p, v: np.linalg.norm(_np(p) - v) <= 1e-5 * np.linalg.norm(v)  # noqa: E731
    assert near(mid[0], da)
    u = q(h) @ w1 + _np(b1)
    du = torch.from_numpy((_np(mid[0]) * _act(u, "silu")[1]).astype(np.float32)).to(dev)
    # du is off by 40 u at most, so it stands beside a tie of its quantisation with a share of 2 * 40 u / 2^-4 =
    # 8e-5 of the values, which are then off by 2^-3 at most: sqrt(8e-5) / 8 = 1.1e-3 of the whole
    dh = q(du) @ w1.T
    assert np.linalg.norm(_np(mid[1]) - dh) <= 2e-3 * np.linalg.norm(dh)
    s64, d64 = _np(s), _np(mid[1]) + 0.0
    s64 = torch.from_numpy(s64).requires_grad_(True)
    g64 = torch.from_numpy(_np(gamma)).requires_grad_(True)
    n = s64 / torch.sqrt((s64 ** 2).mean(1, keepdim=True) + 1e-5) * g64
    ds, dg = torch.autograd.grad(n, (s64, g64), torch.from_numpy(d64))
    assert near(got[0], ds.numpy() + _np(dy)) and near(got[1], dg.numpy())
