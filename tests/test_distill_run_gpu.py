"""A student trained from a frozen teacher, the operators together as a program uses them: the teacher's LM head
in 8 bits, its top logits, the student's loss and the gradients of its weights."""
import numpy as np
import pytest

from oracle import distill_fp8 as orc

pytestmark = pytest.mark.gpu


def _models(dev):
    from nlearn_amd.model import ModelConfig, init_model

    student = ModelConfig(vocab_size=1003, d_model=128, n_heads=2, n_layers=1, d_ff=256, max_seq_len=64)
    teacher = ModelConfig(vocab_size=1003, d_model=512, n_heads=8, n_layers=2, d_ff=2048, max_seq_len=64)
    return (init_model(1, student, dev), student), (init_model(2, teacher, dev), teacher)


def _answers(teacher, ids, k, T):
    import torch
    from nlearn_amd.kernels.distill import top_logits
    from nlearn_amd.kernels.fp8 import fp8_weight, linear_fp8
    from nlearn_amd.model import model_forward_features, output_projection

    params, cfg = teacher
    with torch.no_grad():
        head = fp8_weight(output_projection(params))
        x = model_forward_features(params, ids, cfg)
        logits = linear_fp8(x, head)
        return x, logits, top_logits(logits, k, T)


@pytest.mark.parametrize("head", ["bf16", "fp8"])
def test_student_step_from_a_teacher(dev, head):
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy
    from nlearn_amd.kernels.fp8 import linear_fp8
    from nlearn_amd.kernels.gemm import linear
    from nlearn_amd.model import model_forward_features, output_projection, tree_leaves

    (params, cfg), teacher = _models(dev)
    ids = torch.from_numpy(np.random.default_rng(5).integers(0, 1003, (3, 50)).astype(np.int32)).to(dev)
    T, k = 2.0, 16
    xt, tl, (values, tids, lse) = _answers(teacher, ids, k, T)
    assert tl.shape == (3, 50, 1003) and values.shape == tids.shape == (3, 50, k) and lse.shape == (3, 50)

    # the teacher's logits are the product of its quantised operands (to bf16 and the 8-bit sums, 2^-7 of the scale)
    q = lambda a, g: orc.values(*orc.quantize(a, g), g)[:, :a.shape[1]]  # noqa: E731
    W = output_projection(teacher[0]).detach().double().cpu().numpy()
    x64 = q(xt.double().cpu().numpy().reshape(150, -1), 1) @ q(W, 128)
    got = tl.double().cpu().numpy().reshape(150, -1)
    assert np.abs(got - x64).max() <= 2.0 ** -7 * np.abs(x64).max()
    tid64, lse64 = orc.top(got, k, T)
    np.testing.assert_array_equal(tids.cpu().numpy().reshape(150, k), tid64)

    Wh = output_projection(params)
    x = model_forward_features(params, ids, cfg)
    x.retain_grad()
    logits = linear(x, Wh) if head == "bf16" else linear_fp8(x, Wh)
    z64 = logits.detach().double().cpu().numpy().reshape(150, -1)
    loss = distill_cross_entropy(logits, tids, values, lse, T, inplace=True)
    loss.backward()

    ref, d, _, _ = orc.distill(z64, tid64, values.double().cpu().numpy().reshape(150, k),
                               lse.double().cpu().numpy().reshape(150), T, 1 / 150)
    assert abs(loss.item() - ref.mean()) <= 1e-5 * abs(ref.mean()) + 1e-6
    # dlogits as bf16 (half a step, 2^-8), then the head's products: dX = d W^T, dW = X^T d
    xs, Ws = x.detach().double().cpu().numpy().reshape(150, -1), Wh.detach().double().cpu().numpy()
    if head == "bf16":
        Wb = Wh.detach().to(torch.bfloat16).double().cpu().numpy()
        dx, dW = d @ Wb.T, xs.T @ d
        lx, lw = np.abs(d) @ np.abs(Wb).T, np.abs(xs).T @ np.abs(d)
        # 2^-8 of every term for d's rounding and of the sum for the result's, doubled
        assert (np.abs(x.grad.double().cpu().numpy().reshape(150, -1) - dx) <= 2.0 ** -7 * (lx + np.abs(dx))).all()
        assert (np.abs(Wh.grad.double().cpu().numpy() - dW) <= 2.0 ** -7 * lw).all()
    else:
        db = orc_bf16(d)
        dx = q(db, 1) @ q(Ws, 128).T
        dW = q(xs.T, 1) @ q(db.T, 1).T
        # a rounding of dlogits to the other bf16 neighbour (2^-8) may move it to the next e4m3 value (2^-3)
        lx, lw = np.abs(d) @ np.abs(Ws).T, np.abs(xs).T @ np.abs(d)
        assert (np.abs(x.grad.double().cpu().numpy().reshape(150, -1) - dx) <= 2.0 ** -3 * lx + 2.0 ** -7 * np.abs(dx)).all()
        assert (np.abs(Wh.grad.double().cpu().numpy() - dW) <= 2.0 ** -3 * lw).all()
    for p in tree_leaves(params):
        assert p.grad is not None and torch.isfinite(p.grad).all()
    assert all(p.grad is None for p in tree_leaves(teacher[0]))


def orc_bf16(d):
    from oracle.ops import bf16_round

    return bf16_round(d.astype(np.float32)).astype(np.float64)


def test_no_gradient_is_formed_without_need(dev):
    """Under no_grad the logits stay as they are, in place or not."""
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy, top_logits
    from nlearn_amd.kernels.fp8 import linear_fp8

    x = torch.randn((20, 300), device=dev).to(torch.bfloat16)
    z = x.clone().requires_grad_(True)
    v, i, l = top_logits(x, 4)
    with torch.no_grad():
        loss = distill_cross_entropy(z, i, v, l, inplace=True)
        W = torch.randn((300, 40), device=dev).requires_grad_(True)
        y = linear_fp8(z, W)
    assert torch.equal(z, x) and not loss.requires_grad and not y.requires_grad
    assert torch.equal(loss, distill_cross_entropy(x, i, v, l))


def test_side_stream_and_two_calls_at_once(dev):
    """The same calls on two streams, beside each other, give what one alone gives."""
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy, top_logits

    g = torch.Generator(device=dev).manual_seed(3)
    xs = [(torch.randn((64, 20011), generator=g, device=dev) * 2).to(torch.bfloat16) for _ in range(2)]

    def run(x):
        v, i, l = top_logits(x, 33, 1.5)
        z = x.detach().clone().requires_grad_(True)
        loss = distill_cross_entropy(z, i.flip(1), v.flip(1), l, 1.5)
        loss.backward()
        return v, i, l, loss.detach(), z.grad

    want = [run(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in xs]
    got = []
    for _ in range(3):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(run(x))
    torch.cuda.synchronize()
    for n, outs in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(outs, want[n % 2]))


def test_training_step_in_a_graph(dev):
    """Two 8-bit layers, the loss and all gradients captured once and replayed on new batches; the weights'
    gradients go to buffers, of which the head's has rows off 16 bytes."""
    import torch
    from nlearn_amd.kernels.distill import distill_cross_entropy
    from nlearn_amd.kernels.fp8 import linear_fp8

    g = torch.Generator(device=dev).manual_seed(8)
    M, D, V, k = 70, 256, 301, 9
    W1, W2 = ((torch.randn(s, generator=g, device=dev) / 16).requires_grad_(True) for s in ((D, D), (D, V)))
    sets = [(torch.randn((M, D), generator=g, device=dev).to(torch.bfloat16),
             torch.randint(0, V, (M, k), generator=g, device=dev, dtype=torch.int32),
             torch.randn((M, k), generator=g, device=dev)) for _ in range(3)]

    def step(x, i, v):
        for W in (W1, W2):
            W.main_grad.fill_(float("nan"))
        loss = distill_cross_entropy(linear_fp8(linear_fp8(x, W1), W2), i, v, None, 2.0, inplace=True)
        loss.backward()
        return loss.detach()

    for W in (W1, W2):
        W.main_grad = torch.empty(tuple(W.shape), device=dev)
    want = [(step(*s).clone(), W1.main_grad.clone(), W2.main_grad.clone()) for s in sets]
    bufs = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(*bufs)
    for _ in range(2):
        for s, ref in zip(sets, want):
            for b, t in zip(bufs, s):
                b.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((loss, W1.main_grad, W2.main_grad), ref))
            assert torch.isfinite(W2.main_grad).all() and W1.grad is None and W2.grad is None
            step(*sets[1])
