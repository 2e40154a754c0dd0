"""AdamW without gradient buffers, clipping: gradients that share memory among their elements, leaves without one."""
import pytest

pytestmark = pytest.mark.gpu


def test_broadcast_and_missing_gradients(dev):
    """Every .grad holds the clipped gradient afterwards, and the update is that of dense gradients."""
    import torch
    from nlearn_amd.train import AdamW

    g = torch.Generator(device=dev).manual_seed(7)
    shapes = [(40, 56), (333,), (24, 8), (8, 3, 16), (5,)]
    start = [torch.randn(s, generator=g, device=dev) for s in shapes]
    row = torch.randn((1, 56), generator=g, device=dev)
    dense = torch.randn((333,), generator=g, device=dev)
    column = torch.randn((24, 1), generator=g, device=dev)
    middle = torch.randn((8, 1, 16), generator=g, device=dev)
    grads = [row.expand(40, 56), dense, column.expand(24, 8), middle.expand(8, 3, 16), None]
    kept = [t.clone() for t in (row, column, middle)]
    after = []
    for whole in (False, True):
        leaves = {str(i): t.clone().requires_grad_(True) for i, t in enumerate(start)}
        opt = AdamW(lambda c: 1e-2, clip_norm=2.0, grad_buffers=False)
        state = opt.init(leaves)
        for p, t in zip(leaves.values(), grads):
            p.grad = None if t is None else t.contiguous().clone() if whole else t.clone() if t is dense else t
        opt.update(leaves, state)
        assert leaves["4"].grad is None and torch.equal(leaves["4"].detach(), start[4])
        norm = torch.cat([t.double().flatten() for t in grads[:4]]).norm()
        assert float(norm) > 2 and abs(float(state["gnorm"]) - float(norm)) <= 1e-6 * float(norm)
        for p, t in zip(list(leaves.values())[:4], grads):
            want = t.double() / norm * 2
            assert ((p.grad.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all(), tuple(p.shape)
        after.append([p.detach() for p in leaves.values()] + state["mu"] + state["nu"])
    assert all(torch.equal(a, b) for a, b in zip(*after))
    assert all(torch.equal(a, b) for a, b in zip(kept, (row, column, middle)))  # what was broadcast is the caller's
