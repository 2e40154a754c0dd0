"""nlearn_amd.kernels.distill — a student's loss against a teacher's top logits.

* ``top_logits(logits, k)``: the k largest logits of each row, their ids and the
  row's logsumexp, from one read of the logits: what is kept of a teacher.
* ``distill_cross_entropy(logits, ids, values)``: T^2 KL(teacher || student) over
  those entries, mean over the rows, with the gradient of the student's logits
  from the same pass (as ``cross_entropy`` does it).

The reference has no distillation: these stand beside its softmax cross-entropy
(cross_entropy.py:71-81), whose conventions they keep.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .cross_entropy import _BF16, _ld
from .gemm import _check_device

_F32 = torch.float32
MAX_K = 256  # NL_TOP_MAX_K


def _rows(what: str, logits: torch.Tensor) -> torch.Tensor:
    dim = logits.dim()
    if dim < 1 or logits.dtype is not _BF16:
        raise ValueError(f"{what}: logits must be bfloat16 with the vocabulary as last dimension")
    V = logits.shape[-1]
    if V < 1:
        raise ValueError(f"{what}: an empty vocabulary")
    x = logits if dim == 2 else logits.reshape(-1, V)
    s0, s1 = x.stride()
    if s1 != 1 and V > 1:
        raise ValueError(f"{what}: logits need a unit stride along the vocabulary")
    if max(x.shape) >= 1 << 31:  # the kernels count rows and logits in 32 bits
        raise ValueError(f"{what}: sizes must be less than 2^31, got {tuple(x.shape)}")
    if s0 < V and x.shape[0] > 1:  # rows sharing memory (a broadcast view)
        x = x.contiguous()
    return x


def _dense(t: torch.Tensor, k: int) -> torch.Tensor:
    return t if t.dim() == 2 and t.is_contiguous() else t.reshape(-1, k).contiguous()


def _temperature(what: str, t) -> float:
    t = float(t)
    if not 1e-3 <= t <= 1e6:  # NaN fails too
        raise ValueError(f"{what}: the temperature must lie in [1e-3, 1e6], got {t}")
    return t


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0):
    """(values, ids, lse) of bf16 logits[..., V]: the k largest of each row, largest
    first and equal ones by the lower id, as bf16 [..., k] and int32 [..., k], and
    lse = logsumexp(logits / temperature) over the whole row, fp32 [...].

    exp(values / temperature - lse) are the row's probabilities, to 2^-24 of |lse|: rows
    1e5 and more away from zero are better moved to their maximum first. NaN counts as
    larger than any number. 1 <= k <= min(V, 256). Not differentiable."""
    x = _rows("top_logits", logits)
    T = _temperature("top_logits", temperature)
    M, V = x.shape
    if not 1 <= k <= min(V, MAX_K):
        raise ValueError(f"top_logits: need 1 <= k <= min(V, {MAX_K}), got k = {k} with V = {V}")
    _check_device(x)
    lead = logits.shape[:-1]
    values = torch.empty((*lead, k), dtype=_BF16, device=x.device)
    ids = torch.empty((*lead, k), dtype=torch.int32, device=x.device)
    lse = torch.empty(lead, dtype=_F32, device=x.device)
    _lib.call_on(x, "nl_top_logits", M, V, x.data_ptr(), _ld(x), int(k), T, values.data_ptr(),
                 ids.data_ptr(), lse.data_ptr())
    return values, ids, lse


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, values, lse, T, inplace, need):
        M, V = x.shape
        loss_rows = torch.empty(M, dtype=_F32, device=x.device)
        loss = torch.empty((), dtype=_F32, device=x.device)
        d = None
        if need:
            # rows of the gradient start at the same offsets from 16 bytes as the logits'
            d = x if inplace else torch.empty_strided((M, V), (V + (_ld(x) - V) % 8, 1), dtype=_BF16, device=x.device)
        _lib.call_on(x, "nl_distill_fwd_bwd", M, V, x.data_ptr(), _ld(x), ids.shape[1], ids.data_ptr(),
                     int(ids.dtype is torch.int64), values.data_ptr(),
                     _lib.NL_DTYPE_F32 if values.dtype is _F32 else _lib.NL_DTYPE_BF16,
                     lse.data_ptr() if lse is not None else None, T, loss_rows.data_ptr(), loss.data_ptr(), 1.0 / max(M, 1),
                     d.data_ptr() if d is not None else None, _ld(d) if d is not None else 0)
        ctx.d = d
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        d, ctx.d = ctx.d, None
        if d is None:
            raise RuntimeError("distill_cross_entropy: the gradient is formed once and handed out by the first "
                               "backward pass; call the loss again")
        g = g.to(_F32)
        _lib.call_on(d, "nl_scale_bf16_by_device_scalar", d.data_ptr(), d.shape[0], d.shape[1], _ld(d), g.data_ptr())
        return d, None, None, None, None, None, None


def distill_cross_entropy(logits: torch.Tensor, ids: torch.Tensor, values: torch.Tensor,
                          lse: torch.Tensor | None = None, temperature: float = 1.0,
                          inplace: bool = False) -> torch.Tensor:
    """Mean over the rows of T^2 sum_j p_j (log p_j - log q[id_j]), q = softmax(logits / T).

    logits [..., V] bf16 (the student's), ids [..., k] int32 or int64, values
    [..., k] bf16 or fp32 (the teacher's logits), T the temperature. With ``lse``
    [...] (the teacher's logsumexp at T, as ``top_logits`` gives it) p_j =
    exp(values_j / T - lse); without it p is the softmax of the row's k values / T,
    wherever they stand.

    An entry with a negative id is padding. An id may stand in a row more than
    once: its probabilities add up (a hard target can ride along as an entry of
    its own, with values in log-probabilities, T = 1 and lse of zeros). A row
    without any weight adds 0 to the mean and has a zero gradient. An id >= V, or
    a NaN, makes its row's loss and gradient NaN. 1 <= k <= 256.

    Where logits need a gradient it is formed by the same pass over them (and handed
    out by one backward pass); ``inplace=True`` writes it over ``logits`` (when nothing
    else reads them)."""
    x = _rows("distill_cross_entropy", logits)
    T = _temperature("distill_cross_entropy", temperature)
    M, V = x.shape
    lead = logits.shape[:-1]
    if ids.dim() < 1 or ids.shape[:-1] != lead or values.shape != ids.shape:
        raise ValueError(f"distill_cross_entropy: ids {tuple(ids.shape)} and values {tuple(values.shape)} must both be "
                         f"{tuple(lead)} + (k,)")
    k = ids.shape[-1]
    if not 1 <= k <= MAX_K:
        raise ValueError(f"distill_cross_entropy: need 1 <= k <= {MAX_K}, got {k}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"distill_cross_entropy: ids must be int32 or int64, got {ids.dtype}")
    if values.dtype not in (_BF16, _F32):
        raise ValueError(f"distill_cross_entropy: values must be bfloat16 or float32, got {values.dtype}")
    if values.requires_grad or (lse is not None and lse.requires_grad):
        raise ValueError("distill_cross_entropy: the teacher gets no gradient (detach values and lse)")
    if lse is not None:
        if lse.dtype is not _F32 or lse.shape != lead:
            raise ValueError(f"distill_cross_entropy: lse must be float32 of shape {tuple(lead)}")
        if lse.dim() != 1 or not lse.is_contiguous():
            lse = lse.reshape(-1).contiguous()
    if inplace and x.data_ptr() != logits.data_ptr():
        raise ValueError("distill_cross_entropy: inplace needs logits whose rows can be written where they are")
    ids, values = _dense(ids, k), _dense(values, k)
    _check_device(x, ids, values)
    dev = x.get_device()
    if ids.get_device() != dev or values.get_device() != dev or (lse is not None and lse.get_device() != dev):
        raise ValueError("distill_cross_entropy: all tensors must be on the logits' device")
    return _Distill.apply(x, ids, values, lse, T, bool(inplace), x.requires_grad and torch.is_grad_enabled())
