"""nlearn_amd.kernels.clip — the global norm of many tensors, and clipping by it.

* ``global_norm(tensors)``: the L2 norm over all elements of all of them.
* ``clip_by_global_norm(grads, max_norm)``: optax.clip_by_global_norm, as the reference
  chains it in front of AdamW (train.py:502-506), for gradients in tensors of their own.
  ``train.AdamW`` clips in one pass with its update where the gradients lie in its
  buffer, and through this where they do not.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .gemm import _BF16, _F32, _check_device

_WS = 8192  # NL_GLOBAL_NORM_MULTI_WS


def rows_of(t: torch.Tensor):
    """(rows, columns, row stride) that walk every element of t once, or None."""
    if t.is_contiguous():
        n = t.numel()
        return 1, n, n
    if t.dim() == 2:
        (rows, cols), (ld, one) = t.shape, t.stride()
        if one == 1 and ld > cols and rows > 1:
            return rows, cols, ld
    dims = sorted(((st, n) for n, st in zip(t.shape, t.stride()) if n != 1))
    cols = 1
    while dims and dims[0][0] == cols:      # dense so far
        cols *= dims.pop(0)[1]
    if not dims:
        return 1, cols, cols
    ld, rows = dims.pop(0)
    for st, n in dims:
        if st != ld * rows:
            return None
        rows *= n
    return (rows, cols, ld) if ld >= cols else None


def _table(what: str, tensors, outs):
    """(nl_grad_tensor table, the device's first tensor); ``outs`` gives what each result is written to."""
    words, first = [], tensors[0]
    index = first.get_device()
    for t, o in zip(tensors, outs):
        dtype = t.dtype
        if dtype is _F32:
            code = 0
        elif dtype is _BF16:
            code = 1
        else:
            raise ValueError(f"{what}: tensors must be float32 or bfloat16, got {dtype}")
        if t.get_device() != index:
            raise ValueError(f"{what}: all tensors must be on one device, got {first.device} and {t.device}")
        if t.is_contiguous():
            n = t.numel()
            if n:
                words += (t.data_ptr(), o.data_ptr(), 1, n, n, n, code)
            continue
        lay = rows_of(t)
        if lay is None:
            raise ValueError(f"{what}: a tensor of shape {tuple(t.shape)} with strides {t.stride()} has no rows of one "
                             f"stride (make it contiguous)")
        rows, cols, ld = lay
        words += (t.data_ptr(), o.data_ptr(), rows, cols, ld, ld, code)
    _check_device(first)
    return (ctypes.c_int64 * len(words))(*words), len(words) // 7, first


def global_norm(tensors) -> torch.Tensor:
    """sqrt of the sum of squares of all elements of all ``tensors`` (fp32 or bf16, dense or
    rows of one stride): a 0-d fp32 tensor, summed in fp64 in a fixed order, with no host
    synchronisation. Not differentiable. At least one tensor (it names the device)."""
    tensors = list(tensors)
    if not tensors:
        raise ValueError("global_norm: no tensors")
    table, n, first = _table("global_norm", tensors, tensors)
    norm = torch.empty((), dtype=_F32, device=first.device)
    ws = torch.empty(_WS, dtype=torch.uint8, device=first.device)
    _lib.call_on(first, "nl_global_norm_multi", n, table, norm.data_ptr(), ws.data_ptr(), _WS)
    return norm


def clip_by_global_norm(grads, max_norm: float, inplace: bool = False):
    """(clipped, norm): every gradient g as it is while norm = global_norm(grads) < max_norm,
    else as (g / norm) * max_norm, in g's dtype and layout. The norm stays on the device.
    A new tensor keeps g's strides and so spans as much memory as g does: the result of a
    narrow slice of a wide matrix has nearly that matrix's size (clip a dense copy, or in
    place, where that is too much).

    ``inplace=True`` writes the results over the gradients (which may not overlap) and only
    where the norm reaches max_norm; otherwise they are new tensors. With a norm that is
    infinite finite gradients become 0, with one that is NaN all become NaN, as optax has it."""
    grads = list(grads)
    if not grads:
        raise ValueError("clip_by_global_norm: no gradients")
    max_norm = float(max_norm)
    if not 1e-37 <= max_norm <= 1e38:  # a normal fp32 number; NaN fails too
        raise ValueError(f"clip_by_global_norm: max_norm must lie in [1e-37, 1e38], got {max_norm}")
    if inplace:
        outs = grads
        if len({t.data_ptr() for t in grads if t.numel()}) < sum(t.numel() > 0 for t in grads):
            raise ValueError("clip_by_global_norm: a gradient stands in the list twice")
    else:
        outs = [torch.empty_like(t) if t.is_contiguous() else t.new_empty_strided(t.shape, t.stride()) for t in grads]
    table, n, first = _table("clip_by_global_norm", grads, outs)
    norm = torch.empty((), dtype=_F32, device=first.device)
    ws = torch.empty(_WS, dtype=torch.uint8, device=first.device)
    _lib.call_on(first, "nl_clip_by_global_norm", n, table, max_norm, norm.data_ptr(), ws.data_ptr(), _WS)
    return outs, norm
