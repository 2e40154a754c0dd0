"""nlearn_amd.kernels.fused — the model's non-GEMM layers on the HIP kernels.

* ``layer_norm(x, gamma, beta)`` and ``add_layer_norm(x, r, gamma, beta)``:
  LayerNorm with fp32 statistics (nlearn/model.py:228-241), the second one
  with the residual add of the block folded in (model.py:315-324): it returns
  both LN(x + r) and the new residual stream x + r, reading x and r once.
* ``rms_norm(x, gamma)`` and ``add_rms_norm(x, r, gamma)``: the same pair without
  the mean, as the reference's own blocks have it (model.py:228-241); bf16 or fp32
  rows of any stride. ``fp8.rms_norm_fp8`` writes the result in 8 bits.
* ``ffn(x, W1, b1, W2, b2)``: the FFN (model.py:266-277, with the benchmark's
  tanh-GELU and biases) as two GEMMs whose epilogues add the biases and apply
  the GELU; the backward's dX GEMM applies the GELU derivative in its
  epilogue, so no elementwise kernel runs between the GEMMs.
* ``embedding(ids, tok, pos)``: token + learned-position lookup (model.py:75-85);
  ``embedding_layer_norm`` is the lookup together with the first LayerNorm.

Every op is an autograd Function whose forward and backward are C-ABI calls;
there is no framework fallback.
"""
from __future__ import annotations

import contextlib
import functools

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from . import wgrad
from .gemm import (EPI_BIAS, EPI_BIAS_GELU, EPI_DGELU, _check_device, _kernel_ready, _ld, bf16_shadow, gemm_raw,
                   grad_buffer, padded_empty, weight_grad)

_BF16 = torch.bfloat16
_F32 = torch.float32


def _stream(t: torch.Tensor) -> int:
    return _lib.stream_of(t)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Dense bf16 [rows, D] view of x (copies only if x is not already one)."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.dtype != _BF16:
        x2 = x2.to(_BF16)
    if not x2.is_contiguous() or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    return x2


def _param(p: torch.Tensor) -> torch.Tensor:
    p = p.detach()
    if p.dtype != _F32:
        p = p.to(_F32)
    return p if p.is_contiguous() else p.contiguous()


# ---------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------


def layer_norm_fwd_raw(x2, gamma, beta, eps, residual=None):
    """-> y, s, mean, rstd with s = bf16(x + residual) (None without a residual)."""
    _check_device(x2, gamma, beta)
    rows, D = x2.shape
    y = torch.empty_like(x2)
    s = torch.empty_like(x2) if residual is not None else None
    mean = torch.empty(rows, dtype=_F32, device=x2.device)
    rstd = torch.empty(rows, dtype=_F32, device=x2.device)
    _lib.call("nl_layernorm_fwd", _stream(x2), rows, D, x2.data_ptr(),
              residual.data_ptr() if residual is not None else None, s.data_ptr() if s is not None else None,
              gamma.data_ptr(), beta.data_ptr(), float(eps), y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    return y, s, mean, rstd


_ln_defer: dict | None = None   # set inside defer_layer_norm_param_sums()


@contextlib.contextmanager
def defer_layer_norm_param_sums():
    """Inside the block, a LayerNorm backward that writes dgamma / dbeta into
    main_grad buffers leaves them as partial rows, which the next such
    backward's kernel launch reduces (nl_layernorm_bwd_deferred); leaving the
    block reduces the last ones (nl_layernorm_param_sums). The buffers are
    complete only after the block, so it belongs around a backward pass whose
    parameter gradients an optimizer reads afterwards. The sums are the same
    bit for bit; the chain of 9 LayerNorm backwards loses 8 kernel launches.
    Module-global like kernels.wgrad (the autograd engine runs the backward
    on its own thread); one block at a time."""
    global _ln_defer
    if _ln_defer is not None:
        raise RuntimeError("defer_layer_norm_param_sums() does not nest")
    _ln_defer = {"pending": None}
    try:
        yield
    finally:
        pending, _ln_defer = _ln_defer["pending"], None
        if pending is not None:
            stream, ws, rows, D, dg, db = pending
            _lib.call("nl_layernorm_param_sums", stream, rows, D, ws.data_ptr(), dg.data_ptr(), db.data_ptr(), 0)


def layer_norm_bwd_raw(dy2, xin, mean, rstd, gamma, dres=None, dgamma=None, dbeta=None):
    """-> dx (+ dres), dgamma, dbeta (written into the given buffers if any;
    deferred inside ``defer_layer_norm_param_sums`` when both are given)."""
    rows, D = dy2.shape
    dx = torch.empty_like(dy2)
    wsb = int(_lib.load().nl_layernorm_bwd_ws_bytes(rows, D))
    ws = torch.empty(max(wsb, 16) // 4, dtype=_F32, device=dy2.device)
    dres_ptr = dres.data_ptr() if dres is not None else None
    if _ln_defer is not None and dgamma is not None and dbeta is not None:
        prev = _ln_defer["pending"]
        stream = _stream(dy2)
        if prev is not None and prev[0] != stream:
            raise RuntimeError("layer_norm backward: deferred parameter sums on two streams")
        pargs = (prev[2], prev[3], prev[1].data_ptr(), prev[4].data_ptr(), prev[5].data_ptr(), 0) if prev else \
            (0, 0, None, None, None, 0)
        _lib.call("nl_layernorm_bwd_deferred", stream, rows, D, dy2.data_ptr(), xin.data_ptr(), mean.data_ptr(),
                  rstd.data_ptr(), gamma.data_ptr(), dres_ptr, dx.data_ptr(), ws.data_ptr(), wsb, *pargs)
        # the previous partials are read by the launch just queued: stream order
        # keeps their memory from being reused before it runs
        _ln_defer["pending"] = (stream, ws, rows, D, dgamma, dbeta)
        return dx, dgamma, dbeta
    if dgamma is None:
        dgamma = torch.empty(D, dtype=_F32, device=dy2.device)
    if dbeta is None:
        dbeta = torch.empty(D, dtype=_F32, device=dy2.device)
    _lib.call("nl_layernorm_bwd", _stream(dy2), rows, D, dy2.data_ptr(), xin.data_ptr(), mean.data_ptr(),
              rstd.data_ptr(), gamma.data_ptr(), dres_ptr, dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), 0,
              ws.data_ptr(), wsb)
    return dx, dgamma, dbeta


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        x2 = _rows(x)
        g, b = _param(gamma), _param(beta)
        y, _, mean, rstd = layer_norm_fwd_raw(x2, g, b, eps)
        ctx.save_for_backward(x2, mean, rstd, g)
        ctx.shape = x.shape
        ctx.bufs = (grad_buffer(gamma), grad_buffer(beta))
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, mean, rstd, g = ctx.saved_tensors
        dx, dg, db = layer_norm_bwd_raw(_rows(dy), x2, mean, rstd, g, None, *ctx.bufs)
        return dx.view(ctx.shape), *_unless_buffered(ctx.bufs, (dg, db)), None


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, gamma, beta, eps):
        ctx.set_materialize_grads(False)
        x2, r2 = _rows(x), _rows(r)
        if x2.shape != r2.shape:
            raise ValueError("add_layer_norm: x and r differ in shape")
        g, b = _param(gamma), _param(beta)
        y, s, mean, rstd = layer_norm_fwd_raw(x2, g, b, eps, residual=r2)
        ctx.save_for_backward(s, mean, rstd, g)
        ctx.shape = x.shape
        ctx.bufs = (grad_buffer(gamma), grad_buffer(beta))
        return y.view(x.shape), s.view(x.shape)

    @staticmethod
    def backward(ctx, dy, ds):
        s, mean, rstd, g = ctx.saved_tensors
        if dy is None:
            dx = _rows(ds)
            return dx.view(ctx.shape), dx.view(ctx.shape), None, None, None
        dx, dg, db = layer_norm_bwd_raw(_rows(dy), s, mean, rstd, g, _rows(ds) if ds is not None else None,
                                        *ctx.bufs)
        dx = dx.view(ctx.shape)
        return dx, dx, *_unless_buffered(ctx.bufs, (dg, db)), None


def _wgrad(X, dY, buf):
    """X^T . dY into the gradient buffer (forked when overlapping), or a fresh fp32 tensor."""
    if buf is not None:
        return weight_grad(X, dY, buf)
    return gemm_raw(X, dY, "T", "N", out_dtype=_F32)


def _unless_buffered(bufs, grads):
    """Gradients to hand back to autograd: None where a main_grad buffer took them."""
    return tuple(None if b is not None else g for b, g in zip(bufs, grads))


def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """bf16 LayerNorm over the last dimension, fp32 statistics and parameters."""
    return _LayerNorm.apply(x, gamma, beta, eps)


def add_layer_norm(x: torch.Tensor, r: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                   eps: float = 1e-5):
    """(LN(s), s) with s = bf16(x + r): the residual add and the next LayerNorm in one pass."""
    return _AddLayerNorm.apply(x, r, gamma, beta, eps)


# ---------------------------------------------------------------------------
# RMS norm
# ---------------------------------------------------------------------------

MAX_RMS_COLUMNS = 16384


def _strided_rows(t: torch.Tensor):
    """(t as rows with a unit column stride that share no memory, their stride); copies only if it must."""
    x = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    (rows, D), (s0, s1) = x.shape, x.stride()
    if (D > 1 and s1 != 1) or (rows > 1 and s0 < D):
        return x.contiguous(), D
    return x, s0 if rows > 1 else D


def _check_rms(what: str, x: torch.Tensor, r, gamma: torch.Tensor, eps: float) -> float:
    if x.dim() < 1 or x.dtype not in (_BF16, _F32):
        raise ValueError(f"{what}: rows must be bfloat16 or float32, got {x.dtype} {tuple(x.shape)}")
    D = x.shape[-1]
    if not 1 <= D <= MAX_RMS_COLUMNS:
        raise ValueError(f"{what}: rows of 1 to {MAX_RMS_COLUMNS} elements, got {D}")
    if x.numel() // D >= 1 << 31:
        raise ValueError(f"{what}: fewer than 2^31 rows, got {x.numel() // D}")
    if r is not None and (r.shape != x.shape or r.dtype is not x.dtype):
        raise ValueError(f"{what}: x is {x.dtype} {tuple(x.shape)}, the residual {r.dtype} {tuple(r.shape)}")
    if gamma.shape != (D,) or gamma.dtype not in (_BF16, _F32):
        raise ValueError(f"{what}: gamma must be bfloat16 or float32 of shape {(D,)}, got {gamma.dtype} "
                         f"{tuple(gamma.shape)}")
    eps = float(eps)
    if not 1e-30 <= eps <= 1.0:  # NaN fails too
        raise ValueError(f"{what}: eps must lie in [1e-30, 1], got {eps}")
    dev = x.get_device()
    if gamma.get_device() != dev or (r is not None and r.get_device() != dev) or gamma.is_meta != x.is_meta:
        raise ValueError(f"{what}: all tensors must be on one device, got {x.device}, gamma on {gamma.device}")
    _check_device(x)
    return eps


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    """An empty dense tensor like t, without a gradient (the first form costs half of torch.empty's 2 us)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _rms_code(t: torch.Tensor) -> int:
    return _lib.NL_DTYPE_F32 if t.dtype is _F32 else _lib.NL_DTYPE_BF16


def _rms_fwd(x, r, gamma, eps, keep: bool):
    """(y, s or None, rstd or None), y and s dense of x's shape."""
    y = _dense_like(x)
    s = _dense_like(x) if r is not None else None
    x2, ldx = _strided_rows(x)
    rows, D = x2.shape
    rstd = x2.new_empty((rows,), dtype=_F32) if keep else None
    if rows:
        r2, ldr = _strided_rows(r) if r is not None else (None, 0)
        g = _param(gamma)
        _lib.call_on(x2, "nl_rms_norm_fwd", rows, D, _rms_code(x2), x2.data_ptr(), ldx,
                     r2.data_ptr() if r is not None else None, ldr, s.data_ptr() if r is not None else None, D,
                     g.data_ptr(), eps, y.data_ptr(), D, rstd.data_ptr() if keep else None)
    return y, s, rstd


@functools.lru_cache(maxsize=1024)
def _rms_ws_bytes(rows: int, D: int) -> int:
    return int(_lib.load().nl_rms_norm_bwd_ws_bytes(rows, D))


def _rms_grad_buffer(gamma: torch.Tensor):
    mg = grad_buffer(gamma)
    if mg is not None and (mg.shape != gamma.shape or mg.device != gamma.device or mg.dtype is not _F32
                           or not mg.is_contiguous()):
        raise ValueError(f"rms_norm: main_grad must be a dense float32 tensor of shape {tuple(gamma.shape)} on "
                         f"{gamma.device}")
    return mg


def _rms_bwd(ctx, dy, ds, s, rstd, gamma):
    """(dx, dgamma or None where a main_grad buffer took it)."""
    need_dg = ctx.gamma is not None
    mg = _rms_grad_buffer(ctx.gamma) if need_dg else None
    dx = _dense_like(s)
    s2, lds = _strided_rows(s)
    rows, D = s2.shape
    dg = None
    if need_dg:
        dg = mg if mg is not None else rstd.new_empty((D,))
    if rows == 0:
        if dg is not None:
            dg.zero_()
    else:
        d2, ldd = _strided_rows(dy if dy.dtype is s.dtype else dy.to(s.dtype))
        r2, ldr = _strided_rows(ds if ds.dtype is s.dtype else ds.to(s.dtype)) if ds is not None else (None, 0)
        g = _param(gamma)
        wsb = _rms_ws_bytes(rows, D) if need_dg else 0
        ws = rstd.new_empty((wsb // 4,)) if wsb else None
        _lib.call_on(s2, "nl_rms_norm_bwd", rows, D, _rms_code(s2), d2.data_ptr(), ldd, s2.data_ptr(), lds,
                     rstd.data_ptr(), g.data_ptr(), r2.data_ptr() if ds is not None else None, ldr, dx.data_ptr(), D,
                     dg.data_ptr() if need_dg else None, 0, ws.data_ptr() if wsb else None, wsb)
    return dx, dg.to(gamma.dtype) if need_dg and mg is None else None


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, eps):
        y, _, rstd = _rms_fwd(x, None, gamma, eps, True)
        ctx.save_for_backward(x, rstd, gamma)
        ctx.gamma = gamma if gamma.requires_grad else None  # for its main_grad
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return *_rms_bwd(ctx, dy, None, *ctx.saved_tensors), None


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, gamma, eps):
        ctx.set_materialize_grads(False)
        y, s, rstd = _rms_fwd(x, r, gamma, eps, True)
        ctx.save_for_backward(s, rstd, gamma)
        ctx.gamma = gamma if gamma.requires_grad else None
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        if dy is None:
            return ds, ds, None, None
        dx, dg = _rms_bwd(ctx, dy, ds, *ctx.saved_tensors)
        return dx, dx, dg, None


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * gamma over the last dimension (up to 16384 elements),
    in x's dtype, bf16 or fp32; statistics and gamma's gradient are fp32."""
    eps = _check_rms("rms_norm", x, None, gamma, eps)
    if not (torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad)):
        return _rms_fwd(x, None, gamma, eps, False)[0]
    return _RMSNorm.apply(x, gamma, eps)


def add_rms_norm(x: torch.Tensor, r: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5):
    """(rms_norm(s), s) with s = x + r rounded to their dtype: the residual add and the next norm in one pass."""
    eps = _check_rms("add_rms_norm", x, r, gamma, eps)
    if not (torch.is_grad_enabled() and (x.requires_grad or r.requires_grad or gamma.requires_grad)):
        return _rms_fwd(x, r, gamma, eps, False)[:2]
    return _AddRMSNorm.apply(x, r, gamma, eps)


# ---------------------------------------------------------------------------
# bias gradients
# ---------------------------------------------------------------------------


def colsum(x2: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 column sums of a bf16 [rows, cols] matrix (fixed summation order).

    With a preallocated ``out`` (a bias gradient buffer) the kernels are forked
    onto the weight-gradient stream when one is active (kernels.wgrad)."""
    rows, cols = x2.shape
    x2 = _kernel_ready(x2)
    fresh = out is None
    if fresh:
        out = torch.empty(cols, dtype=_F32, device=x2.device)
    wsb = int(_lib.load().nl_colsum_ws_bytes(rows, cols))
    ws = torch.empty(max(wsb, 16) // 4, dtype=_F32, device=x2.device)

    def run():
        _lib.call("nl_colsum_bf16", _stream(x2), rows, cols, x2.data_ptr(), _ld(x2), out.data_ptr(), 0,
                  ws.data_ptr(), wsb)
        return out

    return run() if fresh else wgrad.fork(run, x2, out, ws)


# ---------------------------------------------------------------------------
# FFN
# ---------------------------------------------------------------------------


class _FFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W1, b1, W2, b2):
        x2 = _rows(x)
        W1b, W2b = bf16_shadow(W1), bf16_shadow(W2)
        b1f, b2f = _param(b1), _param(b2)
        M, F_ = x2.shape[0], W1b.shape[1]
        u = padded_empty(M, F_, _BF16, x2.device)         # pre-activation, kept for the backward
        h = padded_empty(M, F_, _BF16, x2.device)         # gelu(u)
        gemm_raw(x2, W1b, out=h, epi=EPI_BIAS_GELU, bias=b1f, aux=u)
        y = padded_empty(M, W2b.shape[1], _BF16, x2.device)
        gemm_raw(h, W2b, out=y, epi=EPI_BIAS, bias=b2f)
        ctx.save_for_backward(x2, u, h)
        ctx.wb = (W1b, W2b)
        ctx.bufs = tuple(grad_buffer(t) for t in (W1, b1, W2, b2))
        ctx.shape = x.shape
        return y.view(*x.shape[:-1], W2b.shape[1])

    @staticmethod
    def backward(ctx, dy):
        x2, u, h = ctx.saved_tensors
        W1b, W2b = ctx.wb
        gW1, gb1, gW2, gb2 = ctx.bufs
        dy2 = _rows(dy)
        db2 = colsum(dy2, out=gb2)
        dW2 = _wgrad(h, dy2, gW2)                                                  # h^T . dy
        du = padded_empty(u.shape[0], u.shape[1], _BF16, dy2.device)
        gemm_raw(dy2, W2b, "N", "T", out=du, epi=EPI_DGELU, aux=u)               # (dy . W2^T) * gelu'(u)
        db1 = colsum(du, out=gb1)
        dW1 = _wgrad(x2, du, gW1)                                                  # x^T . du
        dx = gemm_raw(du, W1b, "N", "T", out_dtype=_BF16)                          # du . W1^T
        return dx.view(ctx.shape), *_unless_buffered(ctx.bufs, (dW1, db1, dW2, db2))


def ffn(x: torch.Tensor, W1: torch.Tensor, b1: torch.Tensor, W2: torch.Tensor, b2: torch.Tensor) -> torch.Tensor:
    """gelu_tanh(x @ W1 + b1) @ W2 + b2 in bf16 with fp32 accumulation."""
    return _FFN.apply(x, W1, b1, W2, b2)


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------


def _embedding_fwd(ids, tok, pos):
    """-> (bf16 (B, S, D) lookup, int32 ids, dims for the backward)."""
    B, S = ids.shape
    V, D = tok.shape
    if S > pos.shape[0]:
        raise ValueError(f"embedding: sequence {S} exceeds the position table ({pos.shape[0]})")
    ids32 = ids.to(torch.int32).contiguous()
    t, p = _param(tok), _param(pos)
    _check_device(ids32, t, p)
    out = torch.empty((B, S, D), dtype=_BF16, device=ids.device)
    _lib.call("nl_embedding_fwd", _stream(out), B, S, D, V, ids32.data_ptr(), t.data_ptr(), p.data_ptr(),
              out.data_ptr())
    return out, ids32, (B, S, D, V, tuple(pos.shape))


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, tok, pos):
        out, ids32, ctx.dims = _embedding_fwd(ids, tok, pos)
        ctx.save_for_backward(ids32)
        ctx.bufs = (grad_buffer(tok), grad_buffer(pos))
        return out

    @staticmethod
    def backward(ctx, dx):
        (ids32,) = ctx.saved_tensors
        return None, *_embedding_bwd(ids32, dx, ctx.dims, ctx.bufs)


def _embedding_bwd(ids32, dx, dims, bufs):
    """(dtok, dpos) of the lookup, None where a main_grad buffer took them."""
    B, S, D, V, pshape = dims
    dx = dx.to(_BF16).contiguous()
    gt, gp = bufs
    # the kernel writes every row of dtok (zero where no token has the id); of
    # dpos it writes rows [0, S), so only a longer table needs a fill (zero_()
    # is a fill kernel: no memset node when the step is captured)
    dtok = gt if gt is not None else torch.empty((V, D), dtype=_F32, device=dx.device)
    if gp is None:
        dpos = torch.zeros(pshape, dtype=_F32, device=dx.device)
    else:
        dpos = gp.zero_() if pshape[0] > S else gp
    wsb = int(_lib.load().nl_embedding_bwd_ws_bytes(B, S, D, V))
    ws = torch.empty(max(wsb, 16) // 4, dtype=torch.int32, device=dx.device)
    _lib.call("nl_embedding_bwd", _stream(dx), B, S, D, V, ids32.data_ptr(), dx.data_ptr(), dtok.data_ptr(),
              dpos.data_ptr(), 0, ws.data_ptr(), wsb)
    return _unless_buffered(bufs, (dtok, dpos))


def embedding(ids: torch.Tensor, tok: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """bf16 (B, S, D) = tok[ids] + pos[:S] for int ids (B, S)."""
    return _Embedding.apply(ids, tok, pos)


class _EmbeddingLayerNorm(torch.autograd.Function):
    """The lookup and the first block's LayerNorm as one node: the residual
    stream x and LN(x) both leave it, so in the backward the LayerNorm kernel
    adds x's other gradient (dres) while forming its own, and the lookup's
    backward reads the sum (no separate add of the two gradients)."""

    @staticmethod
    def forward(ctx, ids, tok, pos, gamma, beta, eps):
        ctx.set_materialize_grads(False)
        x, ids32, ctx.dims = _embedding_fwd(ids, tok, pos)
        x2 = x.view(-1, x.shape[-1])
        g, b = _param(gamma), _param(beta)
        y, _, mean, rstd = layer_norm_fwd_raw(x2, g, b, eps)
        ctx.save_for_backward(ids32, x2, mean, rstd, g)
        ctx.bufs = (grad_buffer(tok), grad_buffer(pos))
        ctx.ln_bufs = (grad_buffer(gamma), grad_buffer(beta))
        return y.view(x.shape), x2.view(x.shape)

    @staticmethod
    def backward(ctx, dy, dx):
        ids32, x2, mean, rstd, g = ctx.saved_tensors
        ln_grads = (None, None)
        if dy is not None:
            dx2, dg, db = layer_norm_bwd_raw(_rows(dy), x2, mean, rstd, g, _rows(dx) if dx is not None else None,
                                             *ctx.ln_bufs)
            dx = dx2
            ln_grads = _unless_buffered(ctx.ln_bufs, (dg, db))
        if dx is None:
            return None, None, None, *ln_grads, None
        return None, *_embedding_bwd(ids32, dx, ctx.dims, ctx.bufs), *ln_grads, None


def embedding_layer_norm(ids: torch.Tensor, tok: torch.Tensor, pos: torch.Tensor, gamma: torch.Tensor,
                         beta: torch.Tensor, eps: float = 1e-5):
    """(LN(x), x) with x = embedding(ids, tok, pos): the lookup and the first
    LayerNorm, whose backward also takes in x's residual-stream gradient."""
    return _EmbeddingLayerNorm.apply(ids, tok, pos, gamma, beta, eps)
