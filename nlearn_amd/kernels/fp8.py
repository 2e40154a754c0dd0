"""nlearn_amd.kernels.fp8 — products in 8-bit floating point with a scale for each block of 128.

* ``quantize_fp8(x)`` / ``quantize_fp8_both(x)``: a matrix to e4m3 values with one
  power-of-two scale for each block of 128 along the summed axis, per row
  (``group=1``: activations, gradients) or per 128 rows (``group=128``: weights).
* ``rms_norm_fp8(x, gamma)`` / ``add_rms_norm_fp8(x, r, gamma)``: the norm in front of a product,
  written as such an operand.
* ``gemm_fp8(a, b)``: a . b^T of two such operands, bf16 or fp32 out; with bias, activation
  and residual in its epilogue, also in 8 bits for the next product.
* ``linear_fp8(x, W)``: ``linear(x, W)`` with all three products in 8 bits: y = x W,
  dX = dY W^T and dW = X^T dY, every operand quantised along the axis that its
  product sums over. ``fp8_weight(W)`` lays a frozen weight out once.

A block's scale is the least 2^e with max|x| <= 448 * 2^e. A power of two leaves
one rounding per value (to e4m3, half a step being 2^-4 of the value) and is
applied by the matrix unit itself. The reference has no 8-bit path: this stands
beside ``linear`` (gemm.py:93-115), in whose place it can be called.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .fused import _check_rms, _dense_like, _param, _strided_rows
from .gemm import _BF16, _F32, _aligned, _check_device, _ld, grad_buffer, padded_ld

_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu
_NONE = (None, 0, None, 0)  # an output that is not wanted
BLOCK = 128
MAX_COLUMNS = ((1 << 31) - 1) // 1024  # of a product's result: 256 rows of them within 31-bit offsets
MAX_BLOCKS = (1 << 28) - 16            # of a matrix quantised by rows: a launch has fewer than 2^32 threads


def _check_sizes(what: str, *sizes: int) -> None:
    if max(sizes) >= 1 << 31:  # the products count in 32 bits
        raise ValueError(f"{what}: sizes must be less than 2^31, got {sizes}")


def _result(rows: int, cols: int, dtype, device) -> torch.Tensor:
    """An empty result with the row stride of ``padded_empty``, in one call of torch."""
    return torch.empty_strided((rows, cols), (padded_ld(cols), 1), dtype=dtype, device=device)


def _code(t: torch.Tensor) -> int:
    return _lib.NL_DTYPE_F32 if t.dtype is _F32 else _lib.NL_DTYPE_BF16


class Fp8Blocks:
    """A matrix of ``shape`` = (rows, K) in 8 bits, quantised along K.

    q:     float8_e4m3fn [rows, K rounded up to 128], unit column stride, 16-byte
           aligned rows; the columns past K are zero.
    scale: float8_e8m0fnu [ceil(rows / group), blocks of K], unit column stride.
    value[r, k] = q[r, k] * scale[r // group, k // 128].
    """

    __slots__ = ("q", "scale", "shape", "group")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, shape, group: int = 1):
        rows, K = shape
        if group != 1 and group != BLOCK:
            raise ValueError(f"Fp8Blocks: a scale holds for 1 or {BLOCK} rows, not {group}")
        kb, sr = (K + BLOCK - 1) // BLOCK, rows if group == 1 else (rows + BLOCK - 1) // BLOCK
        if q.dtype is not _E4M3 or q.shape != (rows, kb * BLOCK):
            raise ValueError(f"Fp8Blocks: q must be float8_e4m3fn of shape {(rows, kb * BLOCK)}, "
                             f"got {q.dtype} {tuple(q.shape)}")
        if scale.dtype is not _E8M0 or scale.shape != (sr, kb):
            raise ValueError(f"Fp8Blocks: scale must be float8_e8m0fnu of shape {(sr, kb)}, "
                             f"got {scale.dtype} {tuple(scale.shape)}")
        if scale.get_device() != q.get_device():
            raise ValueError("Fp8Blocks: q and scale are on different devices")
        if rows and K:
            (q0, q1), (s0, s1) = q.stride(), scale.stride()
            if q1 != 1 or (rows > 1 and q0 < kb * BLOCK) or (kb > 1 and s1 != 1) or (sr > 1 and s0 < kb):
                raise ValueError("Fp8Blocks: q and scale need a unit column stride and rows of their own")
            if q.data_ptr() % 16 or (rows > 1 and q0 % 16):
                raise ValueError("Fp8Blocks: q needs 16-byte aligned rows")
        self.q, self.scale, self.shape, self.group = q, scale, (rows, K), group

    @classmethod
    def empty(cls, rows: int, K: int, group: int, device) -> "Fp8Blocks":
        kb, sr = (K + BLOCK - 1) // BLOCK, (rows + group - 1) // group
        b = cls.__new__(cls)
        # (empty_strided takes 1.3 us where empty takes 2.1)
        b.q = torch.empty_strided((rows, kb * BLOCK), (kb * BLOCK, 1), dtype=_E4M3, device=device)
        # scale rows padded to whole dwords: the product reads four blocks at a time
        ld = (kb + 3) // 4 * 4
        s = torch.empty_strided((sr, ld), (ld, 1), dtype=_E8M0, device=device)
        b.scale = s if ld == kb else s[:, :kb]
        b.shape, b.group = (rows, K), group
        return b

    def _abi(self):
        """(q, ldq, scale, lds) as the C entry points take them."""
        return self.q.data_ptr(), _row_stride(self.q), self.scale.data_ptr(), _row_stride(self.scale)

    def dequantize(self) -> torch.Tensor:
        """The fp32 values (a plain torch expression, for checks and inspection)."""
        rows, K = self.shape
        s = self.scale.float().repeat_interleave(self.group, 0)[:rows]
        return (self.q.float().view(rows, -1, BLOCK) * s[:, :, None]).view(rows, -1)[:, :K]


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _quantize(x, group: int, along: bool, across: bool):
    """(x in 8 bits or None, x^T in 8 bits or None), one launch."""
    if group != 1 and group != BLOCK:
        raise ValueError(f"quantize_fp8: a scale holds for 1 or {BLOCK} rows, not {group}")
    if x.dim() != 2:
        raise ValueError(f"quantize_fp8: expected a 2-D tensor, got shape {tuple(x.shape)}")
    f32 = x.dtype is _F32
    if not f32 and x.dtype is not _BF16:
        raise ValueError(f"quantize_fp8: x must be bfloat16 or float32, got {x.dtype}")
    _check_device(x)
    (rows, cols), (s0, s1) = x.shape, x.stride()
    if (cols > 1 and s1 != 1) or (rows > 1 and s0 < cols):  # a transposed view, rows that share memory
        x = x.detach().contiguous()
        s0 = cols
    dev = x.device
    a = Fp8Blocks.empty(rows, cols, group, dev) if along else None
    t = Fp8Blocks.empty(cols, rows, group, dev) if across else None
    if rows and cols:
        _lib.call_on(x, "nl_quantize_fp8", rows, cols, x.data_ptr(), 0 if f32 else 1, s0 if rows > 1 else cols, group,
                     *(a._abi() if along else _NONE), *(t._abi() if across else _NONE))
    return a, t


def quantize_fp8(x: torch.Tensor, group: int = 1, transpose: bool = False) -> Fp8Blocks:
    """x (R, C), bf16 or fp32, quantised along its columns; with ``transpose`` x^T
    (C, R), quantised along the rows of x. One scale for each block of 128 and
    each ``group`` rows of the result. Values that are not finite become NaN and
    have no part in the scales. Not differentiable (``linear_fp8`` is)."""
    a, t = _quantize(x, group, not transpose, transpose)
    return t if transpose else a


def quantize_fp8_both(x: torch.Tensor, group: int = 1):
    """(quantize_fp8(x), quantize_fp8(x, transpose=True)) from one read of x."""
    return _quantize(x, group, True, True)


def _rms_norm_fp8(what: str, x, r, gamma, eps):
    eps = _check_rms(what, x, r, gamma, eps)
    (x2, ldx), g = _strided_rows(x), _param(gamma)
    rows, D = x2.shape
    out = Fp8Blocks.empty(rows, D, 1, x.device)
    s = _dense_like(x) if r is not None else None
    if rows:
        r2, ldr = _strided_rows(r) if r is not None else (None, 0)
        _lib.call_on(x2, "nl_rms_norm_fp8", rows, D, _code(x2), x2.data_ptr(), ldx,
                     r2.data_ptr() if r is not None else None, ldr, s.data_ptr() if r is not None else None, D,
                     g.data_ptr(), eps, *out._abi())
    return out, s


def rms_norm_fp8(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5) -> Fp8Blocks:
    """``rms_norm(x, gamma, eps)`` quantised along its last dimension (one scale for each block
    of 128 and row; leading dimensions are flattened), from fp32 values that were not rounded to
    x's dtype before. What ``gemm_fp8`` reads; not differentiable, as ``quantize_fp8``."""
    return _rms_norm_fp8("rms_norm_fp8", x, None, gamma, eps)[0]


def add_rms_norm_fp8(x: torch.Tensor, r: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5):
    """(rms_norm_fp8(s, gamma, eps), s) with s = x + r rounded to their dtype, in one pass."""
    return _rms_norm_fp8("add_rms_norm_fp8", x, r, gamma, eps)


def gemm_fp8_ws(a: Fp8Blocks, b: Fp8Blocks) -> torch.Tensor | None:
    """The workspace gemm_fp8 would allocate for this product (or None)."""
    wsb = _lib.load().nl_gemm_fp8_ws_bytes(a.shape[0], b.shape[0], a.shape[1])
    return torch.empty(wsb // 4, dtype=_F32, device=a.q.device) if wsb else None


ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}  # NL_ACT_*; gelu in the tanh form of ``ffn``


def _act_code(what: str, activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {', '.join(map(repr, ACTIVATIONS))}, got {activation!r}")
    return ACTIVATIONS[activation]


def _check_bias(what: str, bias, N: int, like: torch.Tensor):
    if bias.shape != (N,) or bias.dtype not in (_F32, _BF16) or bias.get_device() != like.get_device():
        raise ValueError(f"{what}: bias must be float32 or bfloat16 of shape {(N,)} on {like.device}, got {bias.dtype} "
                         f"{tuple(bias.shape)} on {bias.device}")


def _whole_rows(rows: int, cols: int, dtype, device) -> torch.Tensor:
    """``_result`` whose last row, too, holds ``cols`` rounded up to 8 elements."""
    if cols % 8 == 0:
        return _result(rows, cols, dtype, device)
    # a tensor of its own over that storage: as a view it could not be written in place behind an autograd Function
    ld = padded_ld(cols)
    base = torch.empty_strided((rows, ld), (ld, 1), dtype=dtype, device=device)
    return base.new_empty((0,)).set_(base.untyped_storage(), 0, (rows, cols), (ld, 1))


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t with 16-byte aligned rows that all hold their length rounded up to 8; copies only if it must."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or cols == 1) and (rows <= 1 or s0 >= cols) and t.data_ptr() % 16 == 0 and (rows <= 1 or s0 % 8 == 0):
        need = t.storage_offset() + max(rows - 1, 0) * s0 + (cols + 7) // 8 * 8
        if cols % 8 == 0 or need * t.element_size() <= t.untyped_storage().nbytes():
            return t
    out = _whole_rows(rows, cols, t.dtype, t.device)
    out.copy_(t)
    return out


def _vector(t):
    """(address, type) of a bias or its gradient."""
    return (None, 0) if t is None else (t.data_ptr(), 0 if t.dtype is _F32 else 1)


def _dense_vector(bias):
    """bias with unit stride; copies only if it must."""
    return bias if bias is None or bias.is_contiguous() else bias.detach().contiguous()


def _bytes(n: int, device) -> torch.Tensor:
    return torch.empty_strided((n,), (1,), dtype=torch.uint8, device=device)


def _fused_product(a: Fp8Blocks, b: Fp8Blocks, out, ws, bias, act: int, residual, round_u: bool, u) -> None:
    """nl_gemm_fp8_fused into ``out``, a tensor whose rows hold N rounded up to 8 or an Fp8Blocks."""
    (M, K), N = a.shape, b.shape[0]
    if ws is None:
        ws = gemm_fp8_ws(a, b)
    qa, lda, sa, ldsa = a._abi()
    qb, ldb, sb, ldsb = b._abi()
    if isinstance(out, Fp8Blocks):
        c, ldc, sc, ldsc = out._abi()
        code = _lib.NL_DTYPE_E4M3
    else:
        c, ldc, sc, ldsc = out.data_ptr(), _ld(out), None, 0
        code = _code(out)
    _lib.call_on(a.q, "nl_gemm_fp8_fused", M, N, K, qa, lda, sa, ldsa, a.group, qb, ldb, sb, ldsb, b.group,
                 *_vector(bias), act, residual.data_ptr() if residual is not None else None,
                 _ld(residual) if residual is not None else 0, round_u, u.data_ptr() if u is not None else None,
                 u.stride(0) if u is not None else 0, c, code, ldc, sc, ldsc,
                 ws.data_ptr() if ws is not None else None, ws.numel() * ws.element_size() if ws is not None else 0)


def _gemm_fp8_fused(a, b, out_dtype, out, ws, bias, activation, residual):
    (M, _), N = a.shape, b.shape[0]
    act = _act_code("gemm_fp8", activation)
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in (_F32, _BF16, _E4M3) or (out is not None and out_dtype is _E4M3):
        raise ValueError("gemm_fp8: a result is float32, bfloat16 or (a new one) float8_e4m3fn, got "
                         f"{out_dtype}")
    dt = _BF16 if out_dtype is _E4M3 else out_dtype
    if bias is not None:
        _check_bias("gemm_fp8", bias, N, a.q)
        bias = _dense_vector(bias)
    if residual is not None and (residual.dtype is not dt or tuple(residual.shape) != (M, N)
                                 or residual.get_device() != a.q.get_device()):
        raise ValueError(f"gemm_fp8: the residual must be {dt} of shape {(M, N)} on {a.q.device}, got "
                         f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
    if out is not None:
        _ld(out)  # refuses rows that overlap
    if ws is not None and (ws.get_device() != a.q.get_device() or not ws.is_contiguous()):
        raise ValueError(f"gemm_fp8: the workspace must be contiguous and on {a.q.device}")
    if out_dtype is _E4M3:
        into = Fp8Blocks.empty(M, N, 1, a.q.device)
    elif out is not None and N % 8 == 0:
        into = out
    else:  # (rows of the caller's own are not written past N)
        into = _whole_rows(M, N, out_dtype, a.q.device)
    if M and N:
        residual = _readable(residual.detach()) if residual is not None else None
        _fused_product(a, b, into, ws, bias, act, residual, False, None)
    return into if out is None else out if into is out else out.copy_(into)


def gemm_fp8(a: Fp8Blocks, b: Fp8Blocks, out_dtype=_BF16, out: torch.Tensor | None = None,
             ws: torch.Tensor | None = None, bias: torch.Tensor | None = None, activation: str | None = None,
             residual: torch.Tensor | None = None):
    """act(a (M, K) . b (N, K)^T + bias) + residual -> (M, N) on the current stream. An fp32
    result is summed in fp32 (scale bytes 3 to 246). A bf16 result is summed by the 8-bit matrix
    instruction, which cuts 8 products at a time to 2^-13 of the largest of them: beside a bf16
    rounding that does not count, unless products cancel to a small part of their size.

    bias (N,) fp32 or bf16, activation "relu", "gelu" (tanh form) or "silu" and residual (M, N) in
    the result's dtype are applied in fp32 behind the sum. ``out_dtype=torch.float8_e4m3fn`` gives
    ``Fp8Blocks``, quantised along N, for the next product (a bf16 residual). It is summed as bf16
    is, which leaves about one value in 1000 a step beside that of fp32 sums; where that matters,
    quantise an fp32 result with ``quantize_fp8``. Not differentiable (``linear_fp8`` is).

    out: fp32 or bf16 with 16-byte aligned rows (it may be the residual). ws: as ``gemm_fp8_ws`` gives
    it (allocated here if None; too small a one is not used and K is summed in one piece)."""
    (M, K), (N, Kb) = a.shape, b.shape
    if K != Kb:
        raise ValueError(f"gemm_fp8: inner dimensions differ ({K} vs {Kb})")
    _check_sizes("gemm_fp8", M, N, K)
    _check_device(a.q, b.q)
    if a.q.get_device() != b.q.get_device():
        raise ValueError(f"gemm_fp8: operands on {a.q.device} and {b.q.device}")
    if bias is not None or activation is not None or residual is not None or out_dtype is _E4M3:
        if out is not None and (tuple(out.shape) != (M, N) or out.device != a.q.device):
            raise ValueError(f"gemm_fp8: output must be of shape {(M, N)} on {a.q.device}")
        return _gemm_fp8_fused(a, b, out_dtype, out, ws, bias, activation, residual)
    if out is None:
        if out_dtype is not _F32 and out_dtype is not _BF16:
            raise ValueError("gemm_fp8: output must be float32 or bfloat16")
        out = _result(M, N, out_dtype, a.q.device)
    elif out.dtype not in (_F32, _BF16) or tuple(out.shape) != (M, N) or out.device != a.q.device:
        raise ValueError(f"gemm_fp8: output must be float32 or bfloat16 of shape {(M, N)} on {a.q.device}")
    if M == 0 or N == 0:
        return out
    if ws is None:
        ws = gemm_fp8_ws(a, b)
    elif ws.get_device() != a.q.get_device() or not ws.is_contiguous():
        raise ValueError(f"gemm_fp8: the workspace must be contiguous and on {a.q.device}")
    qa, lda, sa, ldsa = a._abi()
    qb, ldb, sb, ldsb = b._abi()
    _lib.call_on(a.q, "nl_gemm_fp8", M, N, K, qa, lda, sa, ldsa, a.group, qb, ldb, sb, ldsb, b.group,
                 out.data_ptr(), _lib.NL_DTYPE_F32 if out.dtype is _F32 else _lib.NL_DTYPE_BF16, _ld(out),
                 ws.data_ptr() if ws is not None else None, ws.numel() * ws.element_size() if ws is not None else 0)
    return out


class Fp8Weight:
    """A weight W (K, N) in 8 bits with a scale for each 128 x 128 block, laid out
    for both products that read it: ``fwd`` is W^T (N, K), ``bwd`` W (K, N), the
    same values."""

    __slots__ = ("fwd", "bwd", "shape")

    def __init__(self, fwd: Fp8Blocks, bwd: Fp8Blocks):
        if fwd.shape != bwd.shape[::-1]:
            raise ValueError(f"Fp8Weight: {fwd.shape} is not the transpose of {bwd.shape}")
        self.fwd, self.bwd, self.shape = fwd, bwd, bwd.shape


def fp8_weight(W: torch.Tensor) -> Fp8Weight:
    """W (K, N) quantised once, for a weight that stays as it is (a frozen teacher's)."""
    bwd, fwd = quantize_fp8_both(W, group=BLOCK)
    return Fp8Weight(fwd, bwd)


@functools.lru_cache(maxsize=1024)
def _linear_bytes(M: int, K: int, N: int, need_dx: bool, need_dW: bool):
    """(saved, forward workspace, backward workspace) of one linear, in bytes."""
    lib = _lib.load()
    return (lib.nl_linear_fp8_saved_bytes(M, K, N, need_dx, need_dW),
            lib.nl_linear_fp8_ws_bytes(M, K, N, 0, need_dx, need_dW),
            lib.nl_linear_fp8_ws_bytes(M, K, N, 1, need_dx, need_dW))


def _rows(t: torch.Tensor):
    """t as the quantiser reads it, and its row stride."""
    (rows, cols), (s0, s1) = t.shape, t.stride()
    if (cols > 1 and s1 != 1) or (rows > 1 and s0 < cols):
        return t.detach().contiguous(), cols
    return t, s0 if rows > 1 else cols


def _main_grad(W: torch.Tensor):
    """W's gradient buffer (or None), which the product is written into as an array of W's shape."""
    mg = grad_buffer(W)
    if mg is not None and (mg.shape != W.shape or mg.device != W.device):
        raise ValueError(f"linear_fp8: main_grad {tuple(mg.shape)} on {mg.device} is not laid out like the weight "
                         f"{tuple(W.shape)} on {W.device}")
    return mg


class _LinearFp8(torch.autograd.Function):
    """Both directions are one call of the library each: the host's share of a small
    product is what it costs (20 us against 42 for a forward pass call by call)."""

    @staticmethod
    def forward(ctx, x2, W, need_dx, need_dW):
        ctx.need = need_dx, need_dW
        (M, K), N = x2.shape, W.shape[1]
        ctx.sizes = (M, K, N, x2.dtype, W.dtype, W.is_contiguous())
        # for its main_grad alone, so not by a saved tensor, which a hook or a checkpoint hands back as another object
        ctx.W = W if need_dW and (W.is_leaf or grad_buffer(W) is not None) else None
        y = _result(M, N, x2.dtype, x2.device)
        if M == 0 or K == 0 or N == 0:
            ctx.save_for_backward(None)
            return y.zero_()
        saved_bytes, wsb, _ = _linear_bytes(M, K, N, need_dx, need_dW)
        saved = torch.empty(saved_bytes, dtype=torch.uint8, device=x2.device)
        # with autograd, which frees it after the backward pass and shows it to hooks and checkpoints
        ctx.save_for_backward(saved)
        ws = torch.empty(wsb, dtype=torch.uint8, device=x2.device)
        (x2, ldx), (Wr, ldw) = _rows(x2), _rows(W)
        _lib.call_on(x2, "nl_linear_fp8_fwd", M, K, N, x2.data_ptr(), _code(x2), ldx, Wr.data_ptr(), _code(Wr), ldw,
                     y.data_ptr(), _code(y), _ld(y), need_dx, need_dW, saved.data_ptr(), saved_bytes,
                     ws.data_ptr(), wsb)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (saved,) = ctx.saved_tensors
        need_dx, need_dW = ctx.need
        M, K, N, x_dtype, w_dtype, w_dense = ctx.sizes
        mg = _main_grad(ctx.W) if ctx.W is not None else None
        dev = dy.device
        dx = _result(M, K, x_dtype, dev) if need_dx else None                  # dY . W^T
        # X^T . dY, straight into main_grad where its rows are aligned for the product's stores
        direct = mg is not None and mg.dtype in (_BF16, _F32) and _aligned(mg)
        dW = None
        if direct:
            dW = mg
        elif mg is None and need_dW and w_dense and N % 8 == 0:
            # laid out like W: autograd keeps it as W.grad without a copy
            dW = torch.empty((K, N), dtype=w_dtype, device=dev)
        elif need_dW:
            dW = _result(K, N, w_dtype if mg is None else _F32, dev)
        if M == 0 or K == 0 or N == 0:
            for t in (dx, mg if mg is not None else dW):
                if t is not None:
                    t.zero_()
            return dx, dW if mg is None else None, None, None
        dy, lddy = _rows(dy if dy.dtype in (_BF16, _F32) else dy.to(_F32))
        saved_bytes, _, wsb = _linear_bytes(M, K, N, need_dx, need_dW)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
        _lib.call_on(dy, "nl_linear_fp8_bwd", M, K, N, dy.data_ptr(), _code(dy), lddy, saved.data_ptr(), saved_bytes,
                     need_dx, need_dW,
                     *((dx.data_ptr(), _code(dx), _ld(dx)) if need_dx else (None, 0, 0)),
                     *((dW.data_ptr(), _code(dW), _ld(dW)) if need_dW else (None, 0, 0)), ws.data_ptr(), wsb)
        if mg is None:
            return dx, dW, None, None
        if not direct:
            mg.copy_(dW)
        return dx, None, None, None


class _LinearFp8Frozen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, W):
        ctx.W, ctx.x_dtype = W, x2.dtype
        return gemm_fp8(_quantize(x2, 1, True, False)[0], W.fwd, x2.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy.dtype not in (_BF16, _F32):
            dy = dy.to(_F32)
        return gemm_fp8(_quantize(dy, 1, True, False)[0], ctx.W.bwd, ctx.x_dtype), None      # dY . W^T


@functools.lru_cache(maxsize=1024)
def _linear_fused_bytes(M: int, K: int, N: int, need_dx: bool, need_dW: bool, need_db: bool):
    lib = _lib.load()
    return (lib.nl_linear_fp8_saved_bytes(M, K, N, need_dx, need_dW),
            lib.nl_linear_fp8_fused_ws_bytes(M, K, N, 0, need_dx, need_dW, need_db),
            lib.nl_linear_fp8_fused_ws_bytes(M, K, N, 1, need_dx, need_dW, need_db))


def _bias_grad(bias: torch.Tensor):
    """(what dbias is written to, whether that is bias's main_grad)."""
    mg = grad_buffer(bias)
    if mg is None:
        return torch.empty_strided(bias.shape, (1,), dtype=bias.dtype, device=bias.device), False
    if mg.shape != bias.shape or mg.device != bias.device or mg.dtype not in (_F32, _BF16) or not mg.is_contiguous():
        raise ValueError(f"linear_fp8: the bias's main_grad must be a dense tensor of shape {tuple(bias.shape)} on "
                         f"{bias.device}")
    return mg, True


class _LinearFp8Fused(torch.autograd.Function):
    """act(x W + bias) + residual, W a tensor or (``frozen``) an Fp8Weight; each direction is one
    call of the library, or for a frozen weight a quantisation and a product."""

    @staticmethod
    def forward(ctx, x2, W, bias, res2, frozen, act, need):
        (M, K), N = x2.shape, (W if frozen is None else frozen).shape[1]
        need_dx, need_dW, need_db, _ = need
        ctx.sizes, ctx.need, ctx.act, ctx.frozen = (M, K, N, x2.dtype), need, act, frozen
        # for their main_grad alone
        ctx.W = W if need_dW and (W.is_leaf or grad_buffer(W) is not None) else None
        ctx.w_like = None if W is None else (W.dtype, W.is_contiguous())
        ctx.bias = bias if need_db else None
        dev = x2.device
        y = _whole_rows(M, N, x2.dtype, dev)
        # what act'(u) is formed from, in the dtype of y as the activation itself sees it
        u = _whole_rows(M, N, x2.dtype, dev) if act and (need_dx or need_dW or need_db) else None
        saved = None
        if M and N:
            bias = _dense_vector(bias)
            r = _readable(res2) if res2 is not None else None
            if frozen is not None:
                _fused_product(_quantize(x2, 1, True, False)[0], frozen.fwd, y, None, bias, act, r, bool(act), u)
            elif K == 0:  # no product to quantise for
                none = Fp8Blocks.empty
                _fused_product(none(M, 0, 1, dev), none(N, 0, BLOCK, dev), y, None, bias, act, r, bool(act), u)
            else:
                saved_bytes, wsb, _ = _linear_fused_bytes(M, K, N, need_dx, need_dW, need_db)
                saved, ws = _bytes(saved_bytes, dev), _bytes(wsb, dev)
                (x2, ldx), (Wr, ldw) = _rows(x2), _rows(W)
                _lib.call_on(x2, "nl_linear_fp8_fused_fwd", M, K, N, x2.data_ptr(), _code(x2), ldx, Wr.data_ptr(),
                             _code(Wr), ldw, *_vector(bias), act, r.data_ptr() if r is not None else None,
                             _ld(r) if r is not None else 0, u.data_ptr() if u is not None else None,
                             u.stride(0) if u is not None else 0, y.data_ptr(), _code(y), y.stride(0), need_dx, need_dW,
                             saved.data_ptr(), saved_bytes, ws.data_ptr(), wsb)
        ctx.save_for_backward(saved, u)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        saved, u = ctx.saved_tensors
        M, K, N, x_dtype = ctx.sizes
        need_dx, need_dW, need_db, need_dr = ctx.need
        act, frozen = ctx.act, ctx.frozen
        if dy.dtype is not x_dtype:
            dy = dy.to(x_dtype)
        dr = dy if need_dr else None   # (the residual has x's dtype)
        if not (need_dx or need_dW or need_db):
            return None, None, None, dr, None, None, None
        dev = dy.device
        mg = _main_grad(ctx.W) if ctx.W is not None else None
        db, db_taken = _bias_grad(ctx.bias) if need_db else (None, False)
        dx = _result(M, K, x_dtype, dev) if need_dx else None
        direct = mg is not None and mg.dtype in (_BF16, _F32) and _aligned(mg)
        dW = None
        if need_dW:
            w_dtype, w_dense = ctx.w_like
            if direct:
                dW = mg
            elif mg is None and w_dense and N % 8 == 0:
                # laid out like W: kept as W.grad without a copy
                dW = torch.empty_strided((K, N), (N, 1), dtype=w_dtype, device=dev)
            else:
                dW = _result(K, N, w_dtype if mg is None else _F32, dev)
        if M == 0 or N == 0:
            for t in (dx, dW, db):
                if t is not None:
                    t.zero_()
        else:
            dy2, lddy = _rows(dy)
            up, ldu = (u.data_ptr(), u.stride(0)) if u is not None else (None, 0)
            dbp = _vector(db)
            if frozen is not None or K == 0:
                want_dx = need_dx and K > 0
                q = Fp8Blocks.empty(M, N, 1, dev) if want_dx else None
                wsb = _lib.load().nl_quantize_fp8_dact_ws_bytes(M, N) if need_db else 0
                ws = _bytes(wsb, dev) if wsb else None
                if want_dx or need_db:
                    _lib.call_on(dy2, "nl_quantize_fp8_dact", M, N, dy2.data_ptr(), _code(dy2), lddy, up, ldu, act,
                                 *(q._abi() if want_dx else _NONE), *_NONE, *dbp, ws.data_ptr() if wsb else None, wsb)
                if want_dx:
                    dx = gemm_fp8(q, frozen.bwd, x_dtype, out=dx)                           # dU . W^T
                if need_dW:
                    dW.zero_()  # of no rows
            else:
                saved_bytes, _, wsb = _linear_fused_bytes(M, K, N, need_dx, need_dW, need_db)
                ws = _bytes(wsb, dev)
                _lib.call_on(dy2, "nl_linear_fp8_fused_bwd", M, K, N, dy2.data_ptr(), _code(dy2), lddy, up, ldu, act, *dbp,
                             saved.data_ptr(), saved_bytes, need_dx, need_dW,
                             *((dx.data_ptr(), _code(dx), dx.stride(0)) if need_dx else (None, 0, 0)),
                             *((dW.data_ptr(), _code(dW), _ld(dW)) if need_dW else (None, 0, 0)), ws.data_ptr(), wsb)
        if mg is not None:
            if not direct:
                mg.copy_(dW)
            dW = None
        return dx, dW, None if db_taken else db, dr, None, None, None


def linear_fp8(x: torch.Tensor, W, bias: torch.Tensor | None = None, activation: str | None = None,
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """act(x[..., K] @ W[K, N] + bias) + residual -> [..., N] in x's dtype, with 8-bit products (as
    ``gemm_fp8`` sums them for that dtype; dW's go by W's, or by main_grad's).

    W: an fp32 or bf16 weight, quantised here, or an ``Fp8Weight`` (frozen: it gets
    no gradient). The gradients are those of the product of the quantised
    operands, with the output's gradient quantised too and the rounding taken as the identity. Both run
    on the current stream: dW is not forked within ``overlap_weight_grads()``.

    bias (N,) fp32 or bf16, activation "relu", "gelu" (tanh form) or "silu", residual [..., N] in x's
    dtype: in the product's epilogue. With an activation u = x W + bias is rounded to x's dtype before
    it, as ``ffn`` does it: that u is kept for the backward, which quantises dY act'(u). In front of relu u is
    summed in fp32 whatever x's dtype (scale bytes 3 to 246): its sign decides what a gradient passes. The
    output is the same where no gradient is wanted."""
    if x.dim() < 2:
        raise ValueError("linear_fp8: x needs >= 2 dims")
    frozen = W if isinstance(W, Fp8Weight) else None
    if frozen is None and W.dim() != 2:
        raise ValueError("linear_fp8: W needs exactly 2 dims")
    if x.shape[-1] != W.shape[0]:
        raise ValueError(f"linear_fp8: x has {x.shape[-1]} features, W has {W.shape[0]} rows")
    if x.dtype not in (_BF16, _F32):
        raise ValueError(f"linear_fp8: x must be bfloat16 or float32, got {x.dtype}")
    N = W.shape[1]
    act = _act_code("linear_fp8", activation)
    if bias is not None:
        _check_bias("linear_fp8", bias, N, x)
    if residual is not None and (residual.dtype is not x.dtype or residual.shape != (*x.shape[:-1], N)
                                 or residual.get_device() != x.get_device()):
        raise ValueError(f"linear_fp8: the residual must be {x.dtype} of shape {(*x.shape[:-1], N)} on {x.device}, got "
                         f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
    fused = bias is not None or act or residual is not None
    lead = x.shape[:-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    _check_sizes("linear_fp8", *x2.shape, N)
    grads = torch.is_grad_enabled()
    if bias is not None and grads and bias.requires_grad:
        if (x2.shape[0] + BLOCK - 1) // BLOCK * ((N + BLOCK - 1) // BLOCK) >= 1 << 23:
            raise ValueError(f"linear_fp8: no bias gradient over ({x2.shape[0]}, {N}): 2^23 tiles of 128 x 128 and more")
    if frozen is not None:
        if x2.requires_grad and grads:  # what the product of dY would refuse
            M, (K, N) = x2.shape[0], W.shape
            if K > MAX_COLUMNS - BLOCK or M * ((N + BLOCK - 1) // BLOCK) > MAX_BLOCKS:
                raise ValueError(f"linear_fp8: no input gradient of ({M}, {K}) from an output gradient of ({M}, {N})")
        if not fused:
            y = _LinearFp8Frozen.apply(x2, frozen)
        else:
            _check_device(x2, frozen.fwd.q)
            if x2.get_device() != frozen.fwd.q.get_device():
                raise ValueError(f"linear_fp8: x on {x.device}, W on {frozen.fwd.q.device}")
    else:
        if W.dtype not in (_BF16, _F32):
            raise ValueError(f"linear_fp8: W must be bfloat16 or float32, got {W.dtype}")
        _check_device(x2, W)
        if x2.get_device() != W.get_device():
            raise ValueError(f"linear_fp8: x on {x.device}, W on {W.device}")
        if not fused:
            y = _LinearFp8.apply(x2, W, grads and x2.requires_grad, grads and W.requires_grad)
    if fused:
        res2 = None if residual is None else residual if x.dim() == 2 else residual.reshape(x2.shape[0], N)
        need = tuple(grads and t is not None and t.requires_grad for t in (x2, None if frozen else W, bias, res2))
        y = _LinearFp8Fused.apply(x2, None if frozen else W, bias, res2, frozen, act, need)
    return y if x.dim() == 2 else y.reshape(*lead, N)
