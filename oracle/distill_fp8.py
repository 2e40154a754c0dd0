"""Float64 NumPy definitions of the 8-bit block-scaled operands, of a row's top
logits and of the distillation loss. TEST INFRASTRUCTURE ONLY. The reference has
no such operators: these restate the formulas of include/nlearn_hip.h.
"""
from __future__ import annotations

import numpy as np

BLOCK = 128


def e4m3_table() -> np.ndarray:
    """The value of each of the 256 e4m3 bytes (OCP: no infinity, 0x7f and 0xff NaN)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e.astype(float) - 7))
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(b & 128, -v, v)


def e4m3_bytes(u: np.ndarray) -> np.ndarray:
    """Nearest e4m3 byte (ties to even) of |u| <= 448; NaN for a value that is not finite."""
    a = np.abs(u)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.clip(np.floor(np.log2(np.where((a > 0) & np.isfinite(a), a, 1.0))), -6, 8)
    n = np.round(np.where(np.isfinite(a), a, 0) / 2.0 ** (e - 3))      # 0..16, half to even
    up = n == 16
    e, n = np.where(up, e + 1, e), np.where(up, 8, n)
    bits = np.where(n < 8, n, ((e + 7) * 8 + n - 8)).astype(np.int64)  # below 2^-6: no implied one
    bits = np.where(np.isfinite(u), bits, 0x7f)
    return (bits | np.where(np.signbit(u) & np.isfinite(u), 128, 0)).astype(np.uint8)


def quantize(x: np.ndarray, group: int):
    """(bytes [rows, cols up to 128], scale bytes [ceil(rows/group), blocks]) of blocks along the columns."""
    x = np.asarray(x, np.float64)
    r, c = x.shape
    R, C = -(-r // group) * group, -(-c // BLOCK) * BLOCK
    p = np.zeros((R, C))
    p[:r, :c] = x
    a = np.abs(p)
    a = np.where(np.isfinite(a), a, 0).reshape(R // group, group, C // BLOCK, BLOCK).max(axis=(1, 3), initial=0)
    f, e = np.frexp(a)                       # a = f 2^e, f in [1/2, 1); 448 = 7/8 * 2^9
    e = np.where(a == 0, 0, np.clip(e - 9 + (f > 0.875), -127, 127))
    q = e4m3_bytes(p * np.repeat(np.repeat(2.0 ** -e.astype(float), group, 0), BLOCK, 1))
    return q[:r], (e + 127).astype(np.uint8)


def values(q: np.ndarray, s: np.ndarray, group: int) -> np.ndarray:
    f = np.repeat(np.repeat(2.0 ** (s.astype(float) - 127), group, 0)[:q.shape[0]], BLOCK, 1)
    return e4m3_table()[q] * f


def top(x: np.ndarray, k: int, T: float):
    """(ids [M, k], lse [M]): largest first, NaN above all, equal ones (-0 and 0 too) by the lower id."""
    x = np.asarray(x, np.float64)
    key = np.where(np.isnan(x), np.inf, x)
    ids = np.empty((x.shape[0], k), np.int64)
    for m in range(x.shape[0]):
        ids[m] = np.lexsort((np.arange(x.shape[1]), -key[m], ~np.isnan(x[m])))[:k]
    return ids, lse(x / T)


def lse(x: np.ndarray) -> np.ndarray:
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        at = np.where(np.isfinite(m), m, 0)
        return (np.log(np.exp(x - at).sum(1, keepdims=True)) + at)[:, 0]


def distill(z, ids, v, lse_t, T: float, scale: float):
    """(loss rows, dlogits, S, sum_j p_j |gap_j|) of the definition in include/nlearn_hip.h."""
    z, v = np.asarray(z, np.float64), np.asarray(v, np.float64)
    M, V = z.shape
    loss, d = np.zeros(M), np.zeros((M, V))
    mass, spread = np.zeros(M), np.zeros(M)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        logq = z / T - lse(z / T)[:, None]
        for m in range(M):
            on = ids[m] >= 0
            i, w = ids[m][on], v[m][on] / T
            if (i >= V).any():
                loss[m], d[m] = np.nan, np.nan
                continue
            if lse_t is not None:
                lp = w - lse_t[m]
            else:
                lp = w - lse(w[None])[0] if w.size and w.max() > -np.inf else w
            p = np.exp(lp)
            mass[m] = p.sum()
            if not p.size or mass[m] == 0:
                continue
            gap = np.where(p == 0, 0, lp - logq[m][i])
            loss[m] = T * T * np.where(p == 0, 0, p * gap).sum()
            spread[m] = np.abs(np.where(p == 0, 0, p * gap)).sum()
            d[m] = np.exp(logq[m]) * mass[m]
            np.subtract.at(d[m], i, p)
            d[m] *= scale * T
    return loss, d, mass, spread
