"""Performance cases of the 8-bit product and of distillation.

A student model is trained from a larger frozen teacher: products of both run in
8-bit floating point with a scale for each block of 128, the teacher's largest
logits are picked, and the student's loss and gradient follow from them.

Kinds:
  quantize  values to e4m3 with a power-of-two scale for each block of 128, along
            the rows, in both orientations, or in 128 x 128 blocks (weights)
  gemm      the product of two such operands
  linear    x W forward and backward, quantising on the way (training)
  top       the k largest logits of each row, their ids and the logsumexp
  distill   the loss against a teacher's top logits, with the logits' gradient

``run`` takes the plain form (elementary torch operations in 32 bits) while
``own`` is false and calls the framework while it is true.
"""
from __future__ import annotations

import math

import torch

own = False

_DEV = "cuda"
_BF16 = torch.bfloat16
_F32 = torch.float32
_F64 = torch.float64
_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu
_B = 128
_VOCAB = 50257


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed() -> list:
    return [
        # a few rows before a product: latency
        {"name": "quantize_rows_small", "kind": "quantize", "mode": "rows", "rows": 64, "cols": 512, "f32": False},
        # the feed-forward activations of the default batch (32 x 512), both ways, as training keeps them
        {"name": "quantize_both_ffn", "kind": "quantize", "mode": "both", "rows": 16384, "cols": 2048, "f32": False},
        # the fp32 LM-head weight of 50257 columns, laid out for the forward and the backward
        {"name": "quantize_lm_head", "kind": "quantize", "mode": "weight", "rows": 512, "cols": 50257, "f32": True},
        # a few tokens through the first feed-forward matrix
        {"name": "gemm_few_rows", "kind": "gemm", "m": 8, "n": 2048, "k": 512, "gb": 128, "f32": False},
        # the teacher's logits of the default batch
        {"name": "gemm_lm_head", "kind": "gemm", "m": 16384, "n": 50257, "k": 512, "gb": 128, "f32": False},
        # a large product of a wide model
        {"name": "gemm_large", "kind": "gemm", "m": 8192, "n": 8192, "k": 8192, "gb": 128, "f32": False},
        # the first feed-forward matrix in training, default batch
        {"name": "linear_ffn", "kind": "linear", "m": 16384, "n": 2048, "k": 512},
        # a short last batch through a matrix of odd sizes
        {"name": "linear_ragged", "kind": "linear", "m": 777, "n": 333, "k": 1000},
        # the teacher's answers for a few tokens
        {"name": "top_few_rows", "kind": "top", "m": 8, "v": 50257, "k": 8, "t": 1.0},
        # ... and for the default batch
        {"name": "top_batch", "kind": "top", "m": 16384, "v": 50257, "k": 64, "t": 2.0},
        # a small vocabulary and few rows, entries left out
        {"name": "distill_small", "kind": "distill", "m": 200, "v": 1000, "k": 16, "t": 1.0, "lse": False,
         "f32": True, "gaps": True},
        # the student's loss and gradient of the default batch
        {"name": "distill_batch", "kind": "distill", "m": 16384, "v": 50257, "k": 64, "t": 2.0, "lse": True,
         "f32": False, "gaps": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "gemm", "linear", "top", "distill"])
    if kind == "quantize":
        mode = rng.choice(["rows", "both", "weight"])
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 1, min(_VOCAB, (1 << 25) // rows))
        return {"kind": kind, "mode": mode, "rows": rows, "cols": cols, "f32": rng.random() < 0.5}
    if kind == "gemm":
        m, n = _log(rng, 1, 16384), _log(rng, 1, _VOCAB)
        k = _log(rng, 1, min(16384, (1 << 39) // (m * n)))
        return {"kind": kind, "m": m, "n": n, "k": k, "gb": rng.choice([1, 128]), "f32": rng.random() < 0.4}
    if kind == "linear":
        m, n = _log(rng, 1, 16384), _log(rng, 16, 8192)
        k = _log(rng, 16, min(8192, (1 << 37) // (m * n)))
        return {"kind": kind, "m": m, "n": n, "k": k}
    v = _log(rng, 64, 131072)
    m = _log(rng, 1, min(16384, 16384 * _VOCAB // v))
    t = rng.choice([1.0, 2.0, round(rng.uniform(0.5, 8.0), 2)])
    k = _log(rng, 1, min(256, v) if kind == "top" else min(128, v))
    if kind == "top":
        return {"kind": kind, "m": m, "v": v, "k": k, "t": t}
    return {"kind": kind, "m": m, "v": v, "k": k, "t": t, "lse": rng.random() < 0.5, "f32": rng.random() < 0.5,
            "gaps": rng.random() < 0.5}


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "quantize":
        n = c["rows"] * c["cols"]
        copies = 1 if c["mode"] == "rows" else 2
        return {"bytes": n * ((4 if c["f32"] else 2) + copies), "flops": 0}
    if c["kind"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": (m + n) * k + m * n * (4 if c["f32"] else 2), "flops": 2 * m * n * k}
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": 4 * m * k + 4 * m * n + 8 * n * k, "flops": 6 * m * n * k}
    m, v, k = c["m"], c["v"], c["k"]
    if c["kind"] == "top":
        return {"bytes": 2 * m * v + 6 * m * k + 4 * m, "flops": 0}
    return {"bytes": 4 * m * v + m * k * (8 if c["f32"] else 6) + (4 * m if c["lse"] else 0), "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _normal(g, rows, cols, std, dtype, stride=None):
    """N(0, std^2) in ``dtype``, made a slab of rows at a time."""
    x = torch.zeros((rows, stride or cols), dtype=dtype, device=_DEV)[:, :cols]
    step = max(1, (1 << 27) // cols)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x[r:r + n] = torch.randn((n, cols), generator=g, device=_DEV) * std
    return x


def _activations(g, rows, cols, dtype=_BF16):
    """Activations: rows of unlike sizes and a few columns far above the rest."""
    x = _normal(g, rows, cols, 1.0, dtype)
    x *= torch.exp2(torch.randint(-3, 4, (rows, 1), generator=g, device=_DEV)).to(dtype)
    x[:, torch.randint(0, cols, (1 + cols // 256,), generator=g, device=_DEV)] *= 32
    return x


def _as8(n):
    return (n + 7) // 8 * 8


def prepare(case: dict, seed: int) -> dict:
    c = case
    g = torch.Generator(device=_DEV).manual_seed(int(seed) * 7919 + 17)
    if c["kind"] == "quantize":
        if c["mode"] == "weight":
            x = _normal(g, c["rows"], c["cols"], 0.02, _F32 if c["f32"] else _BF16, _as8(c["cols"]))
        else:
            x = _activations(g, c["rows"], c["cols"], _F32 if c["f32"] else _BF16)
        return {"case": c, "x": x}
    if c["kind"] == "gemm":
        # operands quantised beforehand, as a frozen weight and a shared activation are
        qa, sa = _quantize(_activations(g, c["m"], c["k"]), 1)
        qb, sb = _quantize(_normal(g, c["n"], c["k"], 0.05, _F32), c["gb"])
        return {"case": c, "qa": qa, "sa": sa, "qb": qb, "sb": sb}
    if c["kind"] == "linear":
        x = _activations(g, c["m"], c["k"]).requires_grad_(True)
        W = _normal(g, c["k"], c["n"], 0.05, _F32, _as8(c["n"])).requires_grad_(True)
        return {"case": c, "x": x, "W": W, "dy": _normal(g, c["m"], c["n"], 1e-3, _BF16)}
    m, v, k = c["m"], c["v"], c["k"]
    z = _normal(g, m, v, 2.0, _BF16, _as8(v))
    if c["kind"] == "top":
        return {"case": c, "z": z}
    # the teacher's logits are the student's with some noise; k of them are kept, largest first
    ids = torch.empty((m, k), dtype=torch.int32, device=_DEV)
    values = torch.empty((m, k), dtype=_F32 if c["f32"] else _BF16, device=_DEV)
    lse = torch.empty((m,), dtype=_F32, device=_DEV)
    step = max(1, (1 << 27) // v)
    for r in range(0, m, step):
        t = z[r:r + step].float()
        t = t + torch.randn(t.shape, generator=g, device=_DEV)
        top = torch.topk(t, k, dim=1)
        ids[r:r + step], values[r:r + step] = top.indices, top.values
        lse[r:r + step] = torch.logsumexp(t / c["t"], 1)
    if c["gaps"]:
        # padding entries (-1), some rows without any entry, and an id given twice
        n = torch.randint(0, k + 1, (m, 1), generator=g, device=_DEV)
        n = torch.where(torch.rand((m, 1), generator=g, device=_DEV) < 0.5, k, n)
        if k > 1:
            ids[:, k // 2] = ids[:, 0]
        ids[torch.arange(k, device=_DEV)[None, :] >= n] = -1
    return {"case": c, "z": z.requires_grad_(True), "ids": ids, "values": values, "lse": lse if c["lse"] else None}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _blocks(x, group):
    """fp32 [rows/group, group, cols/128, 128], zero-padded."""
    r, c = x.shape
    p = torch.nn.functional.pad(x.float(), (0, -c % _B, 0, -r % group))
    return p.view(p.shape[0] // group, group, p.shape[1] // _B, _B)


def _exponents(p):
    """Least e with amax <= 448 * 2^e over groups and blocks (frexp is exact; 448 = 0.875 * 2^9)."""
    amax = p.abs().amax((1, 3))
    m, e = torch.frexp(amax)
    e = e - 9 + (m > 0.875).int()
    return torch.where(amax == 0, 0, e).clamp(-127, 127)


def _quantize(x, group):
    """(e4m3 values [rows, cols padded to 128], e8m0 scales [rows/group, cols/128]) of blocks along the columns."""
    p = _blocks(x, group)
    e = _exponents(p)
    q = (p * torch.exp2(-e.float())[:, None, :, None]).to(_E4M3)
    q = q.view(-1, p.shape[2] * _B)[:x.shape[0]]
    return q.contiguous(), (e + 127).to(torch.uint8).view(_E8M0)


def _values(q, s, group, cols):
    """The fp32 values that an operand stands for."""
    f = torch.exp2(s.view(torch.uint8).float() - 127).repeat_interleave(group, 0)[:q.shape[0]]
    return (q.float().view(q.shape[0], -1, _B) * f[:, :, None]).view(q.shape[0], -1)[:, :cols]


def _rounded(x, group=1):
    return _values(*_quantize(x, group), group, x.shape[1])


def _plain(s):
    c = s["case"]
    if c["kind"] == "quantize":
        if c["mode"] == "rows":
            return _quantize(s["x"], 1)
        group = 128 if c["mode"] == "weight" else 1
        return _quantize(s["x"], group) + _quantize(s["x"].t(), group)
    if c["kind"] == "gemm":
        a, b = _values(s["qa"], s["sa"], 1, c["k"]), _values(s["qb"], s["sb"], c["gb"], c["k"])
        return (a @ b.t()).to(_F32 if c["f32"] else _BF16)
    if c["kind"] == "linear":
        x, W, dy = s["x"].detach(), s["W"].detach(), s["dy"]
        Wq = _rounded(W, 128)
        y = _rounded(x) @ Wq
        dx = _rounded(dy) @ Wq.t()
        dW = _rounded(x.t()) @ _rounded(dy.t()).t()
        return y.to(_BF16), dx.to(_BF16), dW
    if c["kind"] == "top":
        z, v = s["z"], c["v"]
        f = z.float() / c["t"]
        m = f.amax(1, keepdim=True)
        lse = (m + (f - m).exp().sum(1, keepdim=True).log())[:, 0]
        # one integer orders by value, then by the lower id
        b = (z + 0.0).view(torch.int16).int()
        b = torch.where(b < 0, b ^ 0x7fff, b).long() * v + torch.arange(v - 1, -1, -1, device=z.device)
        ids = v - 1 - torch.remainder(torch.topk(b, c["k"], dim=1).values, v)
        return z.gather(1, ids), ids.int(), lse
    z, ids, t = s["z"].detach().float(), s["ids"].long(), c["t"]
    there = ids >= 0
    at = ids.clamp(min=0)
    m = z.amax(1, keepdim=True)
    e = ((z - m) / t).exp()
    total = e.sum(1, keepdim=True)
    # the loss is a difference of log-probabilities that may nearly cancel: the k entries in 64 bits
    lse = m.double() / t + total.double().log()
    lp = torch.where(there, s["values"].double() / t, -math.inf)
    if s["lse"] is not None:
        lp = lp - s["lse"].double()[:, None]
    else:
        top = lp.amax(1, keepdim=True).clamp(min=-1e30)
        lp = lp - top - (lp - top).exp().sum(1, keepdim=True).log()
    p = torch.where(there, lp.exp(), 0.0)
    gap = torch.where(there, lp - (z.gather(1, at).double() / t - lse), 0.0)
    loss = (p * gap).sum(1).mean() * (t * t)
    d = e * (p.sum(1, keepdim=True).float() / total)
    d.scatter_add_(1, at, -p.float())
    return loss.float(), (d * (t / z.shape[0])).to(_BF16)


def run(state: dict):
    if not own:
        with torch.no_grad():
            return _plain(state)
    s, c = state, state["case"]
    if c["kind"] == "top":
        from nlearn_amd.kernels.distill import top_logits

        return top_logits(s["z"], c["k"], temperature=c["t"])
    if c["kind"] == "distill":
        from nlearn_amd.kernels.distill import distill_cross_entropy

        loss = distill_cross_entropy(s["z"], s["ids"], s["values"], lse=s["lse"], temperature=c["t"])
        return loss, *torch.autograd.grad(loss, s["z"])
    from nlearn_amd.kernels.fp8 import Fp8Blocks, gemm_fp8, linear_fp8, quantize_fp8, quantize_fp8_both

    if c["kind"] == "quantize":
        if c["mode"] == "rows":
            a = quantize_fp8(s["x"])
            return a.q, a.scale
        a, b = quantize_fp8_both(s["x"], group=128 if c["mode"] == "weight" else 1)
        return a.q, a.scale, b.q, b.scale
    if c["kind"] == "gemm":
        a = Fp8Blocks(s["qa"], s["sa"], (c["m"], c["k"]), 1)
        b = Fp8Blocks(s["qb"], s["sb"], (c["n"], c["k"]), c["gb"])
        return gemm_fp8(a, b, out_dtype=_F32 if c["f32"] else _BF16)
    y = linear_fp8(s["x"], s["W"])
    return y, *torch.autograd.grad(y, (s["x"], s["W"]), s["dy"])


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _scaled64(x, group):
    """(e4m3 value, scale) of every element of x in float64, for blocks of 128 columns by ``group`` rows."""
    r, c = x.shape
    rows, cols = -(-r // group) * group, -(-c // _B) * _B
    p = torch.zeros((rows, cols), dtype=_F64, device=x.device)
    p[:r, :c] = x
    amax = p.abs().reshape(rows // group, group, cols // _B, _B).amax(3).amax(1)
    e = torch.ceil(torch.log2(amax / 448))
    e = torch.where(amax > 448 * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= 448 * torch.exp2(e - 1), e - 1, e)
    scale = torch.where(amax > 0, torch.exp2(e.clamp(-127, 127)), 1.0)
    u = p / scale.repeat_interleave(group, 0).repeat_interleave(_B, 1)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(u / step) * step)[:r], scale


def _exact8(x, group=1):
    q, s = _scaled64(x.double(), group)
    return (q * s.repeat_interleave(group, 0)[:x.shape[0]].repeat_interleave(_B, 1))[:, :x.shape[1]]


def exact(case: dict, seed: int):
    c, s = case, prepare(case, seed)
    with torch.no_grad():
        if c["kind"] == "quantize":
            if c["mode"] == "rows":
                return _scaled64(s["x"], 1)
            group = 128 if c["mode"] == "weight" else 1
            return _scaled64(s["x"], group) + _scaled64(s["x"].t(), group)
        if c["kind"] == "gemm":
            a = s["qa"].double() * s["sa"].double().repeat_interleave(_B, 1)
            b = s["qb"].double() * s["sb"].double().repeat_interleave(c["gb"], 0)[:c["n"]].repeat_interleave(_B, 1)
            return a @ b.t()
        if c["kind"] == "linear":
            W = _exact8(s["W"], 128)
            return (_exact8(s["x"]) @ W, _exact8(s["dy"]) @ W.t(), _exact8(s["x"].t()) @ _exact8(s["dy"].t()).t())
        m, step = c["m"], max(1, (1 << 26) // c["v"])
        if c["kind"] == "top":
            parts = []
            for r in range(0, m, step):
                z = s["z"][r:r + step].double()
                o = torch.sort(z, dim=1, descending=True, stable=True)
                parts.append((o.values[:, :c["k"]], o.indices[:, :c["k"]].int(), torch.logsumexp(z / c["t"], 1)))
            return tuple(torch.cat(p) for p in zip(*parts))
        total, grads = 0.0, []
        for r in range(0, m, step):
            z = s["z"][r:r + step].double() / c["t"]
            ids, v = s["ids"][r:r + step].long(), s["values"][r:r + step].double() / c["t"]
            logq = torch.log_softmax(z, 1)
            w = torch.where(ids >= 0, v, -math.inf)
            logp = w - (s["lse"][r:r + step].double()[:, None] if c["lse"] else torch.logsumexp(w, 1, keepdim=True))
            p = torch.where(ids >= 0, logp.exp(), 0.0)
            at = ids.clamp(min=0)
            total += float(torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0).sum())
            target = torch.zeros_like(z).scatter_add_(1, at, p)
            grads.append((c["t"] / m) * (logq.exp() * p.sum(1, keepdim=True) - target))
        return total * c["t"] ** 2 / m, torch.cat(grads)
