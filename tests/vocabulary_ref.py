"""The vocabulary operators from their definitions, in 64 bits, with bounds on a kernel's error.

Bounds: u is a type's unit roundoff (2^-24 fp32, 2^-8 bf16, 2^-11 fp16).  A sum of k fp32 terms in any
order is within k 2^-24 of the sum of their magnitudes; matrix-core sums are given twice that.
"""

from __future__ import annotations

import torch

U32 = 2.0 ** -24
ROUNDOFF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the distance of the least numbers (subnormal ones; bf16 and fp32 have them far below any value here)
TINY = {torch.float32: 1e-40, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}


def embed(tokens, table, scale):
    """(out, bound)"""
    out = table.double()[tokens.long()] * scale
    exact = torch.zeros_like(out) if scale == 1.0 else out.abs() * (ROUNDOFF[table.dtype] + 2 * U32) + TINY[table.dtype]
    return out, exact


def embed_grad(tokens, grad_out, vocab, scale, padding=None):
    """(grad, bound)"""
    tokens, up = tokens.long().reshape(-1), grad_out.double().reshape(-1, grad_out.shape[-1])
    kept = (tokens >= 0) & (tokens < vocab)
    if padding is not None:
        kept &= tokens != padding
    t, up = tokens[kept], up[kept]
    zero = torch.zeros(vocab, up.shape[1], dtype=torch.float64, device=up.device)
    grad = zero.index_add(0, t, up) * scale
    size = zero.index_add(0, t, up.abs()) * abs(scale)
    count = torch.bincount(t, minlength=vocab).double().unsqueeze(1)
    dtype = grad_out.dtype
    return grad, size * (count + 2) * U32 + grad.abs() * ROUNDOFF[dtype] + TINY[dtype]


def entropy(features, table, targets, upstream, *, ignore_index=-100, reduction="mean", logit_scale=1.0):
    """{loss, features, table} -> (value, bound); upstream: the loss's gradient (a number or one per row)."""
    dtype, vocab, dim = table.dtype, table.shape[0], table.shape[1]
    h, w = features.double().reshape(-1, dim), table.double()
    t = targets.long().reshape(-1)
    valid = t != ignore_index
    h = torch.where(valid.unsqueeze(1), h, torch.zeros_like(h))
    label = torch.where(valid, t, torch.zeros_like(t))
    n, c = h.shape[0], logit_scale
    s = c * (h @ w.T)
    lse = torch.logsumexp(s, 1)
    at = torch.arange(n, device=h.device)
    loss = torch.where(valid, lse - s[at, label], torch.zeros_like(lse))
    count = int(valid.sum())
    # a logit: the dot product's sum (six products of planes for fp32), the scale and its base-2 form
    terms = dim * (6 if dtype == torch.float32 else 1)
    s_err = (2 * (terms + 4) * U32 * abs(c) * (h.abs() @ w.abs().T)).amax(1) + s.abs().amax(1) * 4 * U32
    # the sum of exponentials (each to 2 ulp, the exponent's rounding) and the logarithm
    lse_err = s_err + (vocab + 16) * U32 + 4 * U32 * lse.abs()
    row_err = torch.where(valid, s_err + lse_err + 2 * U32 * loss.abs(), torch.zeros_like(loss))
    out = {}
    if reduction == "none":
        out["loss"] = (loss, row_err)
    else:
        k = count if reduction == "mean" else 1
        out["loss"] = (loss.sum() / k, row_err.sum() / k + 2 * U32 * loss.sum().abs() / k) if k else (loss.sum() / 0.0, loss.sum())
    g = torch.as_tensor(upstream, dtype=torch.float64, device=h.device)
    if reduction == "mean":
        g = g / max(count, 1)
    g = torch.where(valid, g.expand(n), torch.zeros(n, dtype=torch.float64, device=h.device)).unsqueeze(1)
    p = torch.exp(s - lse.unsqueeze(1))
    ds = p.clone()
    ds[at, label] -= 1.0
    # ds: the probability's relative error, and its rounding to the type that the products take
    # (for fp16 held with the largest row's g as the unit: 2^-25 / 2^15 of that at least)
    p_err = (s_err + lse_err + 16 * U32).unsqueeze(1) * p
    least = 2.0 ** -40 * g.abs().max() if dtype == torch.float16 and n else 0.0
    ds_err = torch.where(valid.unsqueeze(1), g.abs() * (p_err + ds.abs() * (ROUNDOFF[dtype] + 4 * U32)) + least,
                         torch.zeros_like(ds))
    ds = ds * g
    for name, left, err, right, k in (("features", ds, ds_err, w, vocab), ("table", ds.T, ds_err.T, h, n)):
        value = c * (left @ right)
        k = k * (6 if dtype == torch.float32 else 1)
        bound = abs(c) * ((err + left.abs() * 2 * (k + 4) * U32) @ right.abs())
        out[name] = (value, bound + value.abs() * ROUNDOFF[dtype] + TINY[dtype])
    return out


def check(got, want, what):
    value, bound = want
    got = got.detach().double().reshape(value.shape).to(value.device)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = ((got - value).abs() / bound.clamp_min(1e-300)).where(got != value, torch.zeros_like(got))
    worst = float(excess.max()) if excess.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} times the bound"
