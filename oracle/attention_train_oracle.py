"""GQA attention and its gradients in float64 torch, with bounds on what the
bf16 kernels may differ by.

Bounds, u = 2^-8 (half a bf16 step) and f = 2^-13 (what the 32-bit parts may
add relative to a term: scores of 64 products, the exponential, sums):
  o   u |o| + (u + f) sum P |v|        output; P
  D   f sum |do| (|o| + sum P |v|) + u sum |do| sum P |v|: of o only the rounding of P
  dS  u |dS| + P err(D) + f P (sum |do| |v| + |D|)
  dv  u |dv| + (u + f) sum P |do|
  dq  u |dq| + scale sum err(dS) |k|
  dk  u |dk| + scale sum err(dS) |q|
"""
from __future__ import annotations

import torch

U, F = 2.0 ** -8, 2.0 ** -13


def analytic(M, N, P, ds=0, de=0, device="cuda"):
    r = torch.arange(M, device=device)[:, None]
    c = torch.arange(N, device=device)
    return torch.where(c < P, (c < ds) | (c >= de), c <= N - M + r)[None]


def by_length(M, N, lengths):
    r = torch.arange(M, device=lengths.device)[:, None]
    c = torch.arange(N, device=lengths.device)
    L = lengths.clamp(0, N)[:, None, None]
    return (c < L) & (r < L)


def train(q, k, v, do, seen, scale=0.125):
    """q, do (B, M, H, 64), k, v (B, N, Hkv, 64), seen (B or 1, M, N) bool.
    Returns {name: (value, bound)} for o, dq, dk, dv, and lse (log2 units)."""
    B, M, H, _ = q.shape
    N, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    q, do = (x.double().transpose(1, 2) for x in (q, do))
    k, v = (x.double().transpose(1, 2).repeat_interleave(G, 1) for x in (k, v))
    s = scale * q @ k.transpose(2, 3)
    s = s.masked_fill(~seen[:, None], float("-inf"))
    lse = torch.logsumexp(s, -1) if N else torch.full(s.shape[:3], float("-inf"), device=s.device)
    p = torch.exp(s - lse.clamp_min(-1e300)[..., None])
    p = torch.where(seen[:, None], p, 0.0)
    o = p @ v
    err_o = U * o.abs() + (U + F) * (p @ v.abs())
    dv, err_dv = p.transpose(2, 3) @ do, p.transpose(2, 3) @ do.abs()
    dp = do @ v.transpose(2, 3)
    D = (do * o).sum(-1, keepdim=True)
    err_D = (do.abs() * (F * o.abs() + (U + F) * (p @ v.abs()))).sum(-1, keepdim=True)
    ds = p * (dp - D)
    err_ds = U * ds.abs() + p * (err_D + F * (do.abs() @ v.abs().transpose(2, 3) + D.abs()))
    dq, dk = scale * ds @ k, scale * ds.transpose(2, 3) @ q
    err_dq = U * dq.abs() + scale * err_ds @ k.abs()
    err_dk = scale * err_ds.transpose(2, 3) @ q.abs()

    def kv(x):
        return x.view(B, Hkv, G, N, 64).sum(2).transpose(1, 2)

    dk, dv = kv(dk), kv(dv)
    return {"o": (o.transpose(1, 2), err_o.transpose(1, 2)),
            "dq": (dq.transpose(1, 2), err_dq.transpose(1, 2)),
            "dk": (dk, U * dk.abs() + kv(err_dk)),
            "dv": (dv, U * dv.abs() + (U + F) * kv(err_dv)),
            "lse": (lse.transpose(1, 2) / 0.6931471805599453, None)}
