"""Per-head RMS norm and position rotation in float64 torch, from the formulas.

``bound`` arguments return, beside each result, the sum of the magnitudes of
the terms it is made of, from which the tests take their rounding bounds.
"""
from __future__ import annotations

import torch


def angles(positions: torch.Tensor, inv_freq: torch.Tensor) -> torch.Tensor:
    """(B, M, 1, pairs) radians, float64."""
    return positions.double()[..., None, None] * inv_freq


def turn(x, theta, amplitude=1.0, interleaved=False, inverse=False):
    """Rotate the first 2 * pairs entries of x (B, M, H, D) by theta."""
    half = theta.shape[-1]
    y = x.double().clone()
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = x.double()[..., ia], x.double()[..., ib]
    c, s = amplitude * torch.cos(theta), amplitude * torch.sin(theta)
    if inverse:
        s = -s
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y


def pair_size(x, theta, interleaved=False):
    """|a| + |b| of the pair each entry belongs to (|x| where not rotated)."""
    half = theta.shape[-1]
    y = x.double().abs().clone()
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    y[..., ia] = y[..., ib] = y[..., ia] + y[..., ib]
    return y


def rms(x, eps):
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def norm_turn_grads(g, x, w, theta, eps, amplitude=1.0, interleaved=False):
    """(dx, dw, |terms of dx|, |terms of dw|) of turn(rms(x) * w)."""
    x, w = x.double(), w.double()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    hat = x * r
    t = turn(g, theta, amplitude, interleaved, inverse=True)
    u = t * w
    dx = r * (u - hat * (u * hat).mean(-1, keepdim=True))
    terms = r * (pair_size(g, theta, interleaved) * amplitude * w.abs() +
                 hat.abs() * (pair_size(g, theta, interleaved) * amplitude * w.abs()
                              * hat.abs()).mean(-1, keepdim=True))
    dw = (t * hat).sum((0, 1, 2))
    dw_terms = (pair_size(g, theta, interleaved) * amplitude * hat.abs()).sum((0, 1, 2))
    return dx, dw, terms, dw_terms
