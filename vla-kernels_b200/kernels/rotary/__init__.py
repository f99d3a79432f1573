"""Rotary positions of query / key heads on B200 (sm_100a), alone or behind a
per-head RMS norm in the same pass, with gradients.

``rotary`` and ``qk_norm_rotary`` go through ``torch.ops.vlak`` like the other
ops: CUDA only, each call one node under ``torch.compile``, launched on the
current stream. They have no counterpart in the reference, which leaves both
to the model's elementwise code. Their outputs are laid out as
``kernels.attention`` wants its q and k.

Heads are (B, M, heads, head_dim), or (tokens, heads, head_dim) for packed
tokens, in fp32, fp16 or bf16 at any strides whose last is one (anything else
is copied first); slices of a packed projection are read in place. The kernels
(vla-kernels_b200/csrc/rotary.cu) read each input once and write each output
once; angles are taken in 64 bits, so far positions keep theirs.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch

from .. import _native

SCALINGS = ("none", "linear", "ntk", "yarn")


@lru_cache(maxsize=1)
def _ext():
    _native.load_ops()

    def like(x):
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)

    def heads(q, k):
        return [like(q)] if k is None else [like(q), like(k)]

    torch.library.register_fake("vlak::rotary")(
        lambda q, k, positions, inv_freq, interleaved=False, amplitude=1.0, inverse=False:
            heads(q, k))
    torch.library.register_fake("vlak::qk_norm_rotary")(
        lambda q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False,
        amplitude=1.0: heads(q, k))
    torch.library.register_fake("vlak::qk_norm_rotary_bwd")(
        lambda grad_q, grad_k, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6,
        interleaved=False, amplitude=1.0: heads(q, k) + heads(q_weight, k_weight))
    return torch.ops.vlak


_registered = False


def _ensure_registered():
    # plain global-bool guard so Dynamo folds this branch instead of breaking
    global _registered
    if not _registered:
        _ext()
        _registered = True


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str = "none",
                       factor: float = 1.0, original_length: int | None = None,
                       slow: float = 1.0, fast: float = 32.0, device=None) -> torch.Tensor:
    """The ``inv_freq`` plan of the ops: rotary_dim / 2 float64 radians per
    position, f_i = base ** (-2 i / rotary_dim), made once and kept.

    ``scaling`` stretches them by ``factor`` for contexts longer than the
    model was trained on:
      "none"    as they are (``factor`` must be 1)
      "linear"  positions interpolated: f_i / factor
      "ntk"     the base grows to base * factor ** (d / (d - 2)), d = rotary_dim:
                the fastest pair keeps its frequency, the slowest is divided
                by ``factor``
      "yarn"    per pair, by the turns r_i = original_length f_i / 2 pi it
                makes over the trained length: f_i where r_i >= fast,
                f_i / factor where r_i <= slow, and between them blended in
                proportion (Peng et al. 2023); ``rotary_amplitude(factor)`` is
                the amplitude that goes with it
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    if scaling == "none" and factor != 1.0:
        raise ValueError("factor needs a scaling")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = torch.pow(torch.tensor(base, dtype=torch.float64), -2.0 * i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if original_length is None or not original_length > 0 or not fast > slow:
            raise ValueError("yarn scaling needs original_length, and fast above slow")
        kept = ((original_length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * kept + f / factor * (1.0 - kept)
    return f.to(device)


def rotary_amplitude(factor: float) -> float:
    """0.1 ln(factor) + 1, the amplitude of scaled contexts (1 for factor <= 1)."""
    return 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


def _packed(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.unsqueeze(0)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
           inv_freq: torch.Tensor, *, interleaved: bool = False, amplitude: float = 1.0):
    """Rotate the first 2 * len(inv_freq) entries of every head by its token's
    position; the other entries pass through.

    q (B, M, H, D) and k (B, M, H_kv, D) share the positions, int32 / int64 of
    shape (B, M), (1, M) or (M,) on the same device; packed q (T, H, D) and
    k (T, H_kv, D) take positions (T,). Pairs are (i, i + rotary_dim / 2), or
    (2i, 2i + 1) when ``interleaved``; both are multiplied by ``amplitude``.
    Differentiable in q and k, any number of times (in reverse mode only: an
    input with a forward-mode tangent is refused), not in the frequencies:
    ``inv_freq`` that requires a gradient is refused. Returns new contiguous
    tensors (q, k); with k None (keys rotated earlier, as in a cache) just q.
    """
    _ensure_registered()
    if q.dim() == 3:
        y = torch.ops.vlak.rotary(_packed(q), _packed(k), positions, inv_freq, interleaved,
                                  amplitude)
        y = [t.squeeze(0) for t in y]
    else:
        y = torch.ops.vlak.rotary(q, k, positions, inv_freq, interleaved, amplitude)
    return y[0] if k is None else (y[0], y[1])


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor,
                   k_weight: torch.Tensor | None, positions: torch.Tensor,
                   inv_freq: torch.Tensor, *, eps: float = 1e-6, interleaved: bool = False,
                   amplitude: float = 1.0):
    """``rotary`` of the RMS-normed heads, x / sqrt(mean(x^2) + eps) * weight
    over head_dim, in one pass; nothing is rounded between norm and rotation.

    q_weight and k_weight are (head_dim,), float32 or of q's dtype.
    Differentiable once, in reverse mode, in q, k and the weights (whose gradients are
    summed in 32 bits in a fixed order, so they repeat bit for bit). Shapes and
    the result are those of ``rotary``; k and k_weight are None together.
    """
    _ensure_registered()
    if q.dim() == 3:
        y = torch.ops.vlak.qk_norm_rotary(_packed(q), _packed(k), q_weight, k_weight, positions,
                                          inv_freq, eps, interleaved, amplitude)
        y = [t.squeeze(0) for t in y]
    else:
        y = torch.ops.vlak.qk_norm_rotary(q, k, q_weight, k_weight, positions, inv_freq, eps,
                                          interleaved, amplitude)
    return y[0] if k is None else (y[0], y[1])
