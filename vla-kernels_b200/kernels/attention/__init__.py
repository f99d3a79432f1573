"""GQA-native fused attention on B200 (sm_100a) behind ``torch.ops.vlak``.

Same API as the reference module (kernels/attention/__init__.py):
``fused_attention`` (the (B, H, M, 64) op with a bool or analytic mask),
``fused_attention_gqa`` and ``fused_attention_gqa_v4`` with their fake (meta)
implementations and register guards, so ``vla/variants.py`` routes to them
unchanged and each call traces as one node under ``torch.compile``. One
additive op has no counterpart there: ``fused_attention_gqa_varlen``
(per-sample lengths, the prefix-attention site the reference leaves on SDPA).
``fused_attention_gqa_train`` is the same attention with gradients.

The bf16 ops run one tcgen05 kernel (vla-kernels_b200/csrc/attention_gqa.cu):
QK^T and PV on the 5th-generation tensor cores with accumulators in tensor
memory, Q/K/V staged by TMA, the G query heads of a kv head sharing its K/V
tiles, the online softmax in registers and the prefix / dead-band / causal
mask computed from indices.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from .. import _native


@lru_cache(maxsize=1)
def _ext():
    _native.load_ops()
    # the ops return CONTIGUOUS tensors of q's shape; the fakes must promise
    # the same strides (kernels/attention/__init__.py:26-30)
    torch.library.register_fake("vlak::fused_attention")(
        lambda q, k, v, scale=-1.0, attn_mask=None, prefix_len=-1:
            torch.empty(q.shape, dtype=q.dtype, device=q.device))
    torch.library.register_fake("vlak::fused_attention_gqa")(
        lambda q, k, v, scale=-1.0, prefix_len=-1, dead_start=0, dead_end=0:
            torch.empty(q.shape, dtype=q.dtype, device=q.device))
    torch.library.register_fake("vlak::fused_attention_gqa_varlen")(
        lambda q, k, v, lengths, scale=-1.0:
            torch.empty(q.shape, dtype=q.dtype, device=q.device))
    return torch.ops.vlak


@lru_cache(maxsize=1)
def _ext_v4():
    _native.load_ops()
    torch.library.register_fake("vlak::fused_attention_gqa_v4")(
        lambda q, k, v, scale=-1.0, prefix_len=-1, dead_start=0, dead_end=0:
            torch.empty(q.shape, dtype=q.dtype, device=q.device))
    return torch.ops.vlak


@lru_cache(maxsize=1)
def _ext_train():
    _native.load_ops()

    def o_like(q):
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)

    torch.library.register_fake("vlak::fused_attention_gqa_train")(
        lambda q, k, v, scale=-1.0, prefix_len=-1, dead_start=0, dead_end=0, lengths=None,
        attn_mask=None: o_like(q))
    torch.library.register_fake("vlak::fused_attention_gqa_fwd_lse")(
        lambda q, k, v, scale=-1.0, prefix_len=-1, dead_start=0, dead_end=0, lengths=None,
        attn_mask=None:
            (o_like(q), torch.empty(q.shape[:3], dtype=torch.float32, device=q.device),
             torch.empty(q.shape, dtype=torch.int8, device=q.device)))
    torch.library.register_fake("vlak::fused_attention_gqa_bwd")(
        lambda grad_o, q, k, v, o, lse, o_low, scale=-1.0, prefix_len=-1, dead_start=0, dead_end=0,
        lengths=None, attn_mask=None, with_kv=True:
            [o_like(t) for t in ((q, k, v) if with_kv else (q,))])
    return torch.ops.vlak


_registered = False
_registered_v4 = False
_registered_train = False


def _ensure_registered():
    global _registered
    if not _registered:
        _ext()
        _registered = True


def _ensure_registered_v4():
    global _registered_v4
    if not _registered_v4:
        _ext_v4()
        _registered_v4 = True


def _ensure_registered_train():
    global _registered_train
    if not _registered_train:
        _ext_train()
        _registered_train = True


def fused_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    scale: float | None = None,
                    attn_mask: torch.Tensor | None = None,
                    prefix_len: int | None = None) -> torch.Tensor:
    """SDPA for (B, H, M, 64) tensors (kernels/attention/__init__.py:80-101).

    Masking, in preference order:
      prefix_len=P  analytic: col visible iff col < P or col <= (N - M) + row;
                    bf16 (tensor-core) path only.
      attn_mask     generic (B, M, N) bool, broadcast over heads.
      neither       unmasked.
    bf16 runs on the tensor cores; fp32 / fp16 / fp64 on the CUDA cores with
    fp32 math. Rows with no visible key are exact zeros.
    """
    _ensure_registered()
    return torch.ops.vlak.fused_attention(
        q, k, v, -1.0 if scale is None else scale, attn_mask,
        -1 if prefix_len is None else prefix_len)


def fused_attention_gqa_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                               lengths: torch.Tensor,
                               scale: float | None = None) -> torch.Tensor:
    """GQA attention with per-sample lengths: q (B, M, H, 64), k/v
    (B, N, H_kv, 64) bf16 at any strides, lengths (B,) int32/int64 on the
    device. visible(r, c) = c < L_b and r < L_b (L_b clamped to [0, N]);
    rows r >= L_b are exact zeros. Returns (B, M, H, 64) contiguous."""
    _ensure_registered()
    return torch.ops.vlak.fused_attention_gqa_varlen(
        q, k, v, lengths, -1.0 if scale is None else scale)


def fused_attention_gqa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        scale: float | None = None,
                        prefix_len: int | None = None,
                        dead_start: int = 0,
                        dead_end: int = 0) -> torch.Tensor:
    """Attention where H query heads share H_kv key/value heads.

    Inputs stay in the layout the projections produce: queries (B, M, H, 64)
    and keys / values (B, N, H_kv, 64), bf16, read in place at whatever
    strides they have (head_dim must be the unit-stride dim). Query head h
    uses kv head h // (H // H_kv). No mask tensor: key c is visible to query
    row r when c < prefix_len and c lies outside [dead_start, dead_end), or
    when c >= prefix_len and c <= (N - M) + r (a causal staircase over the
    trailing keys). prefix_len defaults to N and scale to 1/8.

    The result is a new contiguous (B, M, H, 64) tensor, so flattening the
    heads is a free view. A row that sees no key at all comes back as zeros.
    """
    _ensure_registered()
    return torch.ops.vlak.fused_attention_gqa(
        q, k, v, -1.0 if scale is None else scale,
        -1 if prefix_len is None else prefix_len, dead_start, dead_end)


def fused_attention_gqa_v4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           scale: float | None = None,
                           prefix_len: int | None = None,
                           dead_start: int = 0,
                           dead_end: int = 0) -> torch.Tensor:
    """The reference's v4 entry point; same contract as fused_attention_gqa."""
    _ensure_registered_v4()
    return torch.ops.vlak.fused_attention_gqa_v4(
        q, k, v, -1.0 if scale is None else scale,
        -1 if prefix_len is None else prefix_len, dead_start, dead_end)


def fused_attention_gqa_train(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                              scale: float | None = None,
                              prefix_len: int | None = None,
                              dead_start: int = 0,
                              dead_end: int = 0,
                              lengths: torch.Tensor | None = None,
                              attn_mask: torch.Tensor | None = None) -> torch.Tensor:
    """``fused_attention_gqa`` with gradients of q, k and v.

    Shapes, layouts and the analytic mask are those of ``fused_attention_gqa``;
    instead of it, ``lengths`` masks as in ``fused_attention_gqa_varlen`` or
    ``attn_mask`` (B, M, N) bool, True to attend, over all heads. Head h's
    gradient goes to kv head h // (H // H_kv), summed over its query heads.

    The backward pass (vla-kernels_b200/csrc/attention_bwd.cu) recomputes the
    probabilities; between the passes only q, k, v, the output (with eight
    more bits of each entry) and one float per row are kept. Sums are 32-bit in
    a fixed order, so gradients repeat bit for bit. A row that sees no key is
    zeros and has a zero gradient. Values that no row may see (a dead band,
    positions past a sample's length), and those of rows that see nothing, may be
    anything, NaN included; behind ``attn_mask`` all values must be finite.
    Differentiable once, in reverse mode.

    Precision: probabilities and score gradients are bf16 operands of the second
    products, which leaves errors of up to 1.45 times the rounding of the bf16
    result alone. Short calls (at most eight steps of 128 rows by 64 keys per SM,
    or rows that see at most 128 keys) hold them to 16 bits, and only the result's
    rounding is left. There is no switch: a sample alone and the same one in a
    batch may differ by that much.

    To capture a training step into a CUDA graph, let no eager autograd graph
    of the same leaves live meanwhile (drop its loss and outputs first):
    autograd would order the capture behind that graph's stream.
    """
    _ensure_registered_train()
    return torch.ops.vlak.fused_attention_gqa_train(
        q, k, v, -1.0 if scale is None else scale,
        -1 if prefix_len is None else prefix_len, dead_start, dead_end, lengths, attn_mask)


def device_error() -> int:
    """Synchronous check of the bounded device waits: waits for the device,
    then reads and clears the error words. Returns the status code of a wait
    that ran out since the last check (5, VLAK_ERR_DEVICE_TIMEOUT), else 0.

    Each op also reads the host-mapped error word on entry, without any
    synchronization, and raises RuntimeError when a kernel that has finished
    since the previous op gave up a wait; this call is for callers that want
    to know at a point of their choosing (e.g. after replaying a CUDA graph,
    whose replays run no host code)."""
    _native.load_ops()
    return int(torch.ops.vlak.device_error())


def check_device_error() -> None:
    """device_error(), raising RuntimeError when a wait ran out."""
    code = device_error()
    if code != 0:
        raise RuntimeError(f"vlak: a kernel gave up a bounded device wait (status {code}); "
                           "the output of that call is incomplete")
