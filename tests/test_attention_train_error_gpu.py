"""How much error the attention gradients add to the rounding of their results.

The least error that a bf16 tensor can have is that of the exact result rounded
once; errors are given as multiples of its 2-norm.
  A call of few steps holds P, dS and O to 16 bits or more, 2^8 times finer than
  the result, so what it adds is below 1 %. The limit 1.15 leaves room for dS
  being a difference: where dP and D nearly cancel, their 2^-17 counts more.
  Other calls round P and dS to bf16: as much again as the result's rounding,
  independent of it, so sqrt(2) in the mean; the limit is 1.6.
The limits must also be able to fail: with O's low bytes left out, D takes the
bf16 rounding of O, which for rows of two keys weighs as much as dS itself.
"""
import pytest
import torch

from oracle import attention_train_oracle as orc
from tests.test_attention_train_gpu import make, random_mask, step

pytestmark = pytest.mark.gpu

FEW, MANY = 1.15, 1.6


def excess(x, want):
    return float((x.double() - want).norm() / (want.bfloat16().double() - want).norm())


def errors(got, q, k, v, do, seen):
    ref = orc.train(q, k, v, do, seen)
    return {n: excess(x, ref[n][0]) for n, x in zip(("o", "dq", "dk", "dv"), got)}


@pytest.mark.parametrize("N", [2, 3, 5, 9, 60, 128])
def test_rows_of_few_keys(N):
    # at most two chunks of 64 keys: held in 16 bits whatever the batch
    q, k, v, do = make(4, 400, N, 8, 4, seed=N)
    e = errors(step(q, k, v, do), q, k, v, do, orc.analytic(400, N, N))
    assert max(e.values()) <= FEW, e


@pytest.mark.parametrize("shape", [(1, 50, 291, 15, 5), (2, 241, 241, 3, 1)])
def test_calls_of_few_steps(shape):
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=N)
    e = errors(step(q, k, v, do, prefix_len=N // 2), q, k, v, do, orc.analytic(M, N, N // 2))
    assert max(e.values()) <= FEW, e


@pytest.mark.parametrize("mask", ["analytic", "lengths", "bool"])
def test_calls_of_many_steps(mask):
    B, M, N, H, Hkv = 24, 241, 241, 15, 5
    q, k, v, do = make(B, M, N, H, Hkv, seed=5)
    L = 150 + torch.arange(B, device="cuda") * 91 // (B - 1)
    bits = random_mask(B, M, N, seed=1)
    kw, seen = {"analytic": (dict(prefix_len=100), orc.analytic(M, N, 100)),
                "lengths": (dict(lengths=L), orc.by_length(M, N, L)),
                "bool": (dict(attn_mask=bits), bits)}[mask]
    e = errors(step(q, k, v, do, **kw), q, k, v, do, seen)
    assert max(e.values()) <= MANY, e


def test_the_limit_can_fail():
    q, k, v, do = make(4, 400, 2, 8, 4, seed=2)
    o, lse, low = torch.ops.vlak.fused_attention_gqa_fwd_lse(q, k, v)
    ref = orc.train(q, k, v, do, orc.analytic(400, 2, 2))
    for bytes_, fails in ((low, False), (torch.zeros_like(low), True)):
        dq, dk, _ = torch.ops.vlak.fused_attention_gqa_bwd(do, q, k, v, o, lse, bytes_)
        for x, n in ((dq, "dq"), (dk, "dk")):
            assert (excess(x, ref[n][0]) > FEW) == fails, (n, excess(x, ref[n][0]))
