"""Forward-mode derivatives of the differentiable ops, which they do not have:
a tangent on any of their inputs is refused, not dropped. The refusal stands in
the autograd kernels, ahead of any device, so it is tested on CPU tensors."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from kernels.attention import fused_attention_gqa_train
from kernels.rotary import qk_norm_rotary, rotary, rotary_frequencies

POS = torch.arange(3)


def heads():
    return [torch.randn(1, 3, 2, 64).bfloat16() for _ in range(2)]


def rotary_inputs():
    return [*heads(), rotary_frequencies(64)]


def norm_inputs():
    return [*heads(), torch.ones(64), torch.ones(64), rotary_frequencies(64)]


def attention_inputs():
    return [*heads(), heads()[0]]


OPS = {"rotary": (rotary_inputs, lambda q, k, f: rotary(q, k, POS, f)),
       "norm": (norm_inputs, lambda q, k, wq, wk, f: qk_norm_rotary(q, k, wq, wk, POS, f)),
       "attention": (attention_inputs, fused_attention_gqa_train)}
PLACES = [(op, i) for op, (make, _) in OPS.items() for i in range(len(make()))]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("op,place", PLACES)
def test_a_tangent_is_refused(op, place, grad):
    make, call = OPS[op]
    x = make()
    x[0].requires_grad_(grad)
    with fwd.dual_level():
        x[place] = fwd.make_dual(x[place], torch.ones_like(x[place]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*x)


@pytest.mark.parametrize("op", list(OPS))
def test_jvp_is_refused(op):
    make, call = OPS[op]
    x = tuple(make())
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, x, tuple(torch.ones_like(t) for t in x))


def test_without_queries_own_tangent():
    # the only tensor with a tangent is one that may be absent
    q, k, f = rotary_inputs()
    with fwd.dual_level():
        q = fwd.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rotary(q, None, POS, f)
