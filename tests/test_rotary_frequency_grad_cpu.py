"""Frequencies that want a gradient: the ops have none for them, and refuse
where autograd would have recorded it. Refused ahead of any device, so tested on
CPU tensors."""
import pytest
import torch

from kernels.rotary import qk_norm_rotary, rotary, rotary_frequencies

POS = torch.arange(3)


def calls(f, grad):
    q, k = (torch.randn(1, 3, 2, 64, requires_grad=grad) for _ in range(2))
    w = torch.ones(64, requires_grad=grad)
    return [lambda: rotary(q, k, POS, f), lambda: rotary(q, None, POS, f),
            lambda: qk_norm_rotary(q, k, w, w, POS, f)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("i", range(3))
def test_refused(i, grad):
    f = rotary_frequencies(64).requires_grad_(True)
    with pytest.raises(NotImplementedError, match="inv_freq"):
        calls(f, grad)[i]()


@pytest.mark.parametrize("i", range(3))
def test_not_refused_where_nothing_is_recorded(i):
    # past this check, CPU tensors are refused for what they are
    f = rotary_frequencies(64).requires_grad_(True)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="CPU"):
        calls(f, True)[i]()
    with pytest.raises(NotImplementedError, match="CPU"):
        calls(f.detach(), False)[i]()
