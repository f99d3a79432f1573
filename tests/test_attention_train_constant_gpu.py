"""Calls and samples of attention in which no row sees more than one key: softmax is
constant there, and dq and dk are exactly zero."""
import pytest
import torch

from oracle import attention_train_oracle as orc
from tests.test_attention_train_gpu import check, make, step

pytestmark = pytest.mark.gpu


# B, M, N, H, Hkv, P, ds, de
@pytest.mark.parametrize("case", [
    (2, 9, 1, 6, 2, None, 0, 0),
    (2, 50, 291, 15, 5, 291, 1, 291),      # a dead band but for the first key
    (2, 50, 291, 15, 5, 291, 0, 290),      # or the last
    (3, 40, 200, 4, 4, 200, 0, 199),
    (2, 7, 70, 3, 1, 69, 0, 69),           # a dead prefix, a staircase of one step
    (1, 2000, 70, 8, 1, 70, 1, 70),        # long sides of few heads: joined parts
    (1, 5, 5000, 2, 1, 5000, 0, 4999),
    (40, 100, 130, 8, 8, 130, 1, 130),
], ids=str)
def test_analytic(case):
    B, M, N, H, Hkv, P, ds, de = case
    q, k, v, do = make(*case[:5], seed=N)
    got = step(q, k, v, do, prefix_len=P, dead_start=ds, dead_end=de)
    assert not got[1].any() and not got[2].any()
    check(got, orc.train(q, k, v, do, orc.analytic(M, N, N if P is None else P, ds, de)))


@pytest.mark.parametrize("shape", [(4, 60, 60, 6, 2), (4, 1800, 1800, 2, 1), (300, 70, 70, 4, 4)])
def test_samples_of_one_key(shape):
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=B)
    L = torch.full((B,), N, device="cuda")
    L[::2] = 1
    got = step(q, k, v, do, lengths=L)
    for d in got[1:3]:
        assert not d[::2].any() and d[1::2].any()
    check(got, orc.train(q, k, v, do, orc.by_length(M, N, L)))


def test_two_keys_are_not_taken_for_one():
    for kw in (dict(prefix_len=291, dead_start=1, dead_end=290),
               dict(prefix_len=291, dead_start=0, dead_end=289),
               dict(lengths=torch.tensor([2, 2], device="cuda"))):
        q, k, v, do = make(2, 50, 291, 15, 5)
        got = step(q, k, v, do, **kw)
        assert got[1].any() and got[2].any()
