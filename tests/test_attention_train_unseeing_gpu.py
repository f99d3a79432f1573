"""Rows of attention that see no key by the analytic mask: whatever q and the
gradient of the output hold there, NaN included, reaches nothing."""
import pytest
import torch

from tests.test_attention_train_gpu import make, step

pytestmark = pytest.mark.gpu


# B, M, N, H, Hkv, P, ds, de: more rows than keys, alone and behind a dead prefix; the
# first rows see nothing
@pytest.mark.parametrize("case", [
    (2, 90, 40, 3, 1, 0, 0, 0), (1, 90, 40, 3, 1, 10, 0, 10), (1, 300, 130, 6, 2, 0, 0, 0),
    (2, 100, 100, 4, 4, 37, 0, 37), (1, 70, 300, 15, 5, 260, 0, 260), (1, 50, 20, 128, 1, 3, 0, 3),
    (1, 2000, 300, 2, 1, 100, 0, 100), (3, 33, 64, 5, 1, 64, 0, 64), (30, 200, 150, 6, 6, 0, 0, 0),
], ids=str)
def test_what_they_hold_reaches_nothing(case):
    B, M, N, H, Hkv, P, ds, de = case
    q, k, v, do = make(*case[:5], seed=M + N)
    kw = dict(prefix_len=P, dead_start=ds, dead_end=de)
    none = min(M, max(0, M - N + P))
    ref = step(q, k, v, do, **kw)
    assert none > 0 and not ref[0][:, :none].any() and (none == M or ref[0][:, none:].any())
    q2, do2 = q.clone(), do.clone()
    q2[:, :none] = float("nan")
    do2[:, :none] = float("inf")
    q2[:, :none:2] = float("-inf")
    for name, a, b in zip(("o", "dq", "dk", "dv"), step(q2, k, v, do2, **kw), ref):
        assert torch.equal(a, b), name
