"""Sines and cosines of fp32 heads, read off the rotation of unit vectors.

A pair (1, 0) turns into (cos, sin) with no further rounding. Their angle is the
fraction of a turn in 32 bits, so 2 pi 2^-32 < 1.5e-9 radians off at most; the sine
and cosine are within 2 ulp, 4 e of the value with e = 2^-24, and what the angle has
beyond a float's 24 bits is added with one more rounding. So 6 e |value| + 2e-9, also
where the value is small: near half a turn a float's angle alone is off by 9e-8.
float64 angles of these positions are exact to 1e-12.
"""
import pytest
import torch

from tests.test_rotary_gpu import E, api

pytestmark = pytest.mark.gpu


# the 16-byte path, the path of any width, and its widest heads
@pytest.mark.parametrize("D", [64, 72, 514])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
def test_unit_vectors(D, inter, sign):
    f = api().rotary_frequencies(D, device="cuda")
    pos = sign * torch.arange(4096, device="cuda")
    q = torch.zeros(1, 4096, 1, D, device="cuda")
    a = slice(0, None, 2) if inter else slice(0, D // 2)
    b = slice(1, None, 2) if inter else slice(D // 2, None)
    q[..., a] = 1.0
    y = api().rotary(q, None, pos, f, interleaved=inter).double()
    t = pos.double()[None, :, None, None] * f
    for got, want in ((y[..., a], t.cos()), (y[..., b], t.sin())):
        err = (got - want).abs() - (6 * E * want.abs() + 2e-9)
        assert err.max() <= 0, (float(err.max()), int((err > 0).sum()))
