"""Positions read in place at their own strides, and a closer bound on the turned
entries of each type.

Bounds, e = 2^-24. The fraction of a turn, at most 1/2, is a float: 2 pi 2^-26 =
1.6 e of the angle. fp32 heads: sine and cosine within 2 ulp, 2 e below 1;
amplitude, the factor's product with it, the entry's product and the sum e each.
So at most 3.6 + 4 < 8 e (|a| + |b|) A. 16-bit heads: the angle's product with
2 pi 2^-32 another pi e, that constant's own rounding 1.5 e at most half a turn,
the fast sine and cosine within 2^-21.19 = 7.1 e of the value (absolute, not in
ulp); so at most 1.6 + 3.2 + 1.5 + 7.1 + 4 < 18 e (|a| + |b|) A. The result's own
rounding, half of finfo.eps, comes on top.
"""
import pytest
import torch

from oracle import rotary_oracle as orc
from tests.test_rotary_gpu import DTYPES, E, api, gen, make, within

pytestmark = pytest.mark.gpu


def views(B, M, dtype):
    """(name, positions) all of the values wide[2 b, 3 m], by different strides."""
    g = gen(B + M)
    wide = torch.randint(-4096, 1 << 20, (2 * B, 3 * M + 1), device="cuda", generator=g).to(dtype)
    ref = wide[::2, 1::3].contiguous()
    yield "slice", wide[::2, 1::3], ref
    yield "transposed", ref.t().contiguous().t(), ref
    yield "row", wide[0, 1::3], ref[:1].expand(B, M).contiguous()
    yield "one row", wide[:1, 1::3], ref[:1].expand(B, M).contiguous()
    yield "one row, expanded", wide[:1, 1::3].expand(B, M), ref[:1].expand(B, M).contiguous()
    yield "column, expanded", wide[::2, 1:2].expand(B, M), ref[:, :1].expand(B, M).contiguous()
    yield "reversed order of samples", wide.as_strided((B, M), (2, 2 * B), 3), \
        wide.as_strided((B, M), (2, 2 * B), 3).contiguous()


# the 16-byte path and the path of any width
@pytest.mark.parametrize("D", [64, 72])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_at_any_stride(dtype, D):
    B, M = 3, 11
    q, k = make(B, M, 5, 2, D, torch.bfloat16, seed=D)
    w = 1 + torch.rand(D, device="cuda", generator=gen(2))
    gq, gk = make(B, M, 5, 2, D, torch.bfloat16, seed=D + 1)
    f = api().rotary_frequencies(D, device="cuda")

    def step(pos):
        x = [t.detach().requires_grad_(True) for t in (q, k)]
        y = api().qk_norm_rotary(*x, w, w, pos, f)
        return [*api().rotary(q, k, pos, f), *y, *torch.autograd.grad(y, x, (gq, gk))]

    for name, pos, same in views(B, M, dtype):
        th = orc.angles(same, f)
        got = step(pos)
        within(got[0], orc.turn(q, th), (18 * E + 4 * 2.0 ** -53 * (1 << 20)) * orc.pair_size(q, th))
        for a, b in zip(got, step(same)):
            assert torch.equal(a, b), name


def test_views_are_strided():
    strides = {name: pos.stride() for name, pos, _ in views(3, 11, torch.int64)}
    assert strides["slice"] == (68, 3) and strides["transposed"] == (1, 3)
    assert strides["row"] == (3,) and strides["column, expanded"] == (68, 0)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,rd", [(64, 64), (128, 32), (72, 70), (256, 256)])
def test_turned_entries_closely(D, rd, inter, dt):
    q, k = make(2, 301, 3, 1, D, DTYPES[dt], seed=rd)
    f = api().rotary_frequencies(rd, device="cuda")
    pos = torch.randint(0, 1 << 20, (2, 301), device="cuda", generator=gen(7))
    slack = (8 if dt == "fp32" else 18) * E * 1.25
    # float64 angles carry 2^-53 of their radians, on both sides
    slack += 4 * 2.0 ** -53 * (1 << 20) * 1.25
    th = orc.angles(pos, f)
    for y, x in zip(api().rotary(q, k, pos, f, interleaved=inter, amplitude=1.25), (q, k)):
        within(y, orc.turn(x, th, 1.25, inter), slack * orc.pair_size(x, th, inter))
