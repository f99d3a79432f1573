"""Rows of attention that see a single key, among longer ones: their softmax is
constant, so their true dS, dq and share of dk are zero.

What the kernels leave there is the difference of two 32-bit sums of the same 64
products, dP = do.v and D = do.o with o = v. D adds them with roundings of at
most 2^-24, independent: 2^-24 sqrt(64) = 2^-21 of its size. dP comes from the
tensor cores, whose 64 additions may truncate, each losing 2^-24 of the partial
sum in the mean, on average over the sum at most 64 2^-24 2 / 3 of its size.
Together below 2^-18, in the 2-norm over the rows. An o that is off by eight
bits of its last places (2^-16) is above it.

dq of such a row is scale dS k, so its norm gives dS, but for roundings of 2^-8.
"""
import pytest
import torch

from oracle import attention_train_oracle as orc
from tests.test_attention_train_gpu import make, step

pytestmark = pytest.mark.gpu

LEFT = 2.0 ** -18


def held(q, k, v, do, got, rows, key):
    """rows (B, M) bool: those that see only the key at key (B, M)."""
    B, M, H, _ = q.shape
    G = H // k.shape[2]
    at = key[:, :, None, None].expand(B, M, k.shape[2], 64)
    kk, vv = (torch.gather(t.double(), 1, at).repeat_interleave(G, 2)[rows] for t in (k, v))
    ds = got[1].double()[rows].norm(dim=-1) / (0.125 * kk.norm(dim=-1))
    D = (do.double()[rows] * vv).sum(-1)
    assert rows.any() and ds.norm() <= LEFT * D.norm(), float(ds.norm() / D.norm())
    assert torch.equal(got[0][rows], vv.to(got[0].dtype))  # o is the value


@pytest.mark.parametrize("shape", [(64, 8, 8, 8, 4), (32, 70, 70, 6, 2), (2, 1500, 1500, 2, 1)])
def test_first_row_of_a_staircase(shape):
    q, k, v, do = make(*shape, seed=shape[1])
    got = step(q, k, v, do, prefix_len=0)
    rows = torch.zeros(shape[:2], dtype=torch.bool, device="cuda")
    rows[:, 0] = True
    held(q, k, v, do, got, rows, torch.zeros(shape[:2], dtype=torch.long, device="cuda"))


# calls of few steps, which hold P and dS in more bits, and of many
@pytest.mark.parametrize("shape", [(2, 50, 291, 15, 5), (16, 256, 256, 8, 8), (1, 7, 2000, 4, 2)])
def test_bool_rows_of_one_bit(shape):
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=N)
    g = torch.Generator(device="cuda").manual_seed(M)
    key = torch.randint(0, N, (B, M), device="cuda", generator=g)
    rows = torch.rand(B, M, device="cuda", generator=g) < 0.5
    mask = torch.rand(B, M, N, device="cuda", generator=g) < 0.5
    one = torch.zeros_like(mask).scatter_(2, key[..., None], True)
    mask = torch.where(rows[..., None], one, mask)
    held(q, k, v, do, step(q, k, v, do, attn_mask=mask), rows, key)


@pytest.mark.parametrize("shape", [(8, 40, 300, 6, 2), (40, 300, 300, 4, 4)])
def test_keys_of_such_rows_alone(shape):
    # every row one key: dk is made of nothing else
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=M)
    key = torch.randint(0, N, (B, M), device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(B))
    mask = torch.zeros(B, M, N, dtype=torch.bool, device="cuda").scatter_(2, key[..., None], True)
    got = step(q, k, v, do, attn_mask=mask)
    rows = torch.ones(B, M, dtype=torch.bool, device="cuda")
    held(q, k, v, do, got, rows, key)
    # dk = scale sum dS q with dS of LEFT |D|, independent over rows
    at = key[:, :, None, None].expand(B, M, Hkv, 64)
    vv = torch.gather(v.double(), 1, at).repeat_interleave(H // Hkv, 2)
    D = (do.double() * vv).sum(-1)
    size = 0.125 * (D * q.double().norm(dim=-1)).norm()
    assert got[2].double().norm() <= LEFT * size, float(got[2].double().norm() / size)
    ref = orc.train(q, k, v, do, mask)["dv"]
    assert ((got[3].double() - ref[0]).abs() <= ref[1] + 1e-30).all()


def test_backward_without_the_low_bytes_takes_o_as_it_is():
    # o_low of zeros stands for an o without further bits (the C ABI's NULL): for
    # one key that o is exact
    B, M, N, H, Hkv = 8, 64, 200, 4, 2
    q, k, v, do = make(B, M, N, H, Hkv, seed=3)
    key = torch.randint(0, N, (B, M), device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(1))
    mask = torch.zeros(B, M, N, dtype=torch.bool, device="cuda").scatter_(2, key[..., None], True)
    o, lse, low = torch.ops.vlak.fused_attention_gqa_fwd_lse(q, k, v, attn_mask=mask)
    d = torch.ops.vlak.fused_attention_gqa_bwd(do, q, k, v, o, lse, torch.zeros_like(low),
                                               attn_mask=mask)
    rows = torch.ones(B, M, dtype=torch.bool, device="cuda")
    held(q, k, v, do, [o, *d], rows, key)
    assert not low.any()  # nothing is left of an exact o
