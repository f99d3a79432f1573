"""GPU parity of vlak::fused_attention_gqa_train, forward and gradients, with
the float64 oracle.

Every entry is held to oracle/attention_train_oracle.py's bound, a sum of the
roundings on its way. On large random cases the 2-norm of the error is held
as well: an output goes through at most four independent roundings to bf16, of
at most 2^-8 / sqrt(3) each in the mean square, so 2^-8 * sqrt(4 / 3) of its
norm.
"""
import math

import pytest
import torch

from oracle import attention_train_oracle as orc

pytestmark = pytest.mark.gpu

NORM = 2.0 ** -8 * math.sqrt(4 / 3)


def attend(*a, **kw):
    from kernels.attention import fused_attention_gqa_train
    return fused_attention_gqa_train(*a, **kw)


def make(B, M, N, H, Hkv, seed=0, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    q = (gain * mk(B, M, H, 64).float()).bfloat16()
    return q, mk(B, N, Hkv, 64), mk(B, N, Hkv, 64), mk(B, M, H, 64)


def step(q, k, v, do, **kw):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = attend(q, k, v, **kw)
    assert o.shape == q.shape and o.is_contiguous()
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))


def check(got, ref, norm=False):
    torch.cuda.synchronize()
    for name, x in zip(("o", "dq", "dk", "dv"), got):
        want, bound = ref[name]
        assert x.dtype == torch.bfloat16 and x.is_contiguous()
        err = (x.double() - want).abs()
        bad = ~(err <= bound + 1e-30)
        assert not bad.any(), (name, int(bad.sum()), float(err[bad].max()),
                               bad.nonzero()[:3].tolist())
        if norm and want.norm() > 0:
            assert err.norm() / want.norm() <= NORM, (name, float(err.norm() / want.norm()))


def run(B, M, N, H, Hkv, P=None, ds=0, de=0, seed=0, norm=False, gain=1.0, scale=None):
    q, k, v, do = make(B, M, N, H, Hkv, seed, gain)
    got = step(q, k, v, do, prefix_len=P, dead_start=ds, dead_end=de, scale=scale)
    seen = orc.analytic(M, N, N if P is None else P, ds, de)
    check(got, orc.train(q, k, v, do, seen, scale or 0.125), norm)
    return got


# B, M, N, H, Hkv, P, ds, de
ANALYTIC = [
    (1, 50, 291, 15, 5, 241, 196, 240),
    (4, 50, 241, 15, 5, None, 0, 0),
    (2, 50, 291, 15, 5, 241, 0, 0),
    (1, 1, 1, 1, 1, None, 0, 0),
    (2, 1, 64, 3, 1, None, 0, 0),
    (1, 1, 777, 15, 5, 700, 3, 70),
    (1, 200, 2, 2, 1, 0, 0, 0),
    (1, 64, 64, 1, 1, 0, 0, 0),
    (1, 65, 65, 1, 1, 0, 0, 0),
    (1, 128, 128, 2, 1, 0, 0, 0),
    (2, 129, 129, 2, 2, 0, 0, 0),
    (1, 127, 193, 4, 2, 0, 0, 0),
    (1, 300, 300, 3, 1, 0, 0, 0),
    (1, 300, 300, 3, 1, 130, 10, 129),
    (1, 100, 130, 6, 2, 70, 64, 64),
    (1, 40, 256, 8, 1, 256, 64, 192),
    (1, 40, 256, 8, 1, 256, 1, 255),
    (2, 33, 200, 5, 1, 200, 0, 200),      # no key visible at all
    (1, 90, 40, 3, 1, 0, 0, 0),           # more rows than keys: rows that see none
    (1, 90, 40, 3, 1, 10, 0, 10),         # and a dead prefix
    (1, 3, 70, 128, 1, None, 0, 0),
    (1, 5, 70, 127, 1, 0, 0, 0),
    (1, 7, 90, 96, 1, 30, 2, 9),
    (1, 9, 70, 67, 1, 70, 0, 0),
    (1, 21, 100, 20, 4, 0, 0, 0),
    (1, 1024, 1024, 2, 2, None, 0, 0),
    (1, 700, 1100, 6, 2, 500, 100, 300),
]


@pytest.mark.parametrize("case", ANALYTIC, ids=str)
def test_analytic(case):
    B, M, N, H, Hkv, P, ds, de = case
    run(B, M, N, H, Hkv, P, ds, de, seed=M + N, norm=M * N > 60000)


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 257])
def test_key_counts(N):
    run(1, 50, N, 3, 1, N // 2, 0, N // 4, seed=N)


@pytest.mark.parametrize("M", [1, 2, 20, 21, 22, 42, 43, 63, 64, 65, 85, 128, 130])
@pytest.mark.parametrize("heads", [(3, 1), (4, 2), (2, 2)])
def test_row_counts(M, heads):
    run(1, M, 100, *heads, 60, 5, 40, seed=M)


def test_large_scores_and_scale():
    run(1, 70, 150, 4, 2, 40, 0, 0, gain=30.0)  # nearly one-hot rows
    run(1, 70, 150, 4, 2, 40, 0, 0, scale=0.5)
    run(1, 70, 150, 4, 2, 40, 0, 0, scale=1e-3)


def test_scale_below_the_smallest_float():
    # zero in 32 bits, which must not meet the -inf of masked scores
    run(1, 70, 150, 4, 2, 40, 0, 0, scale=1e-60)
    run(2, 60, 60, 2, 1, 0, 0, 0, scale=1e-300)


@pytest.mark.parametrize("N", [2, 3, 5, 9])
def test_few_keys_keep_their_precision(N):
    # where a row's weight lies on few keys, D = rowsum(do * o) is as large as dP:
    # with o rounded to bf16, its error would be that of dS once more. The
    # gradients' roundings here: P, dS, and the result's, so 2^-8 of the norm
    # (three times 2^-8 / sqrt(3) in the mean square)
    q, k, v, do = make(4, 400, N, 8, 4, seed=N)
    got = step(q, k, v, do)
    ref = orc.train(q, k, v, do, orc.analytic(400, N, N))
    check(got, ref)
    for name, x in zip(("dq", "dk"), got[1:]):
        want = ref[name][0]
        assert (x.double() - want).norm() <= 2.0 ** -8 * want.norm()


def test_one_key_has_no_score_gradient():
    for kw in ({}, dict(P=0)):
        got = run(2, 9, 1, 6, 2, **kw)
        assert not got[1].any() and not got[2].any()


@pytest.mark.parametrize("M,N", [(50, 0), (0, 50), (0, 0)])
@pytest.mark.parametrize("B", [0, 2])
def test_empty(B, M, N):
    q, k, v, do = make(B, M, N, 6, 2)
    got = step(q, k, v, do)
    for t in got:
        assert not t.any()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", [(6, 241, 241, 15, 5), (6, 70, 200, 4, 1), (6, 200, 70, 3, 3)])
def test_lengths(shape, dtype):
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=N)
    L = torch.tensor([0, 1, 64, N - 1, N + 9, -3], device="cuda", dtype=dtype)
    got = step(q, k, v, do, lengths=L)
    check(got, orc.train(q, k, v, do, orc.by_length(M, N, L)))


@pytest.mark.parametrize("shape", [(300, 150, 150, 3, 1), (260, 200, 200, 2, 2), (700, 60, 60, 3, 1),
                                   (400, 1, 64, 4, 2), (500, 70, 1, 2, 1)])
@pytest.mark.parametrize("most", [1.0, 0.3])
def test_many_samples_of_all_lengths(shape, most):
    # far more pieces of work than the GPU takes at once, many of them empty or
    # of a single step, in any order
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=B)
    g = torch.Generator(device="cuda").manual_seed(N)
    L = torch.randint(0, int(most * N) + 1, (B,), device="cuda", generator=g)
    L[B // 3: B // 2] = 0
    check(step(q, k, v, do, lengths=L), orc.train(q, k, v, do, orc.by_length(M, N, L)))


@pytest.mark.parametrize("shape", [(200, 50, 291, 15, 5, 241, 196, 240), (300, 64, 64, 2, 1, 0, 0, 0),
                                   (90, 200, 40, 3, 1, 0, 0, 0), (500, 3, 130, 2, 2, 130, 0, 128)])
def test_many_samples(shape):
    B, M, N, H, Hkv, P, ds, de = shape
    run(*shape[:5], P, ds, de, seed=B)


# few heads and one long side: an output's steps are shared out and joined
@pytest.mark.parametrize("case", [(1, 2000, 1, 8, 1, None, 0, 0), (1, 2000, 70, 8, 1, 70, 5, 66),
                                  (1, 1500, 1500, 1, 1, 0, 0, 0), (1, 1, 5000, 1, 1, None, 0, 0),
                                  (1, 50, 4111, 3, 1, 4000, 100, 3900), (2, 2111, 9, 3, 1, 0, 0, 0),
                                  (1, 7, 3000, 127, 1, 0, 0, 0), (1, 1300, 40, 67, 1, 0, 0, 0)], ids=str)
def test_long_side_of_few_heads(case):
    B, M, N, H, Hkv, P, ds, de = case
    run(*case[:5], P, ds, de, seed=M)


@pytest.mark.parametrize("shape", [(2, 1800, 1800, 2, 1), (1, 30, 3000, 3, 1), (1, 3000, 30, 3, 1)])
def test_long_side_of_few_heads_other_masks(shape):
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=M)
    mask = random_mask(B, M, N, seed=N)
    mask[:, :, N // 3: N // 2] = False
    check(step(q, k, v, do, attn_mask=mask), orc.train(q, k, v, do, mask))
    L = torch.tensor([N // 2, N][:B], device="cuda")
    check(step(q, k, v, do, lengths=L), orc.train(q, k, v, do, orc.by_length(M, N, L)))


def random_mask(B, M, N, seed, share=0.6):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = torch.rand(B, M, N, device="cuda", generator=g) < share
    m &= torch.rand(B, M, 1, device="cuda", generator=g) < 0.9  # rows that see nothing
    m &= torch.rand(B, 1, N, device="cuda", generator=g) < 0.9  # keys that no row sees
    return m


@pytest.mark.parametrize("shape", [(2, 50, 291, 15, 5), (1, 130, 77, 2, 2), (2, 64, 128, 8, 1),
                                   (1, 5, 200, 127, 1), (1, 3, 64, 64, 1), (3, 1, 1, 2, 1)])
def test_bool_mask(shape):
    B, M, N, H, Hkv = shape
    q, k, v, do = make(*shape, seed=M)
    mask = random_mask(B, M, N, seed=N)
    check(step(q, k, v, do, attn_mask=mask), orc.train(q, k, v, do, mask))


def test_bool_mask_forms_agree():
    B, M, N, H, Hkv = 2, 33, 90, 6, 2
    q, k, v, do = make(B, M, N, H, Hkv)
    row = random_mask(1, 1, N, 1)[0, 0]
    ref = step(q, k, v, do, attn_mask=row.expand(B, M, N).contiguous())
    wide = torch.zeros(B, M, N + 3, dtype=torch.bool, device="cuda")
    wide[:, :, 2:-1] = row
    for mask in (row.expand(B, M, N), wide[:, :, 2:-1],
                 row.expand(B, M, N).transpose(1, 2).contiguous().transpose(1, 2)):
        for a, b in zip(step(q, k, v, do, attn_mask=mask), ref):
            assert torch.equal(a, b)
    # the analytic mask as a bool mask
    seen = orc.analytic(M, N, 60, 10, 30).expand(B, M, N).contiguous()
    ref = step(q, k, v, do, prefix_len=60, dead_start=10, dead_end=30)
    for a, b in zip(step(q, k, v, do, attn_mask=seen), ref):
        assert torch.equal(a, b)


def test_forward_agrees_with_the_inference_op():
    # kernels of their own, with other orders of summation: each within the
    # oracle's bound, so no further apart than twice that
    from kernels.attention import fused_attention_gqa, fused_attention_gqa_varlen
    q, k, v, do = make(3, 50, 291, 15, 5)
    a = attend(q, k, v, prefix_len=241, dead_start=196, dead_end=240)
    b = fused_attention_gqa(q, k, v, prefix_len=241, dead_start=196, dead_end=240)
    bound = orc.train(q, k, v, do, orc.analytic(50, 291, 241, 196, 240))["o"][1]
    assert ((a.double() - b.double()).abs() <= 2 * bound).all()
    L = torch.tensor([291, 7, 100], device="cuda")
    q, k, v, do = make(3, 291, 291, 15, 5)
    a, b = attend(q, k, v, lengths=L), fused_attention_gqa_varlen(q, k, v, L)
    bound = orc.train(q, k, v, do, orc.by_length(291, 291, L))["o"][1]
    assert ((a.double() - b.double()).abs() <= 2 * bound).all()
    assert not a.requires_grad
    assert torch.equal(a, attend(q.requires_grad_(True), k, v, lengths=L))


def test_log_sums():
    B, M, N, H, Hkv = 2, 90, 40, 6, 2
    from kernels import attention
    attention._ensure_registered_train()
    for B, M, N, P in ((2, 90, 40, 0), (1, 50, 700, 600), (40, 50, 291, 241)):
        q, k, v, do = make(B, M, N, H, Hkv)
        _, lse, _ = torch.ops.vlak.fused_attention_gqa_fwd_lse(q, k, v, -1.0, P, 0, 0)
        want = orc.train(q, k, v, do, orc.analytic(M, N, P))["lse"][0]
        empty = want.isinf()
        assert torch.equal(lse.double()[empty], want[empty])
        assert (lse.double() - want)[~empty].abs().max() <= 2.0 ** -13 * want[~empty].abs().max()


def test_layouts_read_in_place():
    # a packed projection, head-major (B, H, M, 64) storage, padded rows
    B, M, H, Hkv = 2, 77, 6, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(B, M, H + 2 * Hkv, 64, device="cuda", generator=g).bfloat16()
    q, k, v = x[:, :, :H], x[:, :, H:H + Hkv], x[:, :, H + Hkv:]
    do = torch.randn(B, M, H, 64, device="cuda", generator=g).bfloat16()
    ref = step(*(t.contiguous() for t in (q, k, v)), do, prefix_len=30)
    for a, b in zip(step(q, k, v, do, prefix_len=30), ref):
        assert torch.equal(a, b)
    hm = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    for a, b in zip(step(hm(q), hm(k), hm(v), hm(do), prefix_len=30), ref):
        assert torch.equal(a, b)
    pad = torch.zeros(B, M, H, 72, device="cuda", dtype=torch.bfloat16)
    pad[..., :64] = do
    odd = torch.zeros(B, M, H, 65, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = do
    for grad in (pad[..., :64], odd[..., 1:], do.transpose(2, 3).contiguous().transpose(2, 3)):
        for a, b in zip(step(q, k, v, grad, prefix_len=30), ref):
            assert torch.equal(a, b)


def test_strides_past_32_bits():
    # samples 2^31 + 2^20 entries apart in one buffer, also those of the gradient
    far = (1 << 31) + (1 << 20)
    q, k, v, do = make(2, 70, 70, 6, 2, seed=9)
    buf = torch.empty(far + (1 << 20), device="cuda", dtype=torch.bfloat16)
    placed, at = [], 0
    for t in (q, k, v, do):
        p = buf.as_strided(t.shape, (far, *t.stride()[1:]), at)
        p.copy_(t)
        placed.append(p)
        at += t.stride(0)
    assert at <= 1 << 20
    got, same = step(*placed, prefix_len=0), step(q, k, v, do, prefix_len=0)
    assert all(torch.equal(a, b) for a, b in zip(got, same))


def test_expanded_inputs_and_gradient():
    # a batch that shares its keys, and a loss that hands back one expanded number
    B, M, N, H, Hkv = 3, 20, 60, 4, 2
    q, k, v, _ = make(B, M, N, H, Hkv)
    k1, v1 = (t[:1].detach().requires_grad_(True) for t in (k, v))
    q = q.requires_grad_(True)
    o = attend(q, k1.expand(B, N, Hkv, 64), v1.expand(B, N, Hkv, 64))
    dq, dk, dv = torch.autograd.grad(o.sum(), (q, k1, v1))
    ref = step(q, k1.expand(B, N, Hkv, 64).contiguous(), v1.expand(B, N, Hkv, 64).contiguous(),
               torch.ones_like(q))
    assert torch.equal(dq, ref[1])
    assert torch.equal(dk, ref[2].sum(0, keepdim=True))
    assert torch.equal(dv, ref[3].sum(0, keepdim=True))


def test_one_tensor_as_queries_keys_and_values():
    x, _, _, do = make(2, 150, 150, 4, 4, seed=5)
    leaf = x.detach().requires_grad_(True)
    o = attend(leaf, leaf, leaf, prefix_len=0)
    (d,) = torch.autograd.grad(o, (leaf,), do)
    ref = orc.train(x, x, x, do, orc.analytic(150, 150, 0))
    want = sum(ref[n][0] for n in ("dq", "dk", "dv"))
    # autograd adds the three in bf16: two more roundings of partial sums
    size = sum(ref[n][0].abs() for n in ("dq", "dk", "dv"))
    bound = sum(ref[n][1] for n in ("dq", "dk", "dv")) * (1 + 2 ** -7) + 2 * 2.0 ** -8 * (1 + 2 ** -7) * size
    assert ((d.double() - want).abs() <= bound + 1e-30).all()
    check((o.detach(),), {"o": ref["o"]})


def test_frozen_inputs():
    q, k, v, do = make(2, 50, 100, 6, 2)
    ref = step(q, k, v, do)
    for i in range(3):
        leaf = [t.detach() for t in (q, k, v)]
        leaf[i].requires_grad_(True)
        (d,) = torch.autograd.grad(attend(*leaf), leaf[i], do)
        assert torch.equal(d, ref[1 + i])


def test_values_in_masked_places():
    nan = float("nan")
    q, k, v, do = make(2, 50, 291, 15, 5)
    kw = dict(prefix_len=241, dead_start=100, dead_end=230)
    ref = step(q, k, v, do, **kw)
    k2, v2 = k.clone(), v.clone()
    k2[:, 100:230], v2[:, 100:230] = nan, float("inf")
    got = step(q, k2, v2, do, **kw)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    q, k, v, do = make(3, 100, 100, 6, 2)
    L = torch.tensor([37, 100, 64], device="cuda")
    ref = step(q, k, v, do, lengths=L)
    past = torch.arange(100, device="cuda")[None] >= L[:, None]
    q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
    for t, x in ((q2, nan), (k2, float("inf")), (v2, nan), (do2, nan)):
        t[past] = x
    for a, b in zip(step(q2, k2, v2, do2, lengths=L), ref):
        assert torch.equal(a, b)


def test_seen_nan_is_not_hidden():
    q, k, v, do = make(1, 40, 90, 2, 1)
    for t, at in ((q, (0, 3, 1, 5)), (k, (0, 70, 0, 9)), (v, (0, 70, 0, 9))):
        t2 = t.clone()
        t2[at] = float("nan")
        args = [t2 if x is t else x for x in (q, k, v)]
        assert any(x.isnan().any() for x in step(*args, do))
        assert step(*args, do)[0].isnan().any()


def test_gradients_against_differences():
    # directional derivative of the float64 function by central differences
    # (error of order h^2 taken from a doubled step) against the kernels'
    # gradients, whose own bound is the oracle's
    B, M, N, H, Hkv = 1, 30, 70, 4, 2
    q, k, v, do = make(B, M, N, H, Hkv)
    seen = orc.analytic(M, N, 50, 10, 20)
    ref = orc.train(q, k, v, do, seen)
    got = step(q, k, v, do, prefix_len=50, dead_start=10, dead_end=20)
    d = make(B, M, N, H, Hkv, seed=9)[:3]

    def loss(h):
        x = [t.double() + h * e.double() for t, e in zip((q, k, v), d)]
        return float((orc.train(*x, do, seen)["o"][0] * do.double()).sum())

    h = 2.0 ** -12
    one = (loss(h) - loss(-h)) / (2 * h)
    two = (loss(2 * h) - loss(-2 * h)) / (4 * h)
    along = sum(float((g.double() * e.double()).sum()) for g, e in zip(got[1:], d))
    slack = sum(float((ref[n][1] * e.double().abs()).sum()) for n, e in zip(("dq", "dk", "dv"), d))
    assert abs(along - (4 * one - two) / 3) <= slack + abs(one - two)
    # and the bound is no empty one: the oracle's own gradient agrees closely
    exact = sum(float((ref[n][0] * e.double()).sum()) for n, e in zip(("dq", "dk", "dv"), d))
    assert abs(exact - (4 * one - two) / 3) <= 1e-6 * (abs(exact) + 1) + abs(one - two)


def test_repeats_bit_for_bit():
    q, k, v, do = make(4, 300, 500, 6, 2)
    ref = step(q, k, v, do, prefix_len=200)
    for _ in range(3):
        for a, b in zip(step(q, k, v, do, prefix_len=200), ref):
            assert torch.equal(a, b)


def test_one_sample_equals_its_place_in_a_batch_within_bounds():
    q, k, v, do = make(70, 50, 291, 15, 5)
    got = step(q, k, v, do, prefix_len=241)
    ref = orc.train(q[40:42], k[40:42], v[40:42], do[40:42], orc.analytic(50, 291, 241))
    check([t[40:42].contiguous() for t in got], ref, norm=True)


def test_graph_capture_replays_on_new_inputs():
    q, k, v, do = make(2, 50, 291, 15, 5)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))

    def one():
        o = attend(q, k, v, prefix_len=241)
        return [o, *torch.autograd.grad(o, (q, k, v), do)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):  # two graphs: each has its own workspaces
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out = one()
        graphs[-1] = (graphs[-1], out)
    n = make(2, 50, 291, 15, 5, seed=5)
    with torch.no_grad():
        for t, x in zip((q, k, v, do), n):
            t.copy_(x)
    for graph, _ in graphs:
        graph.replay()
    want = [t.detach() for t in one()]
    for _, out in graphs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_side_streams_at_once():
    sets = [make(2, 200, 300, 6, 2, seed=i) for i in range(3)]
    ref = [step(*x, prefix_len=100) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    torch.cuda.synchronize()
    for s, x in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append(step(*x, prefix_len=100))
    torch.cuda.synchronize()
    for g, r in zip(got, ref):
        for a, b in zip(g, r):
            assert torch.equal(a, b)


def test_compiles_as_one_graph():
    q, k, v, do = make(1, 50, 291, 15, 5)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    ref = step(q, k, v, do, prefix_len=241)
    fn = torch.compile(lambda a, b, c: attend_(a, b, c, prefix_len=241), fullgraph=True,
                       backend="aot_eager")
    from kernels.attention import fused_attention_gqa_train as attend_
    o = fn(q, k, v)
    got = [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


def test_no_error_word():
    from kernels.attention import device_error
    run(1, 50, 291, 15, 5, 241)
    assert device_error() == 0


def test_refusals():
    q, k, v, do = make(2, 10, 20, 6, 2)
    L = torch.tensor([5, 6], device="cuda")
    mask = torch.ones(2, 10, 20, dtype=torch.bool, device="cuda")
    bad = [
        lambda: attend(q.float(), k, v),
        lambda: attend(q[..., :32], k[..., :32], v[..., :32]),
        lambda: attend(q, k, v[:, :19]),
        lambda: attend(q, k[:1], v[:1]),
        lambda: attend(q[:, :, :5], k, v),
        lambda: attend(q, k, v, prefix_len=21),
        lambda: attend(q, k, v, prefix_len=10, dead_start=5, dead_end=11),
        lambda: attend(q, k, v, dead_start=6, dead_end=5),
        lambda: attend(q, k, v, lengths=L, attn_mask=mask),
        lambda: attend(q, k, v, lengths=L, prefix_len=3),
        lambda: attend(q, k, v, attn_mask=mask, dead_end=3),
        lambda: attend(q, k, v, lengths=L[:1]),
        lambda: attend(q, k, v, lengths=L.float()),
        lambda: attend(q, k, v, lengths=L.cpu()),
        lambda: attend(q, k, v, attn_mask=mask[:1]),
        lambda: attend(q, k, v, attn_mask=mask.float()),
        lambda: attend(q, k, v, attn_mask=mask.cpu()),
        lambda: attend(q, k.cpu(), v),
        lambda: attend(q.cpu(), k.cpu(), v.cpu()),
        lambda: attend(torch.randn(2, 10, 6, 65, device="cuda").bfloat16()[..., 1:], k, v),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
            pytest.fail(f"case {i} was accepted")
    o, lse, low = torch.ops.vlak.fused_attention_gqa_fwd_lse(q, k, v)
    for args in ((do.float(), q, k, v, o, lse, low), (do[:1], q, k, v, o, lse, low),
                 (do, q, k, v, o[:, :5], lse, low), (do, q, k, v, o, lse[:1], low),
                 (do, q, k, v, o, lse.double(), low), (do, q, k, v, o, lse, low[:1]),
                 (do, q, k, v, o, lse, low.float())):
        with pytest.raises(RuntimeError):
            torch.ops.vlak.fused_attention_gqa_bwd(*args)
    # differentiable once
    qq = q.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(attend(qq, k, v).float().square().sum(), qq, create_graph=True)
    with pytest.raises(RuntimeError):
        d.float().sum().backward()


@pytest.mark.parametrize("mask", ["analytic", "lengths"])
def test_block_of_norm_rotation_and_attention(mask):
    # the operators in the order a step uses them: packed projection -> norm and
    # rotation -> attention, and all gradients back to the projection
    from kernels.rotary import qk_norm_rotary, rotary_frequencies
    from oracle import rotary_oracle as rot

    B, M, H, Hkv = 2, 90, 6, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(B, M, H + 2 * Hkv, 64, device="cuda", generator=g).bfloat16().requires_grad_(True)
    w = [(1 + 0.2 * torch.randn(64, device="cuda", generator=g)).requires_grad_(True) for _ in range(2)]
    do = torch.randn(B, M, H, 64, device="cuda", generator=g).bfloat16()
    f = rotary_frequencies(64, device="cuda")
    pos = torch.arange(M, device="cuda") + 1000
    L = torch.tensor([90, 41], device="cuda")
    how = dict(prefix_len=30) if mask == "analytic" else dict(lengths=L)
    q, k = qk_norm_rotary(x[:, :, :H], x[:, :, H:H + Hkv], *w, pos, f)
    o = attend(q, k, x[:, :, H + Hkv:], **how)
    got = torch.autograd.grad(o, (x, *w), do)

    xd = x.detach().double().requires_grad_(True)
    wd = [t.detach().double().requires_grad_(True) for t in w]
    th = rot.angles(pos.expand(B, M), f)
    turned = []
    for t, ww in ((xd[:, :, :H], wd[0]), (xd[:, :, H:H + Hkv], wd[1])):
        u = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * ww
        a, b = u[..., :32], u[..., 32:]
        turned.append(torch.cat((a * th.cos() - b * th.sin(), b * th.cos() + a * th.sin()), -1))
    seen = orc.analytic(M, M, 30) if mask == "analytic" else orc.by_length(M, M, L)
    G = H // Hkv
    kk, vv = (t.repeat_interleave(G, 2) for t in (turned[1], xd[:, :, H + Hkv:]))
    s = torch.einsum("bmhd,bnhd->bhmn", turned[0], kk) / 8
    s = s.masked_fill(~seen[:, None], float("-inf"))
    p = torch.softmax(s.masked_fill(~seen.any(-1)[:, None, :, None], 0.0), -1) * seen[:, None]
    od = torch.einsum("bhmn,bnhd->bmhd", p, vv)
    want = torch.autograd.grad(od, (xd, *wd), do.double())
    # roundings to bf16 on the way (q, k, P, o, dS, dq / dk / dv, dx): eight at
    # most, independent, each 2^-8 / sqrt(3) in the mean square
    for a, b in zip((o.detach(), *got), (od.detach(), *want)):
        assert (a.double() - b).norm() <= 2.0 ** -8 * math.sqrt(8 / 3) * b.norm()
