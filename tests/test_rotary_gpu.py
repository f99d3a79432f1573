"""GPU parity of vlak::rotary and vlak::qk_norm_rotary with the float64 oracle.

Bounds. An output is rounded once to its type: at most finfo(t).eps / 2 of its
value. Everything before is 32-bit: with e = 2^-24, cos and sin carry at most
2 ulp plus the angle's own rounding (the fraction of a turn, |x| <= 1/2, as a
float: 2 pi * 2^-26, under 4 e in all), each product and sum e; so a rotated
entry is off by at most 16 e (|a| + |b|) A. The norm adds its rsqrt (2 ulp),
the mean's sum (at most D / 32 + 6 additions deep) and three products: under
(D / 32 + 16) e relative. A gradient's dot product has the same depth.
A weight gradient adds `rows` terms at most one by one: (rows + 64) e of the
sum of the terms' magnitudes.
"""
import itertools

import pytest
import torch

from oracle import rotary_oracle as orc

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def api():
    from kernels import rotary as r
    return r


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(B, M, H, Hkv, D, dtype, seed=0, packed=False):
    g = gen(seed)
    if packed:
        x = torch.randn(B, M, H + 2 * Hkv, D, device="cuda", generator=g).to(dtype)
        return x[:, :, :H], x[:, :, H:H + Hkv]
    return (torch.randn(B, M, H, D, device="cuda", generator=g).to(dtype),
            torch.randn(B, M, Hkv, D, device="cuda", generator=g).to(dtype))


def within(got, ref, slack):
    err = (got.double() - ref).abs()
    tol = torch.finfo(got.dtype).eps / 2 * ref.abs() + slack
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half the subnormal step
    bad = err > tol
    assert not bad.any(), (int(bad.sum()), float((err - tol).max()), float(err.max()))


def check_turn(y, x, theta, amp, inter, inverse=False):
    ref = orc.turn(x, theta, amp, inter, inverse)
    within(y, ref, 16 * E * amp * orc.pair_size(x, theta, inter))


# B, M, H, Hkv, D, rotary_dim: one token, one head, whole and part of the head,
# widths with and without whole 16-byte vectors in each half, wide heads
SHAPES = [
    (1, 1, 1, 1, 2, 2),
    (1, 1, 15, 5, 64, 64),
    (3, 7, 15, 5, 64, 32),
    (2, 50, 12, 12, 64, 16),
    (1, 33, 4, 1, 80, 80),
    (2, 5, 3, 2, 72, 36),
    (1, 9, 8, 2, 128, 64),
    (2, 3, 2, 1, 256, 256),
    (1, 2, 3, 1, 96, 46),
    (1, 3, 2, 1, 512, 512),
    (1, 2, 2, 2, 1024, 514),
    (1, 4097, 3, 1, 32, 32),
]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(shape, inter, dt):
    B, M, H, Hkv, D, rd = shape
    q, k = make(B, M, H, Hkv, D, DTYPES[dt], seed=D + M, packed=(B + M) % 2 == 1)
    f = api().rotary_frequencies(rd, device="cuda")
    pos = torch.randint(-100, 4096, (B, M), device="cuda", generator=gen(1))
    yq, yk = api().rotary(q, k, pos, f, interleaved=inter, amplitude=1.25)
    assert yq.shape == q.shape and yk.shape == k.shape
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == q.dtype
    th = orc.angles(pos, f)
    check_turn(yq, q, th, 1.25, inter)
    check_turn(yk, k, th, 1.25, inter)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rotary(shape, inter, dt):
    B, M, H, Hkv, D, rd = shape
    q, k = make(B, M, H, Hkv, D, DTYPES[dt], seed=D + M, packed=(B + M) % 2 == 0)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    g = gen(2)
    wdt = DTYPES[dt] if inter else torch.float32
    wq, wk = ((1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(wdt).requires_grad_(True)
              for _ in range(2))
    f = api().rotary_frequencies(rd, device="cuda")
    pos = torch.randint(-100, 4096, (B, M), device="cuda", generator=g)
    gq, gk = make(B, M, H, Hkv, D, DTYPES[dt], seed=3)
    y = api().qk_norm_rotary(q, k, wq, wk, pos, f, interleaved=inter, amplitude=0.75, eps=1e-5)
    grads = torch.autograd.grad(y, (q, k, wq, wk), (gq, gk))
    th = orc.angles(pos, f)
    depth = D / 32 + 32
    for x, w, go, yo, dx, dw in ((q, wq, gq, y[0], grads[0], grads[2]),
                                 (k, wk, gk, y[1], grads[1], grads[3])):
        x, w = x.detach(), w.detach()
        u = orc.rms(x, 1e-5) * w.double()
        within(yo.detach(), orc.turn(u, th, 0.75, inter),
               depth * E * 0.75 * orc.pair_size(u, th, inter))
        rx, rw, tx, tw = orc.norm_turn_grads(go, x, w, th, 1e-5, 0.75, inter)
        within(dx, rx, 3 * depth * E * tx)
        assert dw.dtype == wdt
        within(dw, rw, (x.numel() // D + depth) * E * tw)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("inter", [False, True])
def test_more_tokens_than_resident_blocks(inter, dt):
    # a block goes over several tiles, fetching rows of the next ones meanwhile
    test_norm_rotary((1, 5003, 9, 3, 128, 64), inter, dt)
    test_norm_rotary((2, 2501, 7, 1, 80, 80), inter, dt)
    test_rotary((1, 40009, 1, 1, 256, 128), inter, dt)


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("inter", [False, True])
def test_rotary_gradient(inter, dt):
    q, k = make(2, 19, 6, 2, 64, DTYPES[dt], seed=5, packed=True)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    f = api().rotary_frequencies(48, device="cuda")
    pos = torch.arange(19, device="cuda", dtype=torch.int32)
    gq, gk = make(2, 19, 6, 2, 64, DTYPES[dt], seed=6)
    y = api().rotary(q, k, pos, f, interleaved=inter, amplitude=1.5)
    dq, dk = torch.autograd.grad(y, (q, k), (gq, gk))
    th = orc.angles(pos.expand(2, 19), f)
    check_turn(dq, gq, th, 1.5, inter, inverse=True)
    check_turn(dk, gk, th, 1.5, inter, inverse=True)


def test_gradients_against_differences():
    # fp32 gradients along a direction against central differences of the
    # float64 function: h = 2^-13 leaves a truncation of h^2 / 6 of the third
    # derivative along d, taken from a second, doubled step
    B, M, H, D = 2, 5, 3, 64
    q, _ = make(B, M, H, 1, D, torch.float32, seed=7)
    g, d = (make(B, M, H, 1, D, torch.float32, seed=s)[0] for s in (8, 9))
    w = 1 + 0.3 * torch.randn(D, device="cuda", generator=gen(10))
    dw_dir = torch.randn(D, device="cuda", generator=gen(11))
    f = api().rotary_frequencies(D, device="cuda")
    pos = torch.arange(M, device="cuda")
    th = orc.angles(pos.expand(B, M), f)
    q, w = q.requires_grad_(True), w.requires_grad_(True)
    y = api().qk_norm_rotary(q, None, w, None, pos, f, interleaved=True)
    dx, dw = torch.autograd.grad(y, (q, w), g)
    got = float((dx.double() * d.double()).sum() + (dw.double() * dw_dir.double()).sum())

    def loss(h):
        u = orc.rms(q.detach().double() + h * d, 1e-6) * (w.detach().double() + h * dw_dir)
        return float((orc.turn(u, th, 1.0, True) * g.double()).sum())

    h = 2.0 ** -13
    one = (loss(h) - loss(-h)) / (2 * h)
    two = (loss(2 * h) - loss(-2 * h)) / (4 * h)
    ref, trunc = (4 * one - two) / 3, abs(one - two)
    tx, tw = orc.norm_turn_grads(g, q.detach(), w.detach(), th, 1e-6, 1.0, True)[2:]
    slack = E * 200 * float((tx * d.abs()).sum() + (tw * dw_dir.abs()).sum()) + trunc
    assert abs(got - ref) <= slack, (got, ref, slack)


@pytest.mark.parametrize("far", [1 << 20, 1 << 31, 1 << 40])
def test_far_positions_keep_their_angle(far):
    # fp32 outputs at positions where a 32-bit product has no fraction left.
    # float64 angles carry 2^-53 of their radians, on both sides
    q, _ = make(1, 5, 2, 1, 64, torch.float32, seed=1)
    f = api().rotary_frequencies(64, device="cuda")
    pos = far + torch.arange(5, device="cuda").view(1, 5)
    y = api().rotary(q, None, pos, f)
    th = orc.angles(pos, f)
    ps = orc.pair_size(q, th)
    within(y, orc.turn(q, th), (16 * E + 4 * 2.0 ** -53 * far) * ps)


def test_position_forms_and_packed_tokens_agree():
    q, k = make(2, 6, 3, 1, 64, torch.bfloat16)
    f = api().rotary_frequencies(64, device="cuda")
    p1 = torch.arange(6, device="cuda")
    ref = api().rotary(q, k, p1.expand(2, 6).contiguous(), f)
    for pos in (p1, p1[None], p1.int(), p1.expand(2, 6), torch.arange(12, device="cuda")[::2] // 2):
        for a, b in zip(api().rotary(q, k, pos, f), ref):
            assert torch.equal(a, b)
    packed = api().rotary(q.reshape(12, 3, 64), k.reshape(12, 1, 64), p1.repeat(2), f)
    for a, b in zip(packed, ref):
        assert torch.equal(a, b.flatten(0, 1))
    assert torch.equal(api().rotary(q, None, p1, f), ref[0])


def test_strides_read_in_place_or_copied():
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(7, device="cuda")
    base = torch.randn(4, 7, 2, 65, device="cuda", generator=gen(3)).bfloat16()
    w = torch.rand(64, device="cuda", generator=gen(4))
    ws = torch.rand(64, 2, device="cuda", generator=gen(4))[:, 1]
    forms = [base[..., 1:], base[..., :64], base[::2, :, :, :64], base[:, :, :1, :64],
             base[..., :64].transpose(0, 2).contiguous().transpose(0, 2),
             base[:1, :, :, :64].expand(4, 7, 2, 64), base[:, :, :1, :64].expand(4, 7, 3, 64),
             base[..., :64].transpose(2, 3).contiguous().transpose(2, 3)]
    for x in forms:
        assert torch.equal(api().rotary(x, None, pos, f), api().rotary(x.contiguous(), None, pos, f))
        # the sum of squares is taken in another order where vectors do not fit:
        # two orders differ by up to (D / 32 + 6) E relative, which can carry a
        # value over a rounding boundary, so each layout is held to the oracle
        th = orc.angles(pos.expand(x.shape[0], 7), f)
        for ww in (w, ws):
            y = api().qk_norm_rotary(x, None, ww, None, pos, f)
            u = orc.rms(x, 1e-6) * ww.double()
            within(y, orc.turn(u, th), 34 * E * orc.pair_size(u, th))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D", [64, 72])
def test_strides_past_32_bits(D, inter):
    # tokens, and in the other tensor heads, 2^31 + 2^20 entries apart
    far = (1 << 31) + (1 << 20)
    buf = torch.empty(far + (1 << 16), device="cuda", dtype=torch.bfloat16)
    q, k = make(1, 2, 3, 2, D, torch.bfloat16, seed=D)
    fq = buf.as_strided(q.shape, (far * 2, far, D, 1), 0)
    fk = buf.as_strided(k.shape, (far * 2, D, far, 1), 1 << 12)
    fq.copy_(q)
    fk.copy_(k)
    w = 1 + torch.rand(D, device="cuda", generator=gen(3))
    f = api().rotary_frequencies(D - 8 if D == 72 else D, device="cuda")
    pos = torch.tensor([5, 77], device="cuda")
    for call in (lambda a, b: api().rotary(a, b, pos, f, interleaved=inter),
                 lambda a, b: api().qk_norm_rotary(a, b, w, w, pos, f, interleaved=inter)):
        assert all(torch.equal(x, y) for x, y in zip(call(fq, fk), call(q, k)))
    leaf = [t.detach().requires_grad_(True) for t in (fq, fk)]
    near = [t.detach().requires_grad_(True) for t in (q, k)]
    got = torch.autograd.grad(api().qk_norm_rotary(*leaf, w, w, pos, f, interleaved=inter), leaf, (fq, fk))
    want = torch.autograd.grad(api().qk_norm_rotary(*near, w, w, pos, f, interleaved=inter), near, (q, k))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_broadcast_heads_and_gradients():
    # a gradient that is one expanded number, and heads that are one expanded
    # head: their gradient is the sum over the heads
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(4, device="cuda")
    x = torch.randn(1, 4, 1, 64, device="cuda", generator=gen(1)).requires_grad_(True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = api().qk_norm_rotary(x.expand(3, 4, 5, 64), None, w, None, pos, f)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    th = orc.angles(pos.expand(3, 4), f)
    xe = x.detach().expand(3, 4, 5, 64)
    rx, rw, tx, tw = orc.norm_turn_grads(torch.ones_like(xe), xe, w.detach(), th, 1e-6)
    within(dx, rx.sum((0, 2), keepdim=True), 200 * E * tx.sum((0, 2), keepdim=True))
    within(dw, rw, 200 * E * tw)


def test_only_one_output_used():
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(4, device="cuda")
    q, k = (t.requires_grad_(True) for t in make(1, 4, 3, 2, 64, torch.float32))
    wq, wk = (torch.full((64,), v, device="cuda", requires_grad=True) for v in (1.5, 0.5))
    both = torch.autograd.grad([t.sum() for t in api().rotary(q, k, pos, f)], (q, k))
    norm = torch.autograd.grad([t.sum() for t in api().qk_norm_rotary(q, k, wq, wk, pos, f)],
                               (q, k, wq, wk))
    for i in range(2):
        one = torch.autograd.grad(api().rotary(q, k, pos, f)[i].sum(), (q, k), allow_unused=True)
        assert one[1 - i] is None and torch.equal(one[i], both[i])
        one = torch.autograd.grad(api().qk_norm_rotary(q, k, wq, wk, pos, f)[i].sum(),
                                  (q, k, wq, wk), allow_unused=True)
        assert one[1 - i] is None and one[3 - i] is None
        assert torch.equal(one[i], norm[i])
        # a weight's gradient may be added in another order without the other
        # tensor: two orders of n terms differ by at most 2 n E sum |terms|
        x, ww = ((q, wq), (k, wk))[i]
        th = orc.angles(pos.expand(1, 4), f)
        terms = orc.norm_turn_grads(torch.ones_like(x), x.detach(), ww.detach(), th, 1e-6)[3]
        assert ((one[2 + i] - norm[2 + i]).abs() <= 2 * x.numel() // 64 * E * terms).all()
    # a frozen input gets none
    d = torch.autograd.grad(api().rotary(q.detach(), k, pos, f)[1].sum(), k)[0]
    assert torch.equal(d, both[1])


def test_second_derivatives():
    f = api().rotary_frequencies(32, device="cuda")
    pos = torch.arange(3, device="cuda")
    q = make(1, 3, 2, 1, 32, torch.float32)[0].requires_grad_(True)
    y = api().rotary(q, None, pos, f)
    (d,) = torch.autograd.grad((y * y).sum(), q, create_graph=True)  # = 2 q: a rotation keeps lengths
    (dd,) = torch.autograd.grad(d.sum(), q)
    # 16 E of |a| + |b| = 2 in each of the two turns, doubled by the square
    assert (dd - 2).abs().max() <= 256 * E
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = api().qk_norm_rotary(q, None, w, None, pos, f)
    with pytest.raises(RuntimeError):
        (d,) = torch.autograd.grad((y * y).sum(), q, create_graph=True)
        d.sum().backward()


def test_weight_gradient_repeats_bit_for_bit():
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(3001, device="cuda")
    q, k = (t.requires_grad_(True) for t in make(1, 3001, 15, 5, 64, torch.bfloat16))
    w = torch.ones(64, device="cuda", requires_grad=True)
    runs = [torch.autograd.grad([t.float().sum() for t in
                                 api().qk_norm_rotary(q, k, w, w, pos, f)], w)[0] for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
def test_no_tokens(shape):
    B, M = shape
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.zeros(B, M, device="cuda", dtype=torch.long)
    q = torch.empty(B, M, 4, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    assert api().rotary(q, None, pos, f).shape == q.shape
    y = api().qk_norm_rotary(q, None, w, None, pos, f)
    dq, dw = torch.autograd.grad(y.sum(), (q, w))
    assert dq.shape == q.shape and torch.equal(dw, torch.zeros_like(w))


def test_values_at_the_edges():
    # zero heads: the norm is 0 * rsqrt(eps); infinities and NaN stay in their head
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(4, device="cuda")
    q = make(1, 4, 3, 1, 64, torch.bfloat16)[0]
    w = torch.ones(64, device="cuda")
    clean = api().qk_norm_rotary(q, None, w, None, pos, f)
    q2 = q.clone()
    q2[0, 1, 1] = 0
    q2[0, 2, 0, 5] = float("nan")
    q2[0, 3, 2, 7] = float("inf")
    y = api().qk_norm_rotary(q2, None, w, None, pos, f)
    assert torch.equal(y[0, 1, 1], torch.zeros_like(y[0, 1, 1]))
    assert y[0, 2, 0].isnan().all() and y[0, 3, 2].isnan().any()
    same = torch.ones(4, 3, dtype=torch.bool, device="cuda")
    same[1, 1] = same[2, 0] = same[3, 2] = False
    assert torch.equal(y[0][same], clean[0][same])


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", [(96, 32), (128, 64), (70, 34)])
def test_entries_that_are_not_rotated_pass_unchanged(shape, inter, dt):
    D, rd = shape
    f = api().rotary_frequencies(rd, device="cuda")
    pos = torch.arange(4, device="cuda") + 5
    q = make(2, 4, 3, 1, D, DTYPES[dt])[0]
    q[..., rd] = float("inf")
    q[..., rd + 3] = float("nan")
    y = api().rotary(q, None, pos, f, interleaved=inter, amplitude=2.0)
    assert torch.equal(y[..., rd:].nan_to_num(7.0), q[..., rd:].nan_to_num(7.0))
    assert y[..., :rd].isfinite().all()


def test_graph_capture_replays_on_new_inputs():
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(9, device="cuda")
    q, k = (t.requires_grad_(True) for t in make(2, 9, 6, 2, 64, torch.bfloat16))
    w = torch.ones(64, device="cuda", requires_grad=True)

    def step():
        y = api().qk_norm_rotary(q, k, w, w, pos, f)
        return [*y, *torch.autograd.grad(y, (q, k, w), [t.detach() for t in y])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        for t in (q, k):
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen(4)))
        pos.add_(77)
    graph.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_side_stream():
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(50, device="cuda")
    q, k = make(4, 50, 15, 5, 64, torch.bfloat16)
    ref = api().rotary(q, k, pos, f)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = api().rotary(q, k, pos, f)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_compiles_as_one_graph():
    f = api().rotary_frequencies(64, device="cuda")
    pos = torch.arange(5, device="cuda")
    q, k = (t.requires_grad_(True) for t in make(1, 5, 3, 1, 64, torch.float32))
    w = torch.ones(64, device="cuda", requires_grad=True)

    def fn(q, k, w):
        a, b = api_.rotary(q, k, pos, f)
        return api_.qk_norm_rotary(a, b, w, w, pos, f)

    api_ = api()
    ref = fn(q, k, w)
    rg = torch.autograd.grad([t.sum() for t in ref], (q, k, w))
    got = torch.compile(fn, fullgraph=True, backend="aot_eager")(q, k, w)
    gg = torch.autograd.grad([t.sum() for t in got], (q, k, w))
    for a, b in itertools.chain(zip(got, ref), zip(gg, rg)):
        torch.testing.assert_close(a, b, rtol=0, atol=0)


def test_refusals():
    r = api()
    f = r.rotary_frequencies(64, device="cuda")
    pos = torch.arange(4, device="cuda")
    q, k = make(2, 4, 3, 1, 64, torch.bfloat16)
    w = torch.ones(64, device="cuda")
    bad = [
        lambda: r.rotary(q[0, 0], None, pos, f),
        lambda: r.rotary(q.double(), None, pos, f),
        lambda: r.rotary(q, k.float(), pos, f),
        lambda: r.rotary(q, k[:1], pos, f),
        lambda: r.rotary(q, k[..., :32], pos, f),
        lambda: r.rotary(q, k, pos[:3], f),
        lambda: r.rotary(q, k, pos.float(), f),
        lambda: r.rotary(q, k, pos.cpu(), f),
        lambda: r.rotary(q, k, pos, f.float()),
        lambda: r.rotary(q, k, pos, f.cpu()),
        lambda: r.rotary(q[..., :62], None, pos, f),
        lambda: r.rotary(q[..., :63], None, pos, f[:8]),
        lambda: r.rotary(q, k, pos, f[:0]),
        lambda: r.rotary(q, k, pos, f, amplitude=float("nan")),
        lambda: r.rotary(q.cpu(), None, pos, f),
        lambda: r.qk_norm_rotary(q, k, w, None, pos, f),
        lambda: r.qk_norm_rotary(q, k, w[:32], w, pos, f),
        lambda: r.qk_norm_rotary(q, k, w.half(), w.half(), pos, f),
        lambda: r.qk_norm_rotary(q, k, w, w.bfloat16(), pos, f),
        lambda: r.qk_norm_rotary(q, k, w, w.cpu(), pos, f),
        lambda: r.qk_norm_rotary(q, k, w, w, pos, f, eps=-1.0),
        lambda: r.rotary(torch.zeros(1, 4, 1, 1026, device="cuda"), None, pos, f),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
            pytest.fail(f"case {i} was accepted")
