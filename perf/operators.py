"""Cases and plain forms of the training-side attention operators.

Three operators of one attention block, in the order a step uses them:

  rotary            position rotation of queries and keys, and its gradient
  norm              per-head RMS norm of queries and keys with the rotation in
                    the same pass, and its gradients (weights included)
  attention         grouped-query attention with its gradients: the forward
                    pass, and a backward pass that recomputes probabilities

``own`` selects the framework's kernels; without it ``run`` computes the same
results from elementary torch operations in 32 bits (angles and long sums in
64), rounded once at the end.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases

def _rotate(name, op, B, M, H, Hkv, D, rd, dtype="bf16", interleaved=False, base=10000.0,
            factor=1.0, far=512, train=False, packed=False):
    return {"name": name, "op": op, "B": B, "M": M, "H": H, "Hkv": Hkv, "D": D, "rd": rd,
            "dtype": dtype, "interleaved": interleaved, "base": base, "factor": factor,
            "far": far, "train": train, "packed": packed}


def _attend(name, B, M, N, H, Hkv, mask="analytic", P=0, ds=0, de=0, lo=0):
    return {"name": name, "op": "attention", "B": B, "M": M, "N": N, "H": H, "Hkv": Hkv,
            "mask": mask, "P": P, "ds": ds, "de": de, "lo": lo}


def listed():
    return [
        # one token of one robot: the latency of a single control step
        _rotate("rotary_step", "rotary", 1, 1, 15, 5, 64, 64),
        # the action expert's 50 action tokens behind a 241-token prefix, one training step
        _rotate("rotary_expert_train", "rotary", 64, 50, 15, 5, 64, 64, train=True),
        # long contexts: part of the head, interleaved pairs, positions scaled down by 16, queries
        # and keys read in place out of one packed projection
        _rotate("rotary_long_scaled", "rotary", 2, 8192, 32, 8, 128, 64, dtype="fp16",
                interleaved=True, factor=16.0, far=131072, packed=True),
        # full precision, an odd batch, a head width whose halves are no whole vectors
        _rotate("rotary_fp32_odd", "rotary", 3, 241, 15, 5, 72, 36, dtype="fp32", train=True),
        # decode of a small batch, one token each
        _rotate("norm_step", "norm", 8, 1, 15, 5, 64, 64, far=8192),
        # the vision-language prefix of a training batch, read from a packed projection
        _rotate("norm_prefix_train", "norm", 64, 241, 15, 5, 64, 64, train=True, packed=True),
        # wide heads, one long ragged sequence, interleaved pairs
        _rotate("norm_wide_train", "norm", 1, 8191, 32, 8, 128, 128, interleaved=True, far=65536,
                train=True),
        # action expert, one sample: latency bound
        _attend("attn_expert_b1", 1, 50, 291, 15, 5, P=241, ds=196, de=240),
        # action expert, a training batch with the padded prefix tokens as a dead band
        _attend("attn_expert_b64", 64, 50, 291, 15, 5, P=241, ds=196, de=240),
        # prefix self-attention, each sample with a length of its own
        _attend("attn_prefix_lengths", 32, 241, 241, 15, 5, mask="lengths", lo=150),
        # vision tower, no mask, no shared heads
        _attend("attn_vision", 4, 1024, 1024, 12, 12, P=1024),
        # a long causal sequence: bound by the tensor cores
        _attend("attn_causal_long", 2, 4096, 4096, 15, 5, P=0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw_rotation(rng, op):
    H, Hkv = rng.choice([(15, 5), (12, 12), (32, 8), (9, 3), (16, 1), (7, 7)])
    D = rng.choice([64, 64, 72, 80, 96, 128, 128, 256])
    rd = rng.choice([D, D, D // 2, D // 4 * 2, 2 * rng.randint(1, D // 2)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    most = 8191 * 40 * 128 // ((H + Hkv) * D * (2 if dtype == "fp32" else 1))
    tokens = _log(rng, 1, most)
    B = min(tokens, _log(rng, 1, 64))
    factor = rng.choice([1.0, 1.0, 4.0, 16.0])
    return {"op": op, "B": B, "M": max(1, tokens // B), "H": H, "Hkv": Hkv, "D": D, "rd": rd,
            "dtype": dtype, "interleaved": rng.random() < 0.4, "base": rng.choice([10000.0, 500000.0]),
            "factor": factor, "far": _log(rng, 16, 1 << 20), "train": rng.random() < 0.6,
            "packed": rng.random() < 0.4}


def draw(rng):
    op = rng.choice(["rotary", "norm", "attention", "attention"])
    if op != "attention":
        return _draw_rotation(rng, op)
    H, Hkv = rng.choice([(15, 5), (12, 12), (8, 1), (16, 4), (9, 3), (7, 7), (6, 2)])
    N = _log(rng, 1, 4096)
    mask = rng.choice(["analytic", "analytic", "lengths", "bool"])
    if mask == "lengths" or rng.random() < 0.5:
        M = N
    else:
        M = _log(rng, 1, 4096)
    most = min(4096 * 4096 * 15 // (H * M * N), 2 * 4096 * 20 // (H * M + Hkv * N))
    B = _log(rng, 1, max(1, min(64, most)))
    P = ds = de = 0
    if mask == "analytic":
        P = rng.choice([0, N, rng.randint(0, N)])
        if rng.random() < 0.5:
            ds, de = sorted((rng.randint(0, P), rng.randint(0, P)))
    return {"op": op, "B": B, "M": M, "N": N, "H": H, "Hkv": Hkv, "mask": mask, "P": P, "ds": ds,
            "de": de, "lo": rng.randint(min(N, 2), N) if mask == "lengths" else 0}


# ---------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    c, B, M, H, Hkv = case, case["B"], case["M"], case["H"], case["Hkv"]
    if c["op"] == "attention":
        N, bf = c["N"], torch.bfloat16
        s = {"case": c, "q": randn(B, M, H, 64, dtype=bf), "k": randn(B, N, Hkv, 64, dtype=bf),
             "v": randn(B, N, Hkv, 64, dtype=bf), "do": randn(B, M, H, 64, dtype=bf),
             "lengths": None, "mask": None}
        for name in ("q", "k", "v"):
            s[name].requires_grad_(True)
        if c["mask"] == "lengths":
            s["lengths"] = torch.randint(c["lo"], N + 1, (B,), device="cuda", generator=g)
        if c["mask"] == "bool":
            m = torch.rand(B, M, N, device="cuda", generator=g) < 0.7
            s["mask"] = m & (torch.rand(B, M, 1, device="cuda", generator=g) < 0.95)
        return s
    D, rd, dt = c["D"], c["rd"], DTYPES[c["dtype"]]
    if c["packed"]:  # queries, keys and values of one projection, read in place
        x = randn(B, M, H + 2 * Hkv, D, dtype=dt)
        q, k = x[:, :, :H], x[:, :, H:H + Hkv]
    else:
        q, k = randn(B, M, H, D, dtype=dt), randn(B, M, Hkv, D, dtype=dt)
    first = torch.randint(0, max(1, c["far"] - M), (B, 1), device="cuda", generator=g)
    pos = first + torch.arange(M, device="cuda")
    # the plan a program keeps: radians per position, and the amplitude that goes with scaling
    e = torch.arange(rd // 2, device="cuda", dtype=torch.float64) * (-2.0 / rd)
    s = {"case": c, "q": q, "k": k, "pos": pos, "freq": torch.pow(c["base"], e) / c["factor"],
         "amp": 1.0 + 0.1 * math.log(c["factor"]), "gq": None, "gk": None, "wq": None, "wk": None}
    if c["op"] == "norm":
        s["wq"], s["wk"] = 1.0 + 0.2 * randn(D), 1.0 + 0.2 * randn(D)
    if c["train"]:
        s["gq"], s["gk"] = randn(B, M, H, D, dtype=dt), randn(B, M, Hkv, D, dtype=dt)
        s["q"], s["k"] = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        if c["op"] == "norm":
            s["wq"].requires_grad_(True)
            s["wk"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# plain forms

EPS = 1e-6


def _angles(s):
    a = s["pos"].double()[:, :, None] * s["freq"]
    return (a.cos() * s["amp"]).float()[:, :, None], (a.sin() * s["amp"]).float()[:, :, None]


def _turn(x, cos, sin, rd, interleaved):
    """Rotate the first rd entries of the last axis by the angles; the rest pass through."""
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2],
                                                                 x[..., rd // 2:rd])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = _angles(s)
    out = [_turn(s["q"].detach().float(), cos, sin, c["rd"], c["interleaved"]).to(s["q"].dtype),
           _turn(s["k"].detach().float(), cos, sin, c["rd"], c["interleaved"]).to(s["k"].dtype)]
    if c["train"]:  # the transpose of a rotation turns the other way
        out += [_turn(s["gq"].float(), cos, -sin, c["rd"], c["interleaved"]).to(s["q"].dtype),
                _turn(s["gk"].float(), cos, -sin, c["rd"], c["interleaved"]).to(s["k"].dtype)]
    return out


def _plain_norm_one(s, x, w, grad, cos, sin):
    c = s["case"]
    xf, wf = x.detach().float(), w.detach()
    r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + EPS)
    hat = xf * r
    y = _turn(hat * wf, cos, sin, c["rd"], c["interleaved"]).to(x.dtype)
    if grad is None:
        return y, None, None
    t = _turn(grad.float(), cos, -sin, c["rd"], c["interleaved"])
    dw = (t * hat).double().sum((0, 1, 2)).float()
    t = t * wf
    dx = r * (t - hat * (t * hat).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), dw


def _plain_norm(s):
    cos, sin = _angles(s)
    yq, dq, dwq = _plain_norm_one(s, s["q"], s["wq"], s["gq"], cos, sin)
    yk, dk, dwk = _plain_norm_one(s, s["k"], s["wk"], s["gk"], cos, sin)
    return [yq, yk, dq, dk, dwq, dwk] if s["case"]["train"] else [yq, yk]


def _visible(s):
    """(B or 1, 1, 1, M, N): whether query row r sees key col."""
    c = s["case"]
    if s["mask"] is not None:
        return s["mask"][:, None, None]
    r = torch.arange(c["M"], device="cuda")[:, None]
    col = torch.arange(c["N"], device="cuda")
    if s["lengths"] is not None:
        L = s["lengths"][:, None, None]
        return ((col < L) & (r < L))[:, None, None]
    vis = torch.where(col < c["P"], (col < c["ds"]) | (col >= c["de"]),
                      col <= c["N"] - c["M"] + r)
    return vis[None, None, None]


def _plain_attention(s):
    c = s["case"]
    B, M, N, H, Hkv = c["B"], c["M"], c["N"], c["H"], c["Hkv"]
    G, scale = H // Hkv, 0.125

    def rows(x):  # (B, M, H, 64) -> (B, Hkv, G * M, 64)
        return x.float().view(B, M, Hkv, G, 64).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * M, 64)

    def back(x):
        return x.view(B, Hkv, G, M, 64).permute(0, 3, 1, 2, 4).reshape(B, M, H, 64).bfloat16()

    q, do = rows(s["q"].detach()), rows(s["do"])
    k, v = (s[n].detach().float().transpose(1, 2) for n in ("k", "v"))
    p = (q @ k.transpose(2, 3)).mul_(scale).view(B, Hkv, G, M, N)
    p.masked_fill_(~_visible(s), -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_min_(-1e30)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-30))
    p = p.view(B, Hkv, G * M, N)
    o, dv = p @ v, p.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = dp @ k, dp.transpose(2, 3) @ q
    return [back(o), back(dq), dk.transpose(1, 2).bfloat16().contiguous(),
            dv.transpose(1, 2).bfloat16().contiguous()]


# ---------------------------------------------------------------------------
# the framework's calls

def _package():
    root = os.path.join(os.getcwd(), "vla-kernels_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


def _own(s):
    _package()
    c = s["case"]
    if c["op"] == "attention":
        from kernels.attention import fused_attention_gqa_train

        how = {"attn_mask": s["mask"]} if s["mask"] is not None else \
            {"lengths": s["lengths"]} if s["lengths"] is not None else \
            {"prefix_len": c["P"], "dead_start": c["ds"], "dead_end": c["de"]}
        o = fused_attention_gqa_train(s["q"], s["k"], s["v"], **how)
        return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])]
    from kernels.rotary import qk_norm_rotary, rotary

    if c["op"] == "rotary":
        y = rotary(s["q"], s["k"], s["pos"], s["freq"], interleaved=c["interleaved"],
                   amplitude=s["amp"])
        wrt = (s["q"], s["k"])
    else:
        y = qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["freq"], eps=EPS,
                           interleaved=c["interleaved"], amplitude=s["amp"])
        wrt = (s["q"], s["k"], s["wq"], s["wk"])
    if not c["train"]:
        return list(y)
    return [*y, *torch.autograd.grad(y, wrt, (s["gq"], s["gk"]))]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    with torch.no_grad():
        return (_plain_attention if op == "attention" else
                _plain_norm if op == "norm" else _plain_rotary)(state)


# ---------------------------------------------------------------------------
# work: inputs read once, outputs written once, products of the visible pairs

def _pairs(c):
    """Visible (row, key) pairs of one head, over the batch (lengths and random masks: expected)."""
    B, M, N = c["B"], c["M"], c["N"]
    if c["mask"] == "lengths":
        n = N + 1 - c["lo"]
        return B * sum(x * x for x in range(c["lo"], N + 1)) // n
    if c["mask"] == "bool":
        return int(B * M * N * 0.7 * 0.95)
    stairs = sum(max(0, min(N, N - M + r + 1) - c["P"]) for r in range(M))
    return B * (M * (c["P"] - c["de"] + c["ds"]) + stairs)


def work(case):
    c = case
    if c["op"] == "attention":
        q, kv = c["B"] * c["M"] * c["H"] * 128, c["B"] * c["N"] * c["Hkv"] * 128
        extra = c["B"] * c["M"] * c["N"] if c["mask"] == "bool" else 0
        # q, do, k, v in; o, dq, dk, dv out. Products: two forward, four backward (the
        # probabilities' recomputation is not counted)
        return {"bytes": 4 * q + 4 * kv + extra, "flops": 12 * 64 * c["H"] * _pairs(c)}
    size = 4 if c["dtype"] == "fp32" else 2
    n = c["B"] * c["M"] * (c["H"] + c["Hkv"]) * c["D"]
    each = (10 if c["op"] == "norm" else 3) * (3 if c["train"] else 1)
    return {"bytes": n * size * (4 if c["train"] else 2) + 8 * c["B"] * c["M"], "flops": n * each}


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits

def _exact_turn(s, x):
    """The rotation as a product with unit complex numbers of the angles."""
    c, rd = s["case"], s["case"]["rd"]
    turn = torch.polar(torch.full_like(s["freq"], s["amp"]).expand(*s["pos"].shape, rd // 2)
                       .contiguous(), s["pos"].double()[..., None] * s["freq"])[:, :, None]
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :rd].unflatten(-1, (rd // 2, 2)).contiguous()) * turn
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :rd // 2].contiguous(), x[..., rd // 2:rd].contiguous()) * turn
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., rd:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    leaf = {n: s[n].detach().double().requires_grad_(True)
            for n in ("q", "k", "v", "wq", "wk") if s.get(n) is not None}
    if case["op"] == "attention":
        G = case["H"] // case["Hkv"]
        k, v = (leaf[n].repeat_interleave(G, 2) for n in ("k", "v"))
        z = torch.einsum("bmhd,bnhd->bhmn", leaf["q"], k) / 8.0
        seen = _visible(s)[:, :, 0]
        z = z.masked_fill(~seen, -math.inf)
        p = torch.softmax(z.masked_fill(~seen.any(-1, keepdim=True), 0.0), -1)
        o = torch.einsum("bhmn,bnhd->bmhd", p * seen, v)
        got = torch.autograd.grad(o, (leaf["q"], leaf["k"], leaf["v"]), s["do"].double())
        return [o.detach(), *got]
    out = []
    for n, w in (("q", "wq"), ("k", "wk")):
        x = leaf[n]
        if case["op"] == "norm":
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + EPS) * leaf[w]
        out.append(_exact_turn(s, x))
    if not case["train"]:
        return [y.detach() for y in out]
    wrt = [leaf[n] for n in (("q", "k", "wq", "wk") if case["op"] == "norm" else ("q", "k"))]
    got = torch.autograd.grad(out, wrt, (s["gq"].double(), s["gk"].double()))
    return [y.detach() for y in out] + list(got)
