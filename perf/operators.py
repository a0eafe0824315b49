"""Three operators of a training step, through the framework's public entry points, and their plain forms.

``norm``   layer norm (``ops.layer_norm``), alone as for a single token or with its backward as in training
``moe``    tokens sorted by expert and back (``ops.moe.sort_by_expert``, ``permute_tokens``, ``unpermute_tokens``), the way of a MoE layer's
           tokens to its experts and home, alone as in serving or with its gradients as in training
``orth``   orthogonalising a matrix by Newton-Schulz products (``ops.muon.newton_schulz``)
``muon``   one optimiser step of a weight with its momentum, orthogonalised update, decay and bf16 copy (``ops.muon.muon_step``)

A case is a dict of plain values. ``prepare`` makes what a program holds before the call, ``run`` is one pass of the call: with ``own`` the
framework's kernels, without it elementary torch operations in 32 bits. ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-5
# the step sizes of the decoder's configuration; five products with the coefficients that lift small singular values fastest
_LR, _DECAY, _MOMENTUM = 3e-4, 0.1, 0.95
_STEPS, _COEFF, _NORM_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


# ------------------------------------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one token's row of the 4096-wide decoder: what a call costs
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "param": "bf16", "train": False},
        # a ragged fp32 batch whose rows start at odd addresses
        {"name": "norm_ragged_fp32", "kind": "norm", "rows": 1333, "cols": 1001, "dtype": "fp32", "param": "fp32", "train": True},
        # two sequences of 4096 tokens of the 4096-wide decoder, forward and backward; fp32 gain and bias beside bf16 activations
        {"name": "norm_train", "kind": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "param": "fp32", "train": True},
        # a long batch at the width of the tensor-parallel block
        {"name": "norm_train_long", "kind": "norm", "rows": 16384, "cols": 8192, "dtype": "bf16", "param": "bf16", "train": True},
        # one token on its way to 8 of 256 experts and back: serving, latency
        {"name": "moe_token", "kind": "moe", "tokens": 1, "hidden": 7168, "experts": 256, "topk": 8, "dtype": "bf16", "drop": False, "train": False},
        # the default MoE configuration, forward and backward
        {"name": "moe_default", "kind": "moe", "tokens": 1024, "hidden": 1024, "experts": 8, "topk": 2, "dtype": "bf16", "drop": False, "train": True},
        # fp32 tokens of an odd width, a tenth of the assignments dropped for capacity (some tokens keep no expert)
        {"name": "moe_ragged_fp32", "kind": "moe", "tokens": 1333, "hidden": 1001, "experts": 32, "topk": 4, "dtype": "fp32", "drop": True, "train": True},
        # 8192 tokens per rank, top-8 of 256 experts, 7168 wide, forward and backward
        {"name": "moe_large", "kind": "moe", "tokens": 8192, "hidden": 7168, "experts": 256, "topk": 8, "dtype": "bf16", "drop": False, "train": True},
        # a small odd matrix, as of an adapter or a router
        {"name": "orth_odd", "kind": "orth", "batch": 1, "rows": 333, "cols": 1000, "dtype": "fp32"},
        # the down projections of the default MoE configuration's experts, in one call
        {"name": "orth_experts", "kind": "orth", "batch": 8, "rows": 1024, "cols": 128, "dtype": "bf16"},
        # the attention output projection of the 8B-shaped decoder
        {"name": "muon_square", "kind": "muon", "batch": 1, "rows": 4096, "cols": 4096, "dtype": "bf16"},
        # its gate and up projection, the largest matrix of a layer
        {"name": "muon_gate_up", "kind": "muon", "batch": 1, "rows": 28672, "cols": 4096, "dtype": "bf16"},
    ]


def _log_int(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_any(rng) -> dict:
    kind = rng.choice(["norm", "moe", "orth", "muon"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "norm":        # any number of rows; half of the widths are multiples of 8, as models have them
        cols = _log_int(rng, 8, 16384)
        return {"kind": kind, "rows": _log_int(rng, 1, 16384), "cols": cols // 8 * 8 if rng.random() < 0.5 else cols, "dtype": dtype,
                "param": rng.choice(["fp32", dtype]), "train": rng.random() < 0.6}
    if kind == "moe":
        hidden, experts = _log_int(rng, 64, 7168), rng.choice([8, 16, 32, 64, 128, 256])
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192), "hidden": hidden // 8 * 8 if rng.random() < 0.7 else hidden, "experts": experts,
                "topk": rng.choice([1, 2, 4, 8]), "dtype": dtype, "drop": rng.random() < 0.3, "train": rng.random() < 0.6}
    batch = rng.choice([1, 1, 1, 2, 4, 8])
    return {"kind": kind, "batch": batch, "rows": _log_int(rng, 16, 16384), "cols": _log_int(rng, 16, 16384), "dtype": dtype}


def draw(rng) -> dict:
    """One more case of the same ranges, at most as large as the largest listed one of its kind (of either kind for the two that orthogonalise)."""
    most = {}
    for c in listed():
        w, k = work(c), "muon" if c["kind"] == "orth" else c["kind"]
        f, b = most.get(k, (0.0, 0.0))
        most[k] = (max(f, w["flops"]), max(b, w["bytes"]))
    while True:
        c = _draw_any(rng)
        w = work(c)
        f, b = most["muon" if c["kind"] == "orth" else c["kind"]]
        if w["flops"] <= f and w["bytes"] <= b:
            return c


# ------------------------------------------------------------------------------------------------ what a program holds
def _rand(shape, gen, dtype, std: float = 1.0, mean: float = 0.0) -> torch.Tensor:
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=gen).mul_(std).add_(mean).to(dtype)


def _prepare_norm(c, gen):
    shape, dt, pt = (c["rows"], c["cols"]), _DTYPE[c["dtype"]], _DTYPE[c["param"]]
    # a residual stream: channels of different scales and a common offset
    x = torch.randn(*shape, device="cuda", generator=gen)
    x.mul_(torch.rand(c["cols"], device="cuda", generator=gen).mul_(2).add_(0.1)).add_(0.5)
    s = {"x": x.to(dt), "gamma": _rand((c["cols"],), gen, pt, 0.1, 1.0), "beta": _rand((c["cols"],), gen, pt, 0.1)}
    s["dy"] = _rand(shape, gen, dt) if c["train"] else None
    return s


def _prepare_moe(c, gen):
    t, h, e, k, dt = c["tokens"], c["hidden"], c["experts"], c["topk"], _DTYPE[c["dtype"]]
    # experts are not equally popular
    logits = torch.randn(t, e, device="cuda", generator=gen) + 0.7 * torch.randn(e, device="cuda", generator=gen)
    gates, idx = torch.topk(torch.softmax(logits, -1), k, -1)
    idx = idx.to(torch.int32)
    if c["drop"]:
        lost = torch.rand(t, k, device="cuda", generator=gen) < 0.1
        lost |= torch.rand(t, 1, device="cuda", generator=gen) < 0.02
        idx = torch.where(lost, torch.full_like(idx, -1), idx)
    s = {"x": _rand((t, h), gen, dt), "idx": idx.contiguous(), "gates": gates.contiguous(), "experts": e, "y": _rand((t * k, h), gen, dt)}
    s["dout"], s["dxp"] = (_rand((t, h), gen, dt), _rand((t * k, h), gen, dt)) if c["train"] else (None, None)
    return s


def _matrix(c, gen):
    """A gradient: a few directions that carry most of it, over noise."""
    b, m, n = c["batch"], c["rows"], c["cols"]
    r = max(1, min(m, n, 64) // 4)
    g = torch.randn(b, m, n, device="cuda", generator=gen)
    u, v = torch.randn(b, m, r, device="cuda", generator=gen), torch.randn(b, r, n, device="cuda", generator=gen)
    v.mul_(torch.arange(1, r + 1, device="cuda", dtype=torch.float32).rsqrt()[:, None])
    return g.add_(u @ v).mul_(1e-3)


def _prepare_orth(c, gen):
    return {"g": _matrix(c, gen).to(_DTYPE[c["dtype"]])}


def _prepare_muon(c, gen):
    p = _rand((c["batch"], c["rows"], c["cols"]), gen, torch.float32, 0.02)
    return {"p": p, "m": _matrix(c, gen).mul_(4.0), "g": _matrix(c, gen).to(_DTYPE[c["dtype"]]), "p_bf16": p.to(torch.bfloat16)}


_PREPARE = {"norm": _prepare_norm, "moe": _prepare_moe, "orth": _prepare_orth, "muon": _prepare_muon}


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    return {"kind": case["kind"], **_PREPARE[case["kind"]](case, gen)}


# ------------------------------------------------------------------------------------------------ one pass: the framework's calls
def _own_norm(s):
    from parallelkernelbench_b200.ops import layer_norm, layer_norm_bwd, layer_norm_fwd

    if s["dy"] is None:
        return {"y": layer_norm(s["x"], s["gamma"], s["beta"], _EPS)}
    y, mean, rstd = layer_norm_fwd(s["x"], s["gamma"], s["beta"], _EPS)
    dx, dgamma, dbeta = layer_norm_bwd(s["x"], s["gamma"], s["dy"], mean, rstd)
    return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _own_moe(s):
    from parallelkernelbench_b200.ops.moe import permute_tokens, permute_tokens_bwd, sort_by_expert, unpermute_tokens, unpermute_tokens_bwd

    srt = sort_by_expert(s["idx"], s["experts"])
    out = {"offsets": srt.offsets, "order": srt.order, "slots": srt.slots, "xp": permute_tokens(s["x"], srt),
           "out": unpermute_tokens(s["y"], srt, s["gates"])}
    if s["dout"] is not None:
        out["dy"], out["dgates"] = unpermute_tokens_bwd(s["dout"], s["y"], srt, s["gates"])
        out["dx"] = permute_tokens_bwd(s["dxp"], srt)
    return out


def _own_orth(s):
    from parallelkernelbench_b200.ops.muon import newton_schulz

    return {"o": newton_schulz(s["g"], steps=_STEPS, coefficients=_COEFF, eps=_NORM_EPS)}


def _own_muon(s):
    from parallelkernelbench_b200.ops.muon import muon_step

    muon_step(s["p"], s["m"], s["g"], lr=_LR, momentum=_MOMENTUM, nesterov=True, weight_decay=_DECAY, steps=_STEPS, coefficients=_COEFF,
              eps=_NORM_EPS, p_bf16=s["p_bf16"])
    return {"p": s["p"], "m": s["m"], "p_bf16": s["p_bf16"]}


# ------------------------------------------------------------------------------------------------ one pass: the plain forms
def _plain_norm(s):
    x, gamma = s["x"].float(), s["gamma"].float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    xhat = c * rstd
    y = (xhat * gamma + s["beta"].float()).to(s["x"].dtype)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * gamma
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx.to(s["x"].dtype), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}


def _plain_moe(s):
    idx, e, dt = s["idx"], s["experts"], s["x"].dtype
    t, k = idx.shape
    key = torch.where((idx >= 0) & (idx < e), idx, e).view(-1)
    skey, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(skey, torch.arange(e + 1, device=key.device, dtype=key.dtype))
    row = torch.arange(t * k, device=key.device)
    slots = torch.empty_like(row)
    slots[order] = torch.where(skey < e, row, -1)
    kept, there = (skey < e)[:, None], (slots >= 0).view(t, k, 1)
    src = slots.clamp(min=0).view(t, k)
    out = {"offsets": offsets.to(torch.int32), "order": torch.where(skey < e, order, -1).to(torch.int32), "slots": slots.to(torch.int32)}
    out["xp"] = torch.where(kept, s["x"][order // k], 0)
    y = torch.where(there, s["y"][src].float(), 0)
    out["out"] = (y * s["gates"][:, :, None]).sum(1).to(dt)
    if s["dout"] is not None:
        dout = s["dout"].float()
        out["dgates"] = (y * dout[:, None, :]).sum(-1)
        del y
        out["dy"] = torch.where(kept, dout[order // k] * s["gates"].view(-1)[order][:, None], 0).to(dt)
        out["dx"] = torch.where(there, s["dxp"][src].float(), 0).sum(1).to(dt)
    return out


def _plain_newton_schulz(u):
    a, b, c = _COEFF
    wide = u.shape[-2] <= u.shape[-1]
    x = u if wide else u.transpose(-1, -2)
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + _NORM_EPS)
    for _ in range(_STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if wide else x.transpose(-1, -2)


def _plain_orth(s):
    return {"o": _plain_newton_schulz(s["g"].float()).to(torch.bfloat16)}


def _plain_muon(s):
    p, m, g = s["p"], s["m"], s["g"].float()
    m.mul_(_MOMENTUM).add_(g)
    o = _plain_newton_schulz(g + _MOMENTUM * m)
    p.mul_(1 - _LR * _DECAY).sub_(o * (_LR * 0.2 * math.sqrt(max(p.shape[-2:]))))
    s["p_bf16"].copy_(p)
    return {"p": p, "m": m, "p_bf16": s["p_bf16"]}


def run(state: dict):
    kind = state["kind"]
    if own:
        return {"norm": _own_norm, "moe": _own_moe, "orth": _own_orth, "muon": _own_muon}[kind](state)
    return {"norm": _plain_norm, "moe": _plain_moe, "orth": _plain_orth, "muon": _plain_muon}[kind](state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_norm(s):
    x, gamma, beta = s["x"].double(), s["gamma"].double(), s["beta"].double()
    n = x.shape[1]
    mean = x.sum(1) / n
    var = torch.einsum("rc,rc->r", x, x) / n - mean * mean
    rstd = 1 / torch.sqrt(var + _EPS)
    xhat = torch.addcmul(-(mean * rstd)[:, None], x, rstd[:, None])
    y = torch.addcmul(beta, xhat, gamma)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].double()
    c1, c2 = (dy @ gamma) / n, torch.einsum("rc,rc,c->r", dy, xhat, gamma) / n
    dx = (dy * gamma - c1[:, None] - xhat * c2[:, None]) * rstd[:, None]
    return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dgamma": torch.einsum("rc,rc->c", dy, xhat), "dbeta": dy.sum(0)}


def _exact_moe(s):
    idx, e = s["idx"].long(), s["experts"]
    t, k = idx.shape
    flat = idx.reshape(-1)
    flat = torch.where((flat < 0) | (flat >= e), torch.full_like(flat, e), flat)
    n = t * k
    at = torch.arange(n, device=flat.device)
    order = (torch.sort(flat * n + at).values % n)                       # unique keys: expert first, then position
    counts = torch.zeros(e + 1, dtype=torch.long, device=flat.device).index_add_(0, flat, torch.ones_like(flat))[:e]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    keep = int(offsets[-1])                                              # rows behind it have no assignment
    live = order[:keep]
    slots = torch.full((n,), -1, dtype=torch.long, device=flat.device)
    slots[live] = at[:keep]
    res = {"offsets": offsets.int(), "order": torch.cat([live, live.new_full((n - keep,), -1)]).int(), "slots": slots.int()}

    def rows(v):
        return torch.cat([v, v.new_zeros((n - keep, *v.shape[1:]))])

    tok, gate = live // k, s["gates"].double().reshape(-1)[live]
    res["xp"] = rows(s["x"].double()[tok])
    y = s["y"].double()[:keep]
    zero = torch.zeros(t, y.shape[1], dtype=torch.float64, device=y.device)
    res["out"] = zero.index_add(0, tok, y * gate[:, None])
    if s["dout"] is not None:
        dout = s["dout"].double()[tok]
        res["dgates"] = torch.zeros(n, dtype=torch.float64, device=y.device).index_copy(0, live, torch.einsum("rc,rc->r", y, dout)).view(t, k)
        res["dy"] = rows(dout.mul_(gate[:, None]))
        res["dx"] = zero.index_add(0, tok, s["dxp"].double()[:keep])
    return res


def _exact_newton_schulz(u):
    """X (a + b A + c A^2) by its smaller Gram matrix, by Horner's rule."""
    a, b, c = _COEFF
    x = u / (torch.linalg.vector_norm(u, dim=(-2, -1), keepdim=True) + _NORM_EPS)
    tall = x.shape[-2] > x.shape[-1]
    eye = torch.eye(min(x.shape[-2:]), dtype=x.dtype, device=x.device)
    for _ in range(_STEPS):
        gram = x.mT @ x if tall else x @ x.mT
        poly = a * eye + gram @ (b * eye + c * gram)
        x = x @ poly if tall else poly @ x
    return x


def _exact_orth(s):
    return {"o": _exact_newton_schulz(s["g"].double())}


def _exact_muon(s):
    g = s["g"].double()
    m = _MOMENTUM * s["m"].double() + g
    o = _exact_newton_schulz(g + _MOMENTUM * m)
    p = s["p"].double() * (1 - _LR * _DECAY) - _LR * 0.2 * math.sqrt(max(g.shape[-2:])) * o
    return {"p": p, "m": m, "p_bf16": p}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "moe": _exact_moe, "orth": _exact_orth, "muon": _exact_muon}[case["kind"]](s)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    c, kind = case, case["kind"]
    size = {"bf16": 2, "fp32": 4}
    if kind == "norm":
        r, n, s, ps = c["rows"], c["cols"], size[c["dtype"]], size[c["param"]]
        if not c["train"]:
            return {"bytes": 2.0 * r * n * s + 2.0 * n * ps, "flops": 8.0 * r * n}
        return {"bytes": 4.0 * r * n * s + 2.0 * n * ps + 8.0 * n + 8.0 * r, "flops": 20.0 * r * n}
    if kind == "moe":
        t, h, k, s = c["tokens"], c["hidden"], c["topk"], size[c["dtype"]]
        whole = 8.0 * t * k + 4.0 * t * k + 4.0 * t * k + 4.0 * (c["experts"] + 1)       # experts and gates, slots, order, offsets
        forward = 2.0 * t * h * s + 2.0 * t * k * h * s                                  # x, out; xp, y
        if not c["train"]:
            return {"bytes": whole + forward, "flops": 2.0 * t * k * h}
        return {"bytes": whole + forward + 2.0 * t * h * s + 2.0 * t * k * h * s + 4.0 * t * k, "flops": 6.0 * t * k * h}
    b, m, n = c["batch"], min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
    # two symmetric products of which one triangle is enough, and the product with X
    flops = b * _STEPS * (float(m) * (m + 1) * n + float(m) * m * (m + 1) + 2.0 * m * m * n)
    g = size[c["dtype"]]
    return {"bytes": float(b) * m * n * (g + 2.0 if kind == "orth" else g + 18.0), "flops": flops}
