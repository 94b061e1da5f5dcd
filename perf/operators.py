"""Performance cases of the mixture-of-experts block over rows of voxel features:
the calls a program makes on its operators, over the sizes and types it makes
them with.

Five kinds of case:

* ``linear``  -- ``F.grouped_linear``, products grouped by expert with ragged
  sizes: rows gathered from the tokens or already in expert order, forward or
  with all gradients;
* ``route``   -- ``F.route_experts``: the choice of experts, the rows' order and
  the gradient of the logits;
* ``combine`` -- ``F.combine_experts``: the experts' rows added up per token;
* ``norm``    -- ``F.gated_residual_norm``: the norm behind a block, its gate, the
  residual sum and the next block's norm;
* ``dropout`` -- ``F.dropout`` from a counter-based generator.

``own`` False computes them from elementary torch operations in 32 bits,
rounded once at the end; True makes the framework's calls.
"""
from __future__ import annotations

import math
from typing import List

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _linear(name, tokens, k, experts, cin, cout, dtype, gather, relu, train, idle=0.0):
    return {"name": name, "op": "linear", "tokens": tokens, "k": k, "experts": experts, "cin": cin, "cout": cout,
            "dtype": dtype, "gather": gather, "relu": relu, "train": train, "idle": idle}


def _route(name, tokens, k, experts, dtype, renormalize, train, masked):
    return {"name": name, "op": "route", "tokens": tokens, "k": k, "experts": experts, "dtype": dtype,
            "renormalize": renormalize, "train": train, "masked": masked}


def _combine(name, tokens, k, experts, channels, dtype, train, idle=0.0):
    return {"name": name, "op": "combine", "tokens": tokens, "k": k, "experts": experts, "channels": channels,
            "dtype": dtype, "train": train, "idle": idle}


def _norm(name, rows, channels, dtype, gate, sigmoid, train):
    return {"name": name, "op": "norm", "rows": rows, "channels": channels, "dtype": dtype, "gate": gate,
            "sigmoid": sigmoid, "train": train}


def _dropout(name, rows, channels, dtype, p, residual, train):
    return {"name": name, "op": "dropout", "rows": rows, "channels": channels, "dtype": dtype, "p": p,
            "residual": residual, "train": train}


def listed() -> List[dict]:
    return [
        # a serving step of eight queries: few rows, every expert's weights read for one or two of them
        _linear("linear_serve_8", 8, 2, 32, 512, 2048, "bf16", True, True, False),
        # the first expert layer on the voxels of a LiDAR sweep at the UNet's full-resolution width, inference
        _linear("linear_voxels_100k", 100_000, 2, 8, 96, 384, "f16", True, True, False),
        # a small object scan in full precision, rows in expert order, odd widths, a few points without an expert
        _linear("linear_f32_odd_train", 19_999, 1, 4, 63, 130, "f32", False, False, True, 0.05),
        # a training step of a wide expert layer: forward and every gradient, the largest products
        _linear("linear_train_16k", 16_384, 2, 16, 1024, 2048, "bf16", True, True, True),
        # the router of the serving step
        _route("route_serve_8", 8, 2, 32, "bf16", True, False, 0.0),
        # the router in training on a sweep's voxels, with experts masked out for some of them
        _route("route_train_100k", 100_000, 2, 16, "f16", True, True, 0.1),
        # the experts' rows of a sweep added up per voxel, with the gradients
        _combine("combine_train_100k", 100_000, 2, 8, 96, "f16", True),
        # one query's block exit and next entry, where the launch is all there is
        _norm("norm_serve_1", 1, 512, "bf16", "channel", False, False),
        # block exit and next entry on a room scan's voxels, inference, a learned scale per channel
        _norm("norm_voxels_200k", 200_000, 96, "f16", "channel", False, False),
        # the same in a training step of the wide model, gated by a sigmoid of its own tensor
        _norm("norm_train_16k", 16_384, 1024, "bf16", "full", True, True),
        # dropout before the residual sum on a room scan's voxels
        _dropout("dropout_voxels_200k", 200_000, 96, "f16", 0.1, True, False),
        # dropout and its gradient in a training step of the wide model
        _dropout("dropout_train_16k", 16_384, 1024, "bf16", 0.1, False, True),
    ]


def draw(rng) -> dict:
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):
        w = size(lo, hi)
        return max(lo, w // 32 * 32) if w >= 32 and rng.random() < 0.6 else w

    limit = 6.0 * 2 * 16_384 * 1024 * 2048
    while True:
        op = rng.choice(["linear", "linear", "linear", "route", "combine", "norm", "norm", "dropout"])
        dtype = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
        train = rng.random() < 0.5
        if op == "linear":
            experts = size(2, 64)
            case = _linear("", size(1, 131_072), rng.randint(1, min(4, experts)), experts, width(16, 2048),
                           width(16, 2048), dtype, rng.random() < 0.5, rng.random() < 0.5, train,
                           rng.choice([0.0, 0.0, 0.1]))
            # (a sum that rounds to the other side of zero changes the gradients by a whole term, more than
            # 32-bit outputs are compared to)
            case["relu"] &= not (train and dtype == "f32")
            if case["tokens"] * case["k"] * max(case["cin"], case["cout"]) > 7e7:
                continue
        elif op == "route":
            experts = size(2, 256)
            case = _route("", size(1, 262_144), rng.randint(1, min(8, experts)), experts, dtype, rng.random() < 0.7,
                          train, rng.choice([0.0, 0.0, 0.1, 0.5]))
            if case["tokens"] * experts > 3e7:
                continue
        elif op == "combine":
            experts = size(2, 64)
            case = _combine("", size(1, 131_072), rng.randint(1, min(4, experts)), experts, width(16, 2048), dtype,
                            train, rng.choice([0.0, 0.0, 0.1]))
            if case["tokens"] * case["k"] * case["channels"] > 7e7:
                continue
        elif op == "norm":
            case = _norm("", size(1, 300_000), width(16, 4096), dtype, rng.choice(["none", "channel", "row", "full"]),
                         rng.random() < 0.5, train)
            if case["rows"] * case["channels"] > 4e7:
                continue
        else:
            case = _dropout("", size(1, 300_000), width(16, 4096), dtype, rng.choice([0.05, 0.1, 0.5]),
                            rng.random() < 0.5, train)
            if case["rows"] * case["channels"] > 4e7:
                continue
        del case["name"]
        if work(case)["flops"] <= limit and 3072 not in case.values():
            return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _assignments(g, tokens, k, experts, idle):
    """A router's plan for uneven experts: weights, experts, offsets, rows, slots."""
    lean = torch.linspace(1.0, 0.0, experts, device="cuda")
    score = torch.randn(tokens, experts, generator=g, device="cuda") + lean
    chosen = torch.topk(score, k, dim=1).indices
    if idle:
        none = torch.rand(tokens, generator=g, device="cuda") < idle
        chosen = torch.where(none[:, None], torch.full_like(chosen, -1), chosen)
    weights = torch.rand(tokens, k, generator=g, device="cuda") + 0.1
    weights = torch.where(chosen < 0, torch.zeros_like(weights), weights / weights.sum(1, keepdim=True))
    return (weights, *_order(chosen, experts))


def _order(chosen, experts):
    tokens, k = chosen.shape
    flat = torch.where(chosen < 0, experts, chosen).reshape(-1)
    ranked, order = torch.sort(flat, stable=True)
    bounds = torch.arange(experts + 1, device=flat.device)
    offsets = torch.searchsorted(ranked, bounds).to(torch.int32)
    rows = torch.where(ranked < experts, order // k, -1).to(torch.int32)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(tokens * k, device=flat.device)
    slots = torch.where(flat < experts, slots, -1).reshape(tokens, k).to(torch.int32)
    return chosen.to(torch.int32), offsets, rows, slots


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _DTYPES[case["dtype"]], case["op"]
    s = dict(case)
    if op in ("linear", "combine"):
        s["weights"], s["experts_of"], s["offsets"], s["rows_of"], s["slots"] = _assignments(
            g, case["tokens"], case["k"], case["experts"], case["idle"])
    if op == "linear":
        n = case["tokens"] if case["gather"] else case["tokens"] * case["k"]
        s["x"] = _normal(g, n, case["cin"], dtype=dt)
        s["w"] = _normal(g, case["experts"], case["cin"], case["cout"], dtype=dt, scale=case["cin"] ** -0.5)
        s["b"] = _normal(g, case["experts"], case["cout"], dtype=dt, scale=0.1)
        s["grad"] = _normal(g, case["tokens"] * case["k"], case["cout"], dtype=dt) if case["train"] else None
        leaves = ("x", "w", "b")
    elif op == "route":
        logits = _normal(g, case["tokens"], case["experts"], dtype=torch.float32, scale=1.5)
        if case["masked"]:
            out = torch.rand(logits.shape, generator=g, device="cuda") < case["masked"]
            out |= torch.rand(case["tokens"], 1, generator=g, device="cuda") < case["masked"] / 10
            logits = logits.masked_fill(out, -math.inf)
        s["logits"] = logits.to(dt)
        s["grad"] = _normal(g, case["tokens"], case["k"], dtype=torch.float32) if case["train"] else None
        leaves = ("logits",)
    elif op == "combine":
        s["x"] = _normal(g, case["tokens"] * case["k"], case["channels"], dtype=dt)
        s["grad"] = _normal(g, case["tokens"], case["channels"], dtype=dt) if case["train"] else None
        leaves = ("x", "weights")
    elif op == "norm":
        n, c = case["rows"], case["channels"]
        s["x"], s["h"] = _normal(g, n, c, dtype=dt, scale=2.0), _normal(g, n, c, dtype=dt)
        s["w_post"] = 1 + _normal(g, c, dtype=dt, scale=0.1)
        s["w_next"] = 1 + _normal(g, c, dtype=dt, scale=0.1)
        shape = {"none": None, "channel": (c,), "row": (n, 1), "full": (n, c)}[case["gate"]]
        s["gate_form"], s["gate"] = case["gate"], None if shape is None else _normal(g, *shape, dtype=dt)
        s["scale"] = 0.5
        if case["train"]:
            s["grad"], s["grad_next"] = _normal(g, n, c, dtype=dt), _normal(g, n, c, dtype=dt)
        leaves = ("x", "h", "w_post", "w_next", "gate")
    else:
        s["x"] = _normal(g, case["rows"], case["channels"], dtype=dt)
        s["residual_in"] = _normal(g, case["rows"], case["channels"], dtype=dt) if case["residual"] else None
        s["grad"] = _normal(g, case["rows"], case["channels"], dtype=dt) if case["train"] else None
        # (a training run's generator state: its seed and how far it has come)
        s["seed"], s["offset"] = (0x9E3779B97F4A7C15 + seed * 0x1000003) % 2 ** 64, (1 << 33) + seed
        leaves = ("x",)
    s["leaves"] = [s[name] for name in leaves if s[name] is not None]
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _RUN_OWN[state["op"]](state) if own else _plain(state)


def _linear_own(s):
    from spira_amd.nn import functional as F
    groups = s["offsets"]
    if s["gather"]:
        groups = F.ExpertRoutes(s["weights"], s["experts_of"], s["offsets"], s["rows_of"], s["slots"])
    y = F.grouped_linear(s["x"], s["w"], groups, bias=s["b"], relu=s["relu"])
    return (y, *torch.autograd.grad(y, s["leaves"], s["grad"])) if s["train"] else (y,)


def _route_own(s):
    from spira_amd.nn import functional as F
    r = F.route_experts(s["logits"], s["k"], renormalize=s["renormalize"])
    if s["train"]:
        return (*r, *torch.autograd.grad(r.weights, s["leaves"], s["grad"]))
    return tuple(r)


def _combine_own(s):
    from spira_amd.nn import functional as F
    y = F.combine_experts(s["x"], F.ExpertRoutes(s["weights"], s["experts_of"], s["offsets"], s["rows_of"], s["slots"]))
    return (y, *torch.autograd.grad(y, s["leaves"], s["grad"])) if s["train"] else (y,)


def _norm_own(s):
    from spira_amd.nn import functional as F
    r, n = F.gated_residual_norm(s["x"], s["h"], weight=s["w_post"], gate=s["gate"], gate_sigmoid=s["sigmoid"],
                                 scale=s["scale"], next_weight=s["w_next"], eps=_EPS)
    return (r, n, *torch.autograd.grad((r, n), s["leaves"], (s["grad"], s["grad_next"]))) if s["train"] else (r, n)


def _dropout_own(s):
    from spira_amd.nn import functional as F
    y = F.dropout(s["x"], s["p"], s["seed"], s["offset"], residual=s["residual_in"])
    return (y, *torch.autograd.grad(y, s["leaves"], s["grad"])) if s["train"] else (y,)


_RUN_OWN = {"linear": _linear_own, "route": _route_own, "combine": _combine_own, "norm": _norm_own,
            "dropout": _dropout_own}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
@torch.no_grad()
def _plain(s):
    return {"linear": _linear_plain, "route": _route_plain, "combine": _combine_plain, "norm": _norm_plain,
            "dropout": _dropout_plain}[s["op"]](s)


def _linear_plain(s):
    """The groups padded to the longest one, then products over the experts at once."""
    dt, offsets = s["x"].dtype, s["offsets"].long()
    experts, cin, cout = s["w"].shape
    r = torch.arange(s["tokens"] * s["k"], device="cuda")
    e = torch.searchsorted(offsets[1:], r, right=True)
    held = e < experts
    e = e.clamp(max=experts - 1)
    cap = max(1, int((offsets[1:] - offsets[:-1]).max()))
    at = torch.where(held, e * cap + r - offsets[e], experts * cap)  # (the row past the last: no group's)

    def padded(v):
        return v.new_zeros(experts * cap + 1, v.shape[1]).index_copy_(0, at, v.masked_fill(~held[:, None], 0))

    def ragged(v):
        return torch.cat([v.reshape(experts * cap, -1), v.new_zeros(1, v.shape[-1])]).index_select(0, at)

    x, w = s["x"].float(), s["w"].float()
    if s["gather"]:
        x = x.index_select(0, s["rows_of"].long().clamp(min=0))
    xp = padded(x)[:-1].view(experts, cap, cin)
    z = torch.bmm(xp, w) + s["b"].float()[:, None]
    y = ragged(z.clamp(min=0) if s["relu"] else z)
    if not s["train"]:
        return (y.to(dt),)
    dz = padded(s["grad"].float())[:-1].view(experts, cap, cout)
    if s["relu"]:
        dz = dz * (z > 0)
    dx = ragged(torch.bmm(dz, w.transpose(1, 2).contiguous()))
    if s["gather"]:
        slots = s["slots"].long()
        dx = (dx[slots.clamp(min=0)] * (slots >= 0)[:, :, None]).sum(1)
    dw = torch.bmm(xp.transpose(1, 2).contiguous(), dz)
    return y.to(dt), dx.to(dt), dw.to(dt), dz.sum(1).to(dt)


def _route_plain(s):
    logits = s["logits"].float()
    value, chosen = torch.sort(logits, dim=1, descending=True, stable=True)
    value, chosen = value[:, :s["k"]], chosen[:, :s["k"]]
    held = value > -math.inf
    top = value[:, :1].masked_fill(~held[:, :1], 0)
    num = torch.exp(value - top)
    den = num.sum(1, keepdim=True) if s["renormalize"] else torch.exp(logits - top).sum(1, keepdim=True)
    weights = torch.where(held, num / den, 0)
    out = (weights, *_order(torch.where(held, chosen, -1), s["experts"]))
    if not s["train"]:
        return out
    d = s["grad"].masked_fill(~held, 0)
    mean = (d * weights).sum(1, keepdim=True)
    if s["renormalize"]:
        dl = torch.zeros_like(logits).scatter_(1, chosen, weights * (d - mean))
    else:
        p = torch.where(logits > -math.inf, torch.exp(logits - top) / den, 0)
        dl = p * (torch.zeros_like(logits).scatter_(1, chosen, d) - mean)
    return (*out, dl.to(s["logits"].dtype))


def _combine_plain(s):
    slots, w, x = s["slots"].long(), s["weights"], s["x"].float()
    at = slots.clamp(min=0)
    taken = torch.where((slots >= 0)[:, :, None], x[at], 0)
    y = (w[:, :, None] * taken).sum(1)
    if not s["train"]:
        return (y.to(s["x"].dtype),)
    g = s["grad"].float()
    dw = (taken * g[:, None]).sum(2)
    dx = x.new_zeros(x.shape[0] + 1, x.shape[1])
    dx[torch.where(slots >= 0, slots, x.shape[0])] = w[:, :, None] * g[:, None]
    return y.to(s["x"].dtype), dx[:-1].to(s["x"].dtype), dw


def _norm_plain(s):
    dt, x, h = s["x"].dtype, s["x"].float(), s["h"].float()
    wp, wn = s["w_post"].float(), s["w_next"].float()
    rh = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    hh = h * rh
    z = hh * wp
    g = 1.0 if s["gate"] is None else s["gate"].float()
    raw = g
    if s["gate"] is not None and s["sigmoid"]:
        g = 1 / (1 + torch.exp(-raw))
    r = x + s["scale"] * g * z
    rr = torch.rsqrt((r * r).mean(1, keepdim=True) + _EPS)
    rhat = r * rr
    n = rhat * wn
    if not s["train"]:
        return r.to(dt), n.to(dt)
    dn = s["grad_next"].float()
    dx = s["grad"].float() + rr * (dn * wn - rhat * (dn * wn * rhat).mean(1, keepdim=True))
    dz = s["scale"] * g * dx
    dh = rh * (dz * wp - hh * (dz * wp * hh).mean(1, keepdim=True))
    out = [r.to(dt), n.to(dt), dx.to(dt), dh.to(dt), (dz * hh).sum(0).to(dt), (dn * rhat).sum(0).to(dt)]
    if s["gate"] is not None:
        dg = s["scale"] * z * dx
        if s["sigmoid"]:
            dg = dg * g * (1 - g)
        out.append({"channel": lambda: dg.sum(0), "row": lambda: dg.sum(1, keepdim=True),
                    "full": lambda: dg}[s["gate_form"]]().to(dt))
    return tuple(out)


def _product(a, b):
    """(high, low) 32 bits of the product of 32-bit values held in int64."""
    p, q = a * (b & 0xFFFF), a * (b >> 16)
    return (q + (p >> 16)) >> 16, (p + ((q & 0xFFFF) << 16)) & 0xFFFFFFFF


def _keep_plain(count, p, seed, offset):
    """Philox-4x32 with 7 rounds (Salmon et al., SC 2011): counter (i / 4, offset), key seed."""
    i = torch.arange((count + 3) // 4, device="cuda")
    c0, c1 = i & 0xFFFFFFFF, i >> 32
    c2, c3 = torch.full_like(i, offset & 0xFFFFFFFF), torch.full_like(i, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(7):
        h0, l0 = _product(c0, 0xD2511F53)
        h1, l1 = _product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:count] >= int(p * 2 ** 32)


def _dropout_plain(s):
    keep = _keep_plain(s["x"].numel(), s["p"], s["seed"], s["offset"]).view(s["x"].shape)
    y = torch.where(keep, s["x"].float() * (1 / (1 - s["p"])), 0)
    if s["residual_in"] is not None:
        y = y + s["residual_in"].float()
    if not s["train"]:
        return (y.to(s["x"].dtype),)
    return y.to(s["x"].dtype), torch.where(keep, s["grad"].float() * (1 / (1 - s["p"])), 0).to(s["x"].dtype)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "route" and case["tokens"] * case["experts"] * case["k"] > 6e7:
        return None
    s = prepare(case, seed)
    for t in s["leaves"]:
        t.requires_grad_(False)
    return {"linear": _linear_exact, "route": _route_exact, "combine": _combine_exact, "norm": _norm_exact,
            "dropout": _dropout_exact}[case["op"]](s)


def _linear_exact(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    bounds = s["offsets"].tolist()
    y = torch.zeros(s["tokens"] * s["k"], s["cout"], dtype=torch.float64, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for e in range(s["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        source = s["rows_of"][lo:hi].long() if s["gather"] else torch.arange(lo, hi, device="cuda")
        z = x[source] @ w[e] + b[e]
        y[lo:hi] = torch.relu(z) if s["relu"] else z
        if s["train"]:
            dz = s["grad"][lo:hi].double()
            if s["relu"]:
                dz[z <= 0] = 0
            dx.index_add_(0, source, dz @ w[e].T)
            dw[e] = x[source].T @ dz
            db[e] = dz.sum(0)
    return (y, dx, dw, db) if s["train"] else (y,)


def _route_exact(s):
    l = s["logits"].double().cpu()
    chosen = torch.full((s["tokens"], s["k"]), -1)
    left = l.clone()
    for j in range(s["k"]):  # (the first of the largest, one at a time)
        at = (left == left.max(1, keepdim=True).values).to(torch.uint8).argmax(1)
        there = left.gather(1, at[:, None])[:, 0] > -math.inf
        chosen[:, j] = torch.where(there, at, -1)
        left.scatter_(1, at[:, None], -math.inf)
    held = chosen >= 0
    picked = torch.where(held, l.gather(1, chosen.clamp(min=0)), -math.inf)
    over = picked if s["renormalize"] else l
    total = torch.logsumexp(over, 1, keepdim=True)
    w = torch.where(held, torch.exp(picked - total), 0.0)
    out = [w, None, None, None, None]
    if s["train"]:
        d = torch.where(held, s["grad"].double().cpu(), 0.0)
        full = torch.zeros(s["tokens"], s["experts"] + 1, dtype=torch.float64)
        full.scatter_(1, torch.where(held, chosen, s["experts"]), d)
        if s["renormalize"]:
            p = torch.zeros_like(full).scatter_(1, torch.where(held, chosen, s["experts"]), w)[:, :-1]
        else:
            p = torch.where(l > -math.inf, torch.exp(l - total), 0.0)
        out.append(p * (full[:, :-1] - (p * full[:, :-1]).sum(1, keepdim=True)))
    return tuple(out)


def _combine_exact(s):
    x, w, slots = s["x"].double(), s["weights"].double(), s["slots"].long()
    y = torch.zeros(s["tokens"], s["channels"], dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for j in range(s["k"]):
        t = torch.nonzero(slots[:, j] >= 0)[:, 0]
        at = slots[t, j]
        y[t] += w[t, j, None] * x[at]
        if s["train"]:
            dy = s["grad"][t].double()
            dx[at] = w[t, j, None] * dy
            dw[t, j] = (x[at] * dy).sum(1)
    return (y, dx, dw) if s["train"] else (y,)


def _norm_exact(s):
    """The gradients by differentiation of the formula in 64 bits."""
    leaves = {k: s[k].double().requires_grad_(True) for k in ("x", "h", "w_post", "w_next", "gate") if s[k] is not None}
    x, h = leaves["x"], leaves["h"]
    z = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + _EPS) * leaves["w_post"]
    if "gate" in leaves:
        z = z * (torch.sigmoid(leaves["gate"]) if s["sigmoid"] else leaves["gate"])
    r = x + s["scale"] * z
    n = r / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + _EPS) * leaves["w_next"]
    if not s["train"]:
        return r.detach(), n.detach()
    grads = torch.autograd.grad((r, n), list(leaves.values()), (s["grad"].double(), s["grad_next"].double()))
    return (r.detach(), n.detach(), *grads)


def _dropout_exact(s):
    u = np.uint64
    count, low = s["x"].numel(), u(0xFFFFFFFF)
    c = np.zeros(((count + 3) // 4, 4), u)
    c[:, 0] = np.arange(len(c), dtype=u)
    c[:, 2], c[:, 3] = s["offset"] & 0xFFFFFFFF, s["offset"] >> 32
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for _ in range(7):
        a, b = c[:, 0] * u(0xD2511F53), c[:, 2] * u(0xCD9E8D57)
        c = np.stack([(b >> u(32)) ^ c[:, 1] ^ u(key[0]), b & low, (a >> u(32)) ^ c[:, 3] ^ u(key[1]), a & low], 1)
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    keep = torch.from_numpy((c.reshape(-1)[:count] >= u(int(s["p"] * 2 ** 32))).reshape(tuple(s["x"].shape)))

    def thinned(v):
        v = v.double().cpu() / (1 - s["p"])
        v[~keep] = 0
        return v

    y = thinned(s["x"])
    if s["residual_in"] is not None:
        y = y + s["residual_in"].double().cpu()
    return (y, thinned(s["grad"])) if s["train"] else (y,)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    b, op = _BYTES[case["dtype"]], case["op"]
    if op == "linear":
        t, r, ci, co = case["tokens"], case["tokens"] * case["k"], case["cin"], case["cout"]
        # (the experts that some token has chosen, were the choice even)
        used = case["experts"] * (1 - (1 - case["k"] / case["experts"]) ** t)
        x = (t if case["gather"] else r) * ci
        index = 4 * (case["experts"] + 1 + (r if case["gather"] else 0))
        forward = b * (x + used * (ci + 1) * co + r * co) + index
        backward = b * (2 * x + used * ci * co + (2 if case["relu"] else 1) * r * co
                        + case["experts"] * (ci + 1) * co) + index
        flops = 2.0 * r * ci * co
        return {"bytes": forward + backward if case["train"] else forward, "flops": flops * (3 if case["train"] else 1)}
    if op == "route":
        t, k, e = case["tokens"], case["k"], case["experts"]
        forward = b * t * e + 16 * t * k + 4 * (e + 1)
        backward = b * t * e + 4 * t * k + 12 * t * k  # (dlogits written; gradient, weights and experts read)
        return {"bytes": forward + backward if case["train"] else forward, "flops": 4.0 * t * e}
    if op == "combine":
        t, r, c = case["tokens"], case["tokens"] * case["k"], case["channels"]
        forward = b * (r + t) * c + 8 * r
        backward = b * (t + 2 * r) * c + 12 * r
        return {"bytes": forward + backward if case["train"] else forward, "flops": 2.0 * r * c * (3 if case["train"] else 1)}
    n, c = case["rows"], case["channels"]
    if op == "norm":
        gate = {"none": 0, "channel": c, "row": n, "full": n * c}[case["gate"]]
        forward = b * (4 * n * c + gate + 2 * c)
        backward = b * (6 * n * c + 2 * gate + 4 * c)
        return {"bytes": forward + backward if case["train"] else forward,
                "flops": (10.0 + (26 if case["train"] else 0)) * n * c}
    forward = b * n * c * (3 if case["residual"] else 2)
    return {"bytes": forward + (b * n * c * 2 if case["train"] else 0), "flops": 2.0 * n * c * (2 if case["train"] else 1)}
