"""Performance cases of attention over rows of voxel features and of the router's
balance loss: the calls a program makes on these operators, over the sizes and
types it makes them with.

Three kinds of case:

* ``attend``  -- ``F.attention`` over packed sequences (scenes, windows of
  serialised voxels, prompts) with grouped heads: whole sequences, forward or
  with all gradients, and few tokens against a cache of keys;
* ``heads``   -- ``F.norm_rotate_heads``: the norm of each head's queries and
  keys and their rotation by positions;
* ``balance`` -- ``F.balance_loss``: the loss that keeps a router's experts in
  use, the experts' counts and the gradient of the logits.

``own`` False computes them from elementary torch operations in 32 bits (angles
in 64), rounded once at the end; True makes the framework's calls.
"""
from __future__ import annotations

import math
import random
from typing import List

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6
_BASE = 10000.0


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _attend(name, sequences, tokens, cache, heads, kv_heads, dim, dtype, causal, train, uneven):
    """``cache``: keys of all sequences, each with room behind them (0: the tokens' own keys);
    ``uneven``: 0 for sequences of one length, or the seed of their lengths."""
    return {"name": name, "op": "attend", "sequences": sequences, "tokens": tokens, "cache": cache, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal, "train": train, "uneven": uneven}


def _heads(name, rows, heads, kv_heads, dim, dtype, axes, far, train):
    return {"name": name, "op": "heads", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "axes": axes, "far": far, "train": train}


def _balance(name, tokens, k, experts, dtype, masked):
    return {"name": name, "op": "balance", "tokens": tokens, "k": k, "experts": experts, "dtype": dtype,
            "masked": masked}


def listed() -> List[dict]:
    return [
        # one token of one sequence against a short cache, where the launches are all there is
        _attend("attend_token_1", 1, 1, 700, 8, 2, 64, "bf16", True, False, 0),
        # a serving step: a token each of 32 sequences, caches of uneven lengths, read once
        _attend("attend_token_32", 32, 32, 131_072, 32, 8, 128, "bf16", True, False, 5),
        # a LiDAR sweep's voxels at the UNet's full-resolution width, in windows of 1024 along the order of
        # their keys, inference
        _attend("attend_voxels_100k", 98, 100_000, 0, 3, 3, 32, "f16", False, False, 0),
        # a few small scans in full precision, an odd width of head, training
        _attend("attend_f32_odd_train", 7, 1_999, 0, 4, 2, 36, "f32", True, True, 3),
        # a long prompt of one sequence
        _attend("attend_prompt_16k", 1, 16_384, 0, 16, 4, 128, "bf16", True, False, 0),
        # a training step of the wide model on sequences packed behind each other, the largest
        _attend("attend_train_16k", 12, 16_384, 0, 16, 4, 64, "bf16", True, True, 4),
        # the heads of a serving step of eight tokens, far into their sequences
        _heads("heads_token_8", 8, 8, 2, 64, "bf16", 1, 1_000_000, False),
        # the heads of a room scan's voxels, rotated by x, y and z, inference
        _heads("heads_voxels_200k", 200_000, 3, 3, 32, "f16", 3, 1_000, False),
        # a training step of the wide model
        _heads("heads_train_16k", 16_384, 16, 4, 64, "bf16", 1, 16_384, True),
        # the router of a small object scan in full precision
        _balance("balance_2k", 2_000, 1, 8, "f32", 0.0),
        # the router on a sweep's voxels, with experts masked out for some of them
        _balance("balance_100k", 100_000, 2, 16, "f16", 0.1),
        # a wide router of many experts
        _balance("balance_wide_16k", 16_384, 8, 256, "bf16", 0.0),
    ]


def draw(rng) -> dict:
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def head_dim():
        return rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128, rng.randrange(2, 129, 2)])

    limit = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["attend", "attend", "attend", "heads", "balance"])
        dtype = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
        train = rng.random() < 0.5
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        if op == "attend":
            sequences = size(1, 100)
            if rng.random() < 0.4:  # few tokens each, against a cache
                tokens, cache, causal, train = sequences * rng.choice([1, 1, 1, 2, 5]), size(sequences * 8, 300_000), True, False
            else:
                tokens, cache, causal = size(sequences, 40_000), 0, rng.random() < 0.6
            case = _attend("", sequences, tokens, cache, heads, kv_heads, head_dim() - (rng.random() < 0.1), dtype,
                           causal, train, rng.choice([0, rng.randrange(1, 10 ** 6)]))
        elif op == "heads":
            axes = rng.choice([1, 1, 3])
            case = _heads("", size(1, 200_000), heads, kv_heads, max(head_dim(), 2 * axes), dtype, axes,
                          size(16, 1_000_000), train)
            if case["rows"] * (heads + kv_heads) * case["dim"] > 4e7:
                continue
        else:
            experts = size(2, 512)
            case = _balance("", size(1, 262_144), rng.randint(1, min(8, experts)), experts, dtype,
                            rng.choice([0.0, 0.0, 0.1, 0.5]))
            if case["tokens"] * experts > 3e7:
                continue
        del case["name"]
        if _cost(case) <= limit:
            return case


def _cost(case):
    """Products, those in 32 bits at the rate that they have on the matrix cores."""
    flops = work(case)["flops"] * (7 if case["dtype"] == "f32" else 1)
    if case["op"] != "attend":
        return flops
    # (no case of many more values than the listed ones)
    _, _, pairs = _lengths(case)
    kept = case["cache"] or case["tokens"]
    values = (case["tokens"] * case["heads"] + 2 * kept * case["kv_heads"]) * case["dim"]
    return math.inf if values > 3e8 or pairs * case["heads"] > 6e9 else flops


def _lengths(case):
    """Queries and keys of each sequence, and the visible pairs of a head."""
    n, rng = case["sequences"], random.Random(case["uneven"])

    def parts(total):
        if not case["uneven"]:
            size = -(-total // n)
            return [max(0, min(size, total - i * size)) for i in range(n)]
        share = [rng.random() ** 2 for _ in range(n)]
        at = [0]
        for s in share:
            at.append(at[-1] + s)
        at = [int(total * a / at[-1]) for a in at]
        at[-1] = total
        return [b - a for a, b in zip(at, at[1:])]

    if case["cache"]:
        queries = [case["tokens"] // n] * n
        keys = [max(k, q) for k, q in zip(parts(case["cache"]), queries)]
    else:
        queries = keys = parts(case["tokens"])
    pairs = sum(q * k - (q * (q - 1) // 2 if case["causal"] else 0) for q, k in zip(queries, keys))
    return queries, keys, pairs


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = _DTYPES[case["dtype"]], case["op"]
    s = dict(case)
    if op == "attend":
        n, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s["queries"], s["keys"], _ = _lengths(case)
        s["offsets"] = _offsets(s["queries"])
        if case["cache"]:
            # (a cache of whole pages of 64 keys and one of them free)
            room = [k // 64 * 64 + 128 for k in s["keys"]]
            s["key_offsets"] = _offsets(room)
            s["key_counts"] = torch.tensor(s["keys"], dtype=torch.int32, device="cuda")
            s["q"] = _normal(g, n, h, d, dtype=dt)
            s["k"], s["v"] = _normal(g, sum(room), hk, d, dtype=dt), _normal(g, sum(room), hk, d, dtype=dt)
            s["starts"] = [sum(room[:i]) for i in range(len(room))]
        else:
            s["key_offsets"] = s["key_counts"] = None
            # (views of one projection, as it gives them)
            x = _normal(g, n, h + 2 * hk, d, dtype=dt)
            s["q"], s["k"], s["v"] = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
            s["starts"] = [sum(s["keys"][:i]) for i in range(len(s["keys"]))]
        s["grad"] = _normal(g, n, h, d, dtype=dt) if case["train"] else None
        leaves = ("q", "k", "v")
    elif op == "heads":
        n, h, hk, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
        x = _normal(g, n, h + 2 * hk, d, dtype=dt, scale=1.5)
        s["q"], s["k"] = x[:, :h], x[:, h:h + hk]
        s["wq"], s["wk"] = 1 + _normal(g, d, dtype=dt, scale=0.1), 1 + _normal(g, d, dtype=dt, scale=0.1)
        shape = (n,) if case["axes"] == 1 else (n, case["axes"])
        s["positions"] = torch.randint(0, case["far"], shape, generator=g, device="cuda", dtype=torch.int32)
        if case["train"]:
            s["gq"], s["gk"] = _normal(g, n, h, d, dtype=dt), _normal(g, n, hk, d, dtype=dt)
        leaves = ("q", "k", "wq", "wk")
    else:
        t, k, e = case["tokens"], case["k"], case["experts"]
        logits = _normal(g, t, e, dtype=torch.float32, scale=1.5) + torch.linspace(1.0, 0.0, e, device="cuda")
        if case["masked"]:
            out = torch.rand(t, e, generator=g, device="cuda") < case["masked"]
            out |= torch.rand(t, 1, generator=g, device="cuda") < case["masked"] / 10
            logits = logits.masked_fill(out, -math.inf)
        s["logits"] = logits.to(dt)
        top, chosen = torch.topk(s["logits"].float(), k, dim=1)
        chosen = torch.where(top > -math.inf, chosen, e)
        ranked, order = torch.sort(chosen.reshape(-1), stable=True)
        s["offsets"] = torch.searchsorted(ranked, torch.arange(e + 1, device="cuda")).to(torch.int32)
        rows = torch.where(ranked < e, order // k, -1).to(torch.int32)
        slots = torch.empty_like(order)
        slots[order] = torch.arange(t * k, device="cuda")
        slots = torch.where(chosen < e, slots.view(t, k), -1).to(torch.int32)
        weights = torch.where(chosen < e, torch.softmax(top, 1), 0)
        s["routes"] = (weights, torch.where(chosen < e, chosen, -1).to(torch.int32), s["offsets"], rows, slots)
        # (the loss's weight; in fp16 with the factor that a training run's scaling of its losses settles at, or
        # the gradients would be below the type's numbers)
        settled = 2.0 ** math.ceil(math.log2(t * e)) if case["dtype"] == "f16" else 1.0
        s["grad"] = torch.full((), 0.01 * settled, device="cuda")
        leaves = ("logits",)
    s["leaves"] = [s[name].detach() for name in leaves]
    if case.get("train", True):
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _RUN_OWN[state["op"]](state) if own else _plain(state)


def _attend_own(s):
    from spira_amd.nn import functional as F
    y = F.attention(*s["leaves"], s["offsets"], key_offsets=s["key_offsets"], key_counts=s["key_counts"],
                    causal=s["causal"])
    return (y, *torch.autograd.grad(y, s["leaves"], s["grad"])) if s["train"] else (y,)


def _heads_own(s):
    from spira_amd.nn import functional as F
    q, k, wq, wk = s["leaves"]
    out = F.norm_rotate_heads(q, k, query_weight=wq, key_weight=wk, positions=s["positions"], base=_BASE, eps=_EPS)
    return (*out, *torch.autograd.grad(out, s["leaves"], (s["gq"], s["gk"]))) if s["train"] else tuple(out)


def _balance_own(s):
    from spira_amd.nn import functional as F
    r = F.balance_loss(s["leaves"][0], F.ExpertRoutes(*s["routes"]))
    return (*r, *torch.autograd.grad(r.loss, s["leaves"], s["grad"]))


_RUN_OWN = {"attend": _attend_own, "heads": _heads_own, "balance": _balance_own}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
@torch.no_grad()
def _plain(s):
    return {"attend": _attend_plain, "heads": _heads_plain, "balance": _balance_plain}[s["op"]](s)


def _attend_plain(s):
    """Products of a sequence and a key head at a time, the group's query heads below each other."""
    dt, (h, hk, d) = s["q"].dtype, (s["heads"], s["kv_heads"], s["dim"])
    group, scale = h // hk, d ** -0.5
    # (the heads in front, as the products take them)
    q, k, v = (s[x].float().transpose(0, 1).contiguous() for x in "qkv")
    y, first = torch.zeros_like(q), 0
    if s["train"]:
        g = s["grad"].float().transpose(0, 1).contiguous()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for nq, nk, start in zip(s["queries"], s["keys"], s["starts"]):
        rows, cols = slice(first, first + nq), slice(start, start + nk)
        first += nq
        if nq == 0 or nk == 0:
            continue
        if s["causal"]:
            hidden = torch.arange(nk, device="cuda") > torch.arange(nk - nq, nk, device="cuda")[:, None]
        for j in range(hk):
            heads = slice(j * group, (j + 1) * group)
            qs, ks, vs = q[heads, rows].reshape(group * nq, d), k[j, cols], v[j, cols]
            p = (qs * scale) @ ks.t()
            if s["causal"]:
                p.view(group, nq, nk).masked_fill_(hidden, -math.inf)
            p = torch.exp(p - p.amax(1, keepdim=True))
            p /= p.sum(1, keepdim=True)
            y[heads, rows] = (p @ vs).view(group, nq, d)
            if s["train"]:
                gs = g[heads, rows].reshape(group * nq, d)
                dv[j, cols] = p.t() @ gs
                dp = gs @ vs.t()
                dp -= (dp * p).sum(1, keepdim=True)
                dp *= p
                dq[heads, rows] = (dp @ ks).view(group, nq, d) * scale
                dk[j, cols] = (dp.t() @ qs) * scale
    out = (y, dq, dk, dv) if s["train"] else (y,)
    return tuple(t.transpose(0, 1).contiguous().to(dt) for t in out)


def _angles(s):
    """[rows, 1, dim / 2]: band a of the pairs turns with axis a."""
    pairs, axes = s["dim"] // 2, s["axes"]
    at = s["positions"].double().view(-1, axes)
    bands = []
    for a in range(axes):
        n = (a + 1) * pairs // axes - a * pairs // axes
        speed = _BASE ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
        bands.append(at[:, a:a + 1] * speed)
    return torch.cat(bands, 1)[:, None]


def _heads_plain(s):
    dt, half = s["q"].dtype, s["dim"] // 2
    turn = _angles(s)
    cos, sin = torch.cos(turn).float(), torch.sin(turn).float()
    out, grads, sums = [], [], []
    for x, w, name in ((s["q"], s["wq"], "gq"), (s["k"], s["wk"], "gk")):
        x, w = x.float(), w.float()
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        hat = x * inv
        n = hat * w
        a, b = n[..., :half], n[..., half:]
        out.append(torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(dt))
        if s["train"]:
            g = s[name].float()
            a, b = g[..., :half], g[..., half:]
            dn = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
            sums.append((dn * hat).sum((0, 1)).to(dt))
            dn = dn * w
            grads.append((inv * (dn - hat * (dn * hat).mean(-1, keepdim=True))).to(dt))
    return (*out, *grads, *sums)


def _balance_plain(s):
    l, e = s["logits"].float(), s["experts"]
    held = l > -math.inf
    some = held.any(1, keepdim=True)
    top = l.amax(1, keepdim=True).masked_fill(~some, 0)
    p = torch.exp(l - top)
    p = torch.where(some, p / p.sum(1, keepdim=True), 0)
    tokens = some.sum().clamp(min=1)
    counts = s["offsets"][1:] - s["offsets"][:-1]
    share = counts.float() / counts.sum().clamp(min=1)
    mean = p.sum(0) / tokens
    loss = e * (share * mean).sum()
    dl = s["grad"] * e / tokens * p * (share - (p * share).sum(1, keepdim=True))
    return loss, counts, mean, dl.to(s["logits"].dtype)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _attend_exact, "heads": _heads_exact, "balance": _balance_exact}[case["op"]](s)


def _attend_exact(s):
    """One head of one sequence at a time, the gradients by differentiation."""
    q, k, v = (s[x].double() for x in "qkv")
    y = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if s["train"] else []
    at = s["offsets"].tolist()
    for b, (start, nk) in enumerate(zip(s["starts"], s["keys"])):
        lo, hi = at[b], at[b + 1]
        if lo == hi or nk == 0:
            continue
        # (query i of n stands at key nk - n + i)
        reach = torch.ones(hi - lo, nk, dtype=torch.bool, device="cuda")
        if s["causal"]:
            reach = reach.tril(nk - (hi - lo))
        for j in range(s["heads"]):
            kj = j // (s["heads"] // s["kv_heads"])
            leaf = [t.contiguous().requires_grad_(s["train"])
                    for t in (q[lo:hi, j], k[start:start + nk, kj], v[start:start + nk, kj])]
            score = leaf[0] @ leaf[1].t().contiguous() / math.sqrt(s["dim"])
            o = torch.softmax(torch.where(reach, score, -math.inf), 1) @ leaf[2]
            y[lo:hi, j] = o.detach()
            if s["train"]:
                d = torch.autograd.grad(o, leaf, s["grad"][lo:hi, j].double())
                grads[0][lo:hi, j] = d[0]
                grads[1][start:start + nk, kj] += d[1]
                grads[2][start:start + nk, kj] += d[2]
            del leaf, score, o
    return (y, *grads)


def _heads_exact(s):
    """Pairs as complex numbers, multiplied by a turn; the gradients by differentiation."""
    leaves = [s[name].double().detach().requires_grad_(s["train"]) for name in ("q", "k", "wq", "wk")]
    half, axes = s["dim"] // 2, s["axes"]
    axis = [a for a in range(axes) for _ in range(a * half // axes, (a + 1) * half // axes)]
    place = [i - axis.index(a) for i, a in enumerate(axis)]
    speed = torch.tensor([_BASE ** (-j / axis.count(a)) for j, a in zip(place, axis)], dtype=torch.float64, device="cuda")
    at = s["positions"].double().view(-1, axes)[:, axis]
    turn = torch.polar(torch.ones_like(at), at * speed)[:, None]
    out = []
    for x, w in ((leaves[0], leaves[2]), (leaves[1], leaves[3])):
        n = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + _EPS) * w
        z = torch.complex(n[..., :half].contiguous(), n[..., half:].contiguous()) * turn
        out.append(torch.cat([z.real, z.imag], -1))
    if not s["train"]:
        return tuple(out)
    grads = torch.autograd.grad(out, leaves, (s["gq"].double(), s["gk"].double()))
    return (*(t.detach() for t in out), *grads)


def _balance_exact(s):
    l = s["logits"].double().detach().requires_grad_(True)
    some = (l > -math.inf).any(1)
    counts = torch.bincount(s["routes"][1].reshape(-1).long() + 1, minlength=s["experts"] + 1)[1:].double()
    if not bool(some.any()):
        zero = torch.zeros_like(counts)
        return zero.sum(), None, zero, torch.zeros_like(l)
    mean = torch.softmax(l[some], 1).mean(0)
    loss = s["experts"] * (counts / counts.sum() * mean).sum()
    (dl,) = torch.autograd.grad(loss, l, s["grad"].double())
    return loss.detach(), None, mean.detach(), dl


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    b, op = _BYTES[case["dtype"]], case["op"]
    if op == "attend":
        queries, keys, pairs = _lengths(case)
        q, kv = sum(queries) * case["heads"] * case["dim"], sum(keys) * case["kv_heads"] * case["dim"]
        forward = b * (2 * q + 2 * kv)
        backward = b * (3 * q + 4 * kv)  # (q, k, v and the gradient read, three gradients written)
        flops = 4.0 * pairs * case["heads"] * case["dim"]
        if not case["train"]:
            return {"bytes": forward, "flops": flops}
        return {"bytes": forward + backward, "flops": 3.5 * flops}
    if op == "heads":
        n, d = case["rows"], case["dim"]
        values = n * (case["heads"] + case["kv_heads"]) * d
        forward = b * (2 * values + 2 * d) + 4 * n * case["axes"]
        backward = b * (3 * values + 4 * d) + 4 * n * case["axes"]
        return {"bytes": forward + backward if case["train"] else forward, "flops": (26.0 if case["train"] else 8.0) * values}
    t, e = case["tokens"], case["experts"]
    return {"bytes": 3 * b * t * e + 12 * e, "flops": 10.0 * t * e}
