"""What stands between two routed layers, as measurable cases: the choice of experts (softmax or sigmoid scores, a bias for
balance, groups of experts, renormalised weights) and its gradient, the norms before and after a block with its gate and
residual, and their gradient, and the clip of many gradients by their global norm.

A case is a dict of plain values.  `listed()` holds the fixed ones, `draw(rng)` one more of the same ranges;
`prepare(case, seed)` makes what a program holds before the call, `run(state)` is one pass, through the library's entry
points where `own` is set and in elementary torch operations where it is not, `work(case)` the bytes and operations the
pass cannot do without, and `exact(case, seed)` the pass's result in 64 bits, written apart from both.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def _route(name, rows, experts, topk, dtype, score, bias, groups, taken, group_top, renormalize, scale, mask):
    return dict(name=name, kind="route", rows=rows, experts=experts, topk=topk, dtype=dtype, score=score, bias=bias,
                groups=groups, taken=taken, group_top=group_top, renormalize=renormalize, scale=scale, mask=mask)


def _route_bwd(name, rows, experts, topk, dtype, score, renormalize, scale, mask):
    return dict(name=name, kind="route_backward", rows=rows, experts=experts, topk=topk, dtype=dtype, score=score,
                renormalize=renormalize, scale=scale, mask=mask)


def _norm(name, kind, rows, width, dtype, residual, post, pre, gate, wdtype, offset, residual_scale, block_scale):
    return dict(name=name, kind=kind, rows=rows, width=width, dtype=dtype, residual=residual, post=post, pre=pre, gate=gate,
                wdtype=wdtype, offset=offset, residual_scale=residual_scale, block_scale=block_scale)


def _clip(name, layers, hidden, inter, experts, vocab, dtype):
    return dict(name=name, kind="clip", layers=layers, hidden=hidden, inter=inter, experts=experts, vocab=vocab, dtype=dtype)


def listed():
    return [
        # a decode batch's choice of 8 among 256 experts, out of the best 4 of 8 groups: latency
        _route("route_32rows_e256_top8_of_4_groups", 32, 256, 8, "f32", "sigmoid", True, 8, 4, 2, True, 2.5, False),
        # one sequence through a layer of 60 experts whose scores keep their softmax values
        _route("route_2047rows_e60_top4_softmax", 2047, 60, 4, "bf16", "softmax", False, 1, 1, 1, False, 1.0, False),
        # a training step's padded batch, grouped and with the balance bias
        _route("route_65521rows_e256_top8_of_4_groups", 65521, 256, 8, "bf16", "sigmoid", True, 8, 4, 2, True, 2.5, True),
        # the gradient of a short micro-batch's softmax scores, not renormalised: a whole row each
        _route_bwd("route_gradient_333rows_e160_top6_softmax", 333, 160, 6, "f16", "softmax", False, 16.0, False),
        # the gradient of the training step's padded batch
        _route_bwd("route_gradient_65521rows_e256_top8_sigmoid", 65521, 256, 8, "bf16", "sigmoid", True, 2.5, True),
        # one token between two blocks: the norm after, the residual, the norm before the next: latency
        _norm("norm_1row_4096_post_pre", "norm", 1, 4096, "bf16", "bf16", True, True, "none", "bf16", 0.0, 1.0, 1.0),
        # a prompt's rows onto a 32-bit residual stream, a gate of one value a channel
        _norm("norm_2047rows_5120_gated", "norm", 2047, 5120, "f16", "f32", False, True, "channel", "f32", 0.0, 1.0, 0.22),
        # a training step's rows, both norms with weights around zero, a gate of one value a token
        _norm("norm_16384rows_4096_post_pre", "norm", 16384, 4096, "bf16", "bf16", True, True, "row", "bf16", 1.0, 1.0, 1.0),
        # the gradient of a ragged micro-batch through the gate, the pre norm alone
        _norm("norm_gradient_333rows_2560_gated", "norm_backward", 333, 2560, "f16", "f32", False, True, "channel", "f32",
              0.0, 1.0, 0.22),
        # the gradient of the training step's rows
        _norm("norm_gradient_16384rows_4096_post_pre", "norm_backward", 16384, 4096, "bf16", "bf16", True, True, "row",
              "bf16", 1.0, 1.0, 1.0),
        # the biases, norm weights and router of one layer: latency and launches
        _clip("clip_1layer_h2048", 1, 2048, 768, 60, 0, "f32"),
        # those of 32 layers in 16 and 32 bits, and an embedding
        _clip("clip_32layers_h4096_vocab", 32, 4096, 14336, 128, 65521, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges: routers of 1 .. 65536 rows and 8 to 512 experts in 1 to 16 groups, norms of
    1 .. 16384 rows of 128 .. 8192 values, odd widths among them, and the gradients of 1 to 48 layers."""
    kind = rng.choice(["route", "route", "route_backward", "norm", "norm", "norm_backward", "clip"])
    if kind in ("route", "route_backward"):
        experts = rng.choice([8, 16, 60, 64, 100, 128, 160, 256, 384, 512])
        topk = rng.choice([1, 2, 4, 6, 8])
        c = dict(kind=kind, rows=min(_log(rng, 1, 65536), 65536 * 256 // experts), experts=experts, topk=topk,
                 dtype=rng.choice(["f32", "bf16", "f16"]), score=rng.choice(["softmax", "sigmoid"]),
                 renormalize=rng.random() < 0.6, scale=rng.choice([1.0, 2.5, 16.0]), mask=rng.random() < 0.4)
        if kind == "route_backward":
            return c
        groups = rng.choice([g for g in (1, 1, 4, 8, 16) if experts % g == 0 and experts // g >= 2])
        taken = rng.randint(-(-topk * groups // experts), groups)
        return dict(c, bias=rng.random() < 0.6, groups=groups, taken=taken, group_top=rng.choice([1, 2]) if groups > 1 else 1)
    if kind == "clip":
        return dict(kind=kind, layers=rng.choice([1, 2, 7, 24, 48]), hidden=_log(rng, 512, 4096), inter=_log(rng, 512, 14336),
                    experts=rng.choice([8, 60, 128]), vocab=rng.choice([0, 0, 1001, 32000]), dtype=rng.choice(["f32", "bf16", "f16"]))
    width = rng.choice([8 * _log(rng, 16, 1024), _log(rng, 128, 8192)])
    rows = min(_log(rng, 1, 16384), 16384 * 4096 // width)
    dtype = rng.choice(["bf16", "f16", "bf16", "f32"])
    post = rng.random() < 0.6
    return dict(kind=kind, rows=rows, width=width, dtype=dtype, residual=rng.choice([dtype, "f32"]), post=post,
                pre=not post or rng.random() < 0.8, gate=rng.choice(["none", "channel", "row", "full"]),
                wdtype=rng.choice([dtype, "f32"]), offset=rng.choice([0.0, 1.0]), residual_scale=rng.choice([1.0, 0.5]),
                block_scale=rng.choice([1.0, 0.22]))


# ---------------------------------------------------------------------------------------------------------------
# Inputs


def _route_inputs(case, g):
    rows, E, k = case["rows"], case["experts"], case["topk"]
    # a trained router's logits: each expert at a level of its own
    logits = torch.randn(rows, E, device=DEV, generator=g) + torch.randn(E, device=DEV, generator=g) * 0.5
    s = dict(logits=logits.to(DTYPES[case["dtype"]]), mask=None)
    if case["mask"]:
        s["mask"] = torch.rand(rows, device=DEV, generator=g) < 0.8
    if case["kind"] == "route":
        # the bias a balancing rule has moved by steps of a thousandth
        s["bias"] = torch.randint(-150, 151, (E,), device=DEV, generator=g).float() * 1e-3 if case["bias"] else None
        return s
    s["inds"] = torch.topk(s["logits"].float(), k, dim=-1).indices.int()
    if case["mask"]:  # slots that an expert's capacity dropped
        s["inds"] = torch.where(torch.rand(rows, k, device=DEV, generator=g) < 0.02, -1, s["inds"])
    s["dscores"] = torch.randn(rows, k, device=DEV, generator=g)
    return s


def _norm_inputs(case, g):
    rows, D = case["rows"], case["width"]
    T, R, W = DTYPES[case["dtype"]], DTYPES[case["residual"]], DTYPES[case["wdtype"]]
    normal = lambda *n: torch.randn(*n, device=DEV, generator=g)  # noqa: E731
    weight = lambda on: (1 - case["offset"] + 0.2 * normal(D)).to(W) if on else None  # noqa: E731
    # hidden states: each token at a scale of its own, one channel in 64 eight times as wide
    wide = torch.where(torch.rand(D, device=DEV, generator=g) < 1 / 64, 8.0, 1.0)
    level = torch.exp(0.5 * normal(rows, 1))
    s = dict(y=(normal(rows, D) * wide * level).to(T), h=(2 * normal(rows, D) * wide).to(R), post=weight(case["post"]),
             pre=weight(case["pre"]))
    s["gate"] = {"none": lambda: None, "channel": lambda: (0.5 + 0.2 * normal(D)).to(W),
                 "row": lambda: torch.sigmoid(normal(rows, 1)).to(T), "full": lambda: torch.sigmoid(normal(rows, D)).to(T)}[case["gate"]]()
    if case["kind"] == "norm_backward":
        # gradients of a loss scaled by 2^10, so that the 16-bit ones stay in their range
        s["dh"] = normal(rows, D).to(R)
        s["dx"] = normal(rows, D).to(T) if case["pre"] else None
    return s


def _clip_inputs(case, g):
    dt, h = DTYPES[case["dtype"]], case["hidden"]
    grads = []
    for layer in range(case["layers"]):
        level = 1e-3 * 2.0 ** (layer % 5)
        for n, t in ((h, torch.float32), (case["inter"], dt), (h, torch.float32), (h, torch.float32), (case["experts"] * h, dt),
                     (case["experts"], torch.float32)):
            grads.append((torch.randn(n, device=DEV, generator=g) * level).to(t))
    if case["vocab"]:
        grads.append((torch.randn(case["vocab"], h, device=DEV, generator=g) * 1e-3).to(dt))
    flat = {t: torch.zeros(size, dtype=t, device=DEV) for t, size in _places(grads)[1].items()}
    return dict(grads=grads, flat=flat, out=_views(grads, flat), max_norm=0.1)


def _places(grads):
    """Where each gradient begins in the buffer of its type, in whole 128-byte lines, and the buffers' lengths."""
    at, end = [], {}
    for t in grads:
        at.append(end.get(t.dtype, 0))
        line = 128 // t.element_size()
        end[t.dtype] = at[-1] + -(-t.numel() // line) * line
    return at, end


def _views(grads, flat):
    """What an optimizer reads: the gradients as views of one buffer a type."""
    return [flat[t.dtype][a:a + t.numel()].view(t.shape) for t, a in zip(grads, _places(grads)[0])]


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"].startswith("route"):
        return _route_inputs(case, g)
    return _clip_inputs(case, g) if case["kind"] == "clip" else _norm_inputs(case, g)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    return s


EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------
# A pass


def _run_own(s):
    from sushi_amd import exl3

    c = s["case"]
    if c["kind"] == "route":
        return exl3.moe_route(s["logits"], c["topk"], bias=s["bias"], score=c["score"], groups=c["groups"],
                              topk_groups=c["taken"], group_top=c["group_top"], renormalize=c["renormalize"],
                              scale=c["scale"], mask=s["mask"])
    if c["kind"] == "route_backward":
        return exl3.moe_route_backward(s["logits"], s["inds"], s["dscores"], score=c["score"], renormalize=c["renormalize"],
                                       scale=c["scale"], mask=s["mask"])
    if c["kind"] == "clip":
        r = exl3.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
        return [r.norm, *s["flat"].values()]
    kw = dict(post_weight=s["post"], pre_weight=s["pre"], gate=s["gate"], eps=EPS, weight_offset=c["offset"],
              residual_scale=c["residual_scale"], block_scale=c["block_scale"])
    if c["kind"] == "norm":
        r = exl3.block_norm(s["y"], s["h"], **kw)
        return [t for t in (r.h, r.x) if t is not None]
    r = exl3.block_norm_backward(s["dh"], s["dx"], s["y"], s["h"], **kw)
    return [t for t in (r.dy, r.dresidual, r.dpost_weight, r.dpre_weight, r.dgate) if t is not None]


def _first_best(v, n):
    """The places of the n largest values of each row, largest first, equal ones by their place; -1 where only -inf is left."""
    place = torch.arange(v.shape[-1], device=v.device)
    v, out = v.clone(), []
    for _ in range(n):
        best = v.amax(-1, keepdim=True)
        at = torch.where(v == best, place, v.shape[-1]).amin(-1, keepdim=True)
        out.append(torch.where(best == -math.inf, -1, at))
        v.scatter_(-1, at, -math.inf)
    return torch.cat(out, -1)


def _plain_route(s):
    c = s["case"]
    rows, E, G, k = c["rows"], c["experts"], c["groups"], c["topk"]
    x = s["logits"].double()  # two experts' values may lie close
    top = x.amax(-1, keepdim=True)
    if c["score"] == "softmax":
        e = torch.exp(x - top)
        p = e / e.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    v = x if s["bias"] is None and c["group_top"] == 1 else p if s["bias"] is None else p + s["bias"].double()
    if G > 1:
        per = v.reshape(rows, G, E // G)
        best = _first_best(per.reshape(rows * G, E // G), c["group_top"]).reshape(rows, G, -1)
        worth = torch.gather(per, 2, best).sum(-1)
        taken = _first_best(worth, c["taken"])
        open_ = (taken[..., None] == torch.arange(G, device=DEV)).any(1)
        v = torch.where(open_[..., None], per, -math.inf).reshape(rows, E)
    inds = _first_best(v, k)
    w = torch.gather(p, 1, inds)
    if c["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    w = (w * c["scale"]).float()
    if s["mask"] is not None:
        inds = torch.where(s["mask"][:, None], inds, -1)
        w = torch.where(s["mask"][:, None], w, 0.0)
    return inds.int(), w


def _plain_route_gradient(s):
    c = s["case"]
    x, kept = s["logits"].float(), s["inds"] >= 0
    at = s["inds"].clamp(min=0).long()
    ds = torch.where(kept, s["dscores"] * c["scale"], 0.0)
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    w = torch.where(kept, torch.gather(p, 1, at), 0.0)
    if c["renormalize"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-38)
        t = w * (ds - (w * ds).sum(-1, keepdim=True))
    else:
        t = w * ds
    if c["score"] == "sigmoid":
        t = t * torch.where(kept, 1 / (1 + torch.exp(torch.gather(x, 1, at))), 0.0)
    d = ((at[..., None] == torch.arange(x.shape[1], device=DEV)) * t[..., None]).sum(1)
    if c["score"] == "softmax" and not c["renormalize"]:
        d = d - p * t.sum(-1, keepdim=True)
    if s["mask"] is not None:
        d = torch.where(s["mask"][:, None], d, 0.0)
    return d.to(s["logits"].dtype)


def _plain_norm(s):
    c = s["case"]
    n = s["y"].float()
    if s["post"] is not None:
        n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + EPS) * (c["offset"] + s["post"].float())
    if s["gate"] is not None:
        n = n * s["gate"].float()
    h = c["residual_scale"] * s["h"].float() + c["block_scale"] * n
    out = [h.to(s["h"].dtype)]
    if s["pre"] is not None:
        x = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * (c["offset"] + s["pre"].float())
        out.append(x.to(s["y"].dtype))
    return out


def _plain_norm_gradient(s):
    c = s["case"]
    y, d = s["y"].float(), s["dh"].float()
    dpre = dpost = dgate = None
    if s["pre"] is not None:
        h, dx = s["h"].float(), s["dx"].float()
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        dpre = (dx * (h * r)).sum(0)
        u = dx * (c["offset"] + s["pre"].float())
        d = d + r * (u - h * r * (u * (h * r)).mean(-1, keepdim=True))
    dres = (c["residual_scale"] * d).to(s["h"].dtype)
    d = c["block_scale"] * d
    n = y
    if s["post"] is not None:
        q = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
        n = y * q * (c["offset"] + s["post"].float())
    if s["gate"] is not None:
        dgate = d * n
        dgate = {"channel": lambda: dgate.sum(0), "row": lambda: dgate.sum(1, keepdim=True),
                 "full": lambda: dgate.to(s["y"].dtype)}[c["gate"]]()
        d = d * s["gate"].float()
    if s["post"] is not None:
        dpost = (d * (y * q)).sum(0)
        v = d * (c["offset"] + s["post"].float())
        d = q * (v - y * q * (v * (y * q)).mean(-1, keepdim=True))
    return [t for t in (d.to(s["y"].dtype), dres, dpost, dpre, dgate) if t is not None]


def _plain_clip(s):
    norm = torch.sqrt(sum((t.double() ** 2).sum() for t in s["grads"]))
    scale = (s["max_norm"] / norm).clamp(max=1.0).float()
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * scale)
    return [norm.float(), *s["flat"].values()]


def run(s):
    if own:
        return _run_own(s)
    return {"route": _plain_route, "route_backward": _plain_route_gradient, "norm": _plain_norm,
            "norm_backward": _plain_norm_gradient, "clip": _plain_clip}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    if case["kind"] == "clip":
        h, size = case["hidden"], SIZE[case["dtype"]]
        small = case["layers"] * (3 * h + case["experts"])
        big = case["layers"] * (case["inter"] + case["experts"] * h) + case["vocab"] * h
        return {"bytes": 2 * (4 * small + size * big), "flops": 3 * (small + big)}
    rows, size = case["rows"], SIZE[case["dtype"]]
    if case["kind"] == "route":  # the logits in, a number and a score a slot out
        E = case["experts"]
        by = rows * (E * size + 8 * case["topk"] + case["mask"]) + (4 * E if case["bias"] else 0)
        return {"bytes": by, "flops": 4 * rows * E}
    if case["kind"] == "route_backward":  # a renormalised or sigmoid gradient reads the picked logits alone
        E, k = case["experts"], case["topk"]
        read = E if case["score"] == "softmax" and not case["renormalize"] else k
        return {"bytes": rows * ((read + E) * size + 8 * k + case["mask"]), "flops": rows * (4 * read + 6 * k)}
    D, rsize = case["width"], SIZE[case["residual"]]
    gate = {"none": 0, "channel": D * SIZE[case["wdtype"]], "row": rows * size, "full": rows * D * size}[case["gate"]]
    by = gate + (case["post"] + case["pre"]) * D * SIZE[case["wdtype"]]
    if case["kind"] == "norm":
        return {"bytes": by + rows * D * ((1 + case["pre"]) * size + 2 * rsize), "flops": rows * D * 9}
    by += 4 * D * (case["post"] + case["pre"] + (case["gate"] == "channel"))
    by += {"none": 0, "channel": 0, "row": 4 * rows, "full": rows * D * size}[case["gate"]]
    return {"bytes": by + rows * D * ((2 + case["pre"]) * size + (2 + case["pre"]) * rsize), "flops": rows * D * 24}


# ---------------------------------------------------------------------------------------------------------------
# The same results in 64 bits, from the definitions


def _exact_route(case, s):
    x = s["logits"].double()
    R, E = x.shape
    G, k = case["groups"], case["topk"]
    logp = torch.log_softmax(x, -1) if case["score"] == "softmax" else torch.nn.functional.logsigmoid(x)
    p = torch.exp(logp) if case["score"] == "softmax" else torch.sigmoid(x)
    ranked_by_logit = s["bias"] is None and case["group_top"] == 1
    key = x if ranked_by_logit else p + (0 if s["bias"] is None else s["bias"].double())
    if G > 1:
        tops = key.reshape(R, G, -1).sort(dim=-1, descending=True).values[..., :case["group_top"]].sum(-1)
        rank = tops.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
        key = key.masked_fill((rank >= case["taken"]).repeat_interleave(E // G, 1), -math.inf)
    inds = key.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    lw = logp.gather(1, inds)
    w = case["scale"] * torch.exp(lw - torch.logsumexp(lw, -1, keepdim=True) if case["renormalize"] else lw)
    if s["mask"] is not None:
        inds = inds.masked_fill(~s["mask"][:, None], -1)
        w = w * s["mask"][:, None]
    return inds.int(), w


def _exact_route_gradient(case, s):
    x = s["logits"].double()
    d = torch.zeros_like(x)
    k = case["topk"]
    ids, has = s["inds"].long().clamp(min=0), s["inds"] >= 0
    z = x.gather(1, ids)
    if case["score"] == "softmax":
        p, own_slope = torch.exp(z - torch.logsumexp(x, -1, keepdim=True)), torch.ones_like(z)
    else:
        p, own_slope = torch.sigmoid(z), torch.sigmoid(-z)  # d log p / dx
    p = p * has
    total = p.sum(-1, keepdim=True)
    ds = s["dscores"].double() * has * case["scale"]
    if case["renormalize"]:
        r = torch.where(total > 0, p / total, torch.zeros_like(p))
        mean = (r * ds).sum(-1)
        for i in range(k):  # through the weight's logarithm
            d.scatter_add_(1, ids[:, i:i + 1], (r[:, i] * (ds[:, i] - mean) * own_slope[:, i])[:, None])
    else:
        for i in range(k):
            d.scatter_add_(1, ids[:, i:i + 1], (p[:, i] * ds[:, i] * own_slope[:, i])[:, None])
        if case["score"] == "softmax":
            d -= torch.softmax(x, -1) * (p * ds).sum(-1, keepdim=True)
    return d if s["mask"] is None else d * s["mask"][:, None]


def _exact_norm(case, s):
    """Forward in 64 bits; for the gradient autograd goes through the same formulas at the given h'."""
    grad = case["kind"] == "norm_backward"
    leaf = lambda t: None if t is None else t.double().requires_grad_(grad)  # noqa: E731
    y, h, post, pre, gate = (leaf(s[n]) for n in ("y", "h", "post", "pre", "gate"))
    a, b, o = case["residual_scale"], case["block_scale"], case["offset"]

    def rms(v, w):
        return v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt() * (o + w)

    branch = y if post is None else rms(y, post)
    branch = b * (branch if gate is None else branch * gate)
    if not grad:
        new = a * h + branch
        return [new] if pre is None else [new, rms(new, pre)]
    # h is h' here: the gradient of h' in whole, then of the branch that it came from
    total = s["dh"].double()
    wanted = []
    if pre is not None:
        total_h, dpre = torch.autograd.grad(rms(h, pre), (h, pre), s["dx"].double())
        total = total + total_h
    leaves = [t for t in (y, post, gate) if t is not None]
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(branch, leaves, total)))
    wanted = [got[id(y)], a * total]
    if post is not None:
        wanted.append(got[id(post)])
    if pre is not None:
        wanted.append(dpre)
    if gate is not None:
        wanted.append(got[id(gate)])
    return wanted


def _exact_clip(case, s):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for t in s["grads"]:
        total += torch.linalg.vector_norm(t.double()).square()
    norm = total.sqrt()
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))
    flat = {t: torch.zeros(v.numel(), dtype=torch.float64, device=DEV) for t, v in s["flat"].items()}
    for t, o in zip(s["grads"], _views(s["grads"], flat)):
        o.copy_(t.double() * factor)
    return [norm, *flat.values()]


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "clip":
        return _exact_clip(case, s)
    if kind.startswith("norm"):
        return [t.detach() for t in _exact_norm(case, s)]
    return _exact_route(case, s) if kind == "route" else _exact_route_gradient(case, s)
