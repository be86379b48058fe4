"""Linears with an epilogue and the router's balance loss, as measurable cases: a frozen trellis linear with bias,
activation and residual at serving and training widths, its gradients, the balance loss with the experts' counts, and
the gradient of the router's logits.

A case is a dict of plain values.  `listed()` holds the fixed ones, `draw(rng)` one more of the same ranges;
`prepare(case, seed)` makes what a program holds before the call, `run(state)` is one pass, through the library's entry
points where `own` is set and in elementary torch operations where it is not, `work(case)` the bytes and operations the
pass cannot do without, and `exact(case, seed)` the pass's result in 64 bits, written apart from both.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def _fwd(name, rows, fin, fout, n, codebook, dtype, bias, act, residual, pre):
    return dict(name=name, kind="forward", rows=rows, fin=fin, fout=fout, n=n, codebook=codebook, dtype=dtype,
                bias=bias, act=act, residual=residual, pre=pre)


def _bwd(name, rows, fin, fout, n, codebook, dtype, act, dbias):
    return dict(name=name, kind="backward", rows=rows, fin=fin, fout=fout, n=n, codebook=codebook, dtype=dtype,
                act=act, dbias=dbias)


def _router(name, kind, rows, experts, topk, dtype, mask):
    return dict(name=name, kind=kind, rows=rows, experts=experts, topk=topk, dtype=dtype, mask=mask)


def listed():
    return [
        # one token through an attention output projection, its bias and the residual stream: latency and launches
        _fwd("epilogue_1row_4096x4096_k4", 1, 4096, 4096, 64, "3inst", "f16", True, "none", True, False),
        # a 7-row speculative verify step through a down projection onto the residual stream
        _fwd("epilogue_7rows_14336x4096_k3", 7, 14336, 4096, 48, "mcg", "bf16", False, "none", True, False),
        # a short prompt through a 6-bit up projection with bias and exact gelu
        _fwd("epilogue_200rows_2560x16384_k6", 200, 2560, 16384, 96, "mcg", "bf16", True, "gelu", False, False),
        # a 2048-token training step's up projection, its pre-activations kept for the backward pass
        _fwd("epilogue_2048rows_4096x14336_k3", 2048, 4096, 14336, 48, "3inst", "bf16", True, "gelu_tanh", False, True),
        # the gradient of a few adapted tokens through an output projection
        _bwd("gradient_5rows_4096x4096_k4", 5, 4096, 4096, 64, "3inst", "f16", "none", True),
        # a ragged micro-batch's gradient through a 6-bit up projection and its gelu
        _bwd("gradient_333rows_2560x16384_k6", 333, 2560, 16384, 96, "mcg", "bf16", "gelu", True),
        # a 2048-token step's gradient through the 3-bit up projection and its activation
        _bwd("gradient_2048rows_4096x14336_k3", 2048, 4096, 14336, 48, "3inst", "bf16", "gelu_tanh", True),
        # a decode batch's expert load and balance
        _router("balance_32rows_e256_top8", "balance", 32, 256, 8, "f32", False),
        # a training step's router, a padded batch with dropped slots
        _router("balance_65521rows_e128_top6", "balance", 65521, 128, 6, "bf16", True),
        # the router's gradient for one sequence
        _router("router_gradient_2048rows_e256_top8", "router_gradient", 2048, 256, 8, "f32", False),
        # and for a training step's padded batch
        _router("router_gradient_65521rows_e128_top6", "router_gradient", 65521, 128, 6, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges: linears of 1 .. 2048 rows, 1 to 8 bits and widths of 1280 to 14336, every
    activation, both directions; routers of 1 .. 65536 rows and 8 to 512 experts."""
    kind = rng.choice(["forward", "forward", "backward", "backward", "balance", "router_gradient"])
    if kind in ("balance", "router_gradient"):
        experts = rng.choice([8, 16, 60, 64, 100, 128, 160, 256, 384, 512])
        return dict(kind=kind, rows=min(_log(rng, 1, 65536), 65536 * 128 // experts), experts=experts,
                    topk=rng.choice([1, 2, 4, 6, 8]), dtype=rng.choice(["f32", "bf16", "f16"]),
                    mask=rng.random() < 0.5)
    rows = _log(rng, 1, 2048)
    while True:
        fin, fout = (128 * _log(rng, 10, 112) for _ in range(2))
        if fin * fout <= 4096 * 14336:
            break
    c = dict(kind=kind, rows=rows, fin=fin, fout=fout, n=rng.choice([16, 24, 32, 40, 48, 64, 80, 96, 128]),
             codebook=rng.choice(["mcg", "mcg", "3inst", "mul1"]), dtype=rng.choice(["f16", "bf16", "bf16", "f32"]),
             act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]))
    if kind == "forward":
        return dict(c, bias=rng.random() < 0.6, residual=rng.random() < 0.5, pre=rng.random() < 0.3)
    return dict(c, dbias=rng.random() < 0.6)


# ---------------------------------------------------------------------------------------------------------------
# Inputs


def _scales(g, width):
    """Sign x magnitude, as a pack's suh / svh: +-1 times 0.5 .. 1.5."""
    sign = torch.randint(0, 2, (1, width), device=DEV, generator=g).float() * 2 - 1
    return sign * (0.5 + torch.rand(1, width, device=DEV, generator=g))


def _linear_inputs(case, g):
    rows, fin, fout, n, dt = case["rows"], case["fin"], case["fout"], case["n"], DTYPES[case["dtype"]]
    s = dict(trellis=torch.randint(-32768, 32768, (1, fin // 16, fout // 16, n), dtype=torch.int16, device=DEV,
                                   generator=g),
             suh=_scales(g, fin).half(), svh=(_scales(g, fout) / math.sqrt(fin)).half())
    normal = lambda r, w: torch.randn(r, w, device=DEV, generator=g)  # noqa: E731
    if case["kind"] == "forward":
        # hidden states: N(0, 1) with one channel in 64 eight times as wide (activation outliers)
        wide = torch.rand(fin, device=DEV, generator=g) < 1 / 64
        s["x"] = (normal(rows, fin) * torch.where(wide, 8.0, 1.0)).to(dt)
        s["bias"] = torch.randn(fout, device=DEV, generator=g).to(dt) if case["bias"] else None
        s["residual"] = (2 * normal(rows, fout)).to(dt) if case["residual"] else None
    else:
        # gradients: small, each row (token) at its own scale
        scale = 1e-3 * torch.exp(normal(rows, 1))
        s["dy"] = (normal(rows, fout) * scale).to(dt)
        s["pre"] = normal(rows, fout).to(dt) if case["act"] != "none" else None
    return s


def _router_inputs(case, g):
    rows, E, k = case["rows"], case["experts"], case["topk"]
    logits = torch.randn(rows, E, device=DEV, generator=g) + torch.randn(E, device=DEV, generator=g) * 0.5
    logits = logits.to(DTYPES[case["dtype"]])
    s = dict(logits=logits, inds=torch.topk(logits.float(), k, dim=-1).indices.int(), mask=None)
    if case["mask"]:  # padded rows, and slots that an expert's capacity dropped
        s["mask"] = torch.rand(rows, device=DEV, generator=g) < 0.8
        s["inds"] = torch.where(torch.rand(rows, k, device=DEV, generator=g) < 0.02, -1, s["inds"])
    s["coef"] = 0.01
    if case["kind"] == "router_gradient":
        live = s["mask"] if s["mask"] is not None else torch.ones(rows, dtype=torch.bool, device=DEV)
        hit = (s["inds"][..., None] == torch.arange(E, device=DEV)).any(1) & live[:, None]
        s["weight"] = s["coef"] * E * hit.sum(0).float() / (live.sum() ** 2 * k).clamp(min=1)
        # a loss scale of one per row keeps every type's gradients in its range
        s["dscores"] = torch.randn(rows, k, device=DEV, generator=g) * 1e-2
        s["dloss"] = torch.full((), float(rows), device=DEV)
    return s


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return _linear_inputs(case, g) if case["kind"] in ("forward", "backward") else _router_inputs(case, g)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------------------------------------------------------
# A pass


def _run_own(s):
    from sushi_amd import exl3

    c = s["case"]
    if c["kind"] == "balance":
        b = exl3.moe_balance_loss(s["logits"], s["inds"], mask=s["mask"], coef=s["coef"])
        return dict(loss=b.loss, counts=b.counts, weight=b.weight)
    if c["kind"] == "router_gradient":
        return exl3.moe_router_backward(s["logits"], s["inds"], dscores=s["dscores"], weight=s["weight"],
                                        dloss=s["dloss"], mask=s["mask"])
    p = exl3.Proj(s["trellis"], s["suh"], s["svh"])
    dec = {"mcg": exl3.MCG, "mul1": exl3.MUL1, "3inst": exl3.INST3}[c["codebook"]]
    if c["kind"] == "forward":
        return exl3.linear_epilogue(s["x"], p, dec, bias=s["bias"], act=c["act"], residual=s["residual"],
                                    with_pre=c["pre"])
    dx, dbias = exl3.linear_epilogue_backward(s["dy"], p, dec, act=c["act"], pre=s["pre"], with_dbias=c["dbias"])
    return (dx, dbias) if c["dbias"] else dx


def _plain_weights(trellis, codebook):
    """The inner weight [in, out], f32, of a trellis [1, in/16, out/16, n] (16x16 tiles of 256 codewords, each the 16 bits
    up to stream bit (t + 1) n / 16 of a circular stream of 32-bit words, first bit highest)."""
    _, it, ot, n = trellis.shape
    hw = trellis.reshape(it * ot, n // 2, 2).long() & 0xFFFF
    words = hw[..., 0] | (hw[..., 1] << 16)
    t = torch.arange(256, device=DEV)
    last = ((t + 1) * n) // 16 - 1
    at = last >> 5
    two = (words[:, (at - 1) % (n // 2)] << 32) | words[:, at]
    cw = (two >> (31 - (last & 31))) & 0xFFFF
    f16 = lambda b: torch.where(b >= 32768, b - 65536, b).to(torch.int16).view(torch.float16).float()  # noqa: E731
    if codebook == "mul1":
        p = (cw * 0x83DCD12D) & 0xFFFFFFFF
        total = (p & 255) + ((p >> 8) & 255) + ((p >> 16) & 255) + (p >> 24)
        one = lambda b: f16(torch.full((), b, device=DEV))  # noqa: E731
        w = ((1024 + total).float() * one(0x1EEE) + one(0xC931)).half().float()
    else:
        p = (cw * 89226354 + 64248484 if codebook == "3inst" else cw * 0xCBAC1FED) & 0xFFFFFFFF
        p = (p & 0x8FFF8FFF) ^ 0x3B603B60
        w = (f16(p & 0xFFFF) + f16(p >> 16)).half().float()
    lane, i = t >> 3, t & 7
    row, col = 2 * (lane & 3) + (i & 1) + 8 * ((i >> 1) & 1), (lane >> 2) + 8 * (i >> 2)
    tile = torch.empty(it * ot, 256, device=DEV)
    tile[:, row * 16 + col] = w
    return tile.reshape(it, ot, 16, 16).transpose(1, 2).reshape(it * 16, ot * 16)


def _plain_had(v):
    """The Hadamard transform of every 128 values, over sqrt(128)."""
    i = torch.arange(128, device=DEV)
    odd = (((i[:, None] & i[None, :])[..., None] >> torch.arange(7, device=DEV)) & 1).sum(-1) & 1
    return (v.reshape(*v.shape[:-1], -1, 128) @ ((1 - 2 * odd).float() / math.sqrt(128))).reshape(v.shape)


def _plain_softmax(x):
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return z * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_forward(s):
    c = s["case"]
    # the prepared input is f16 by the format's definition
    u = _plain_had(s["x"].half().float() * s["suh"].float()).half().float()
    z = _plain_had(u @ _plain_weights(s["trellis"], c["codebook"])) * s["svh"].float()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _plain_act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    dt = DTYPES[c["dtype"]]
    return (y.to(dt), z.to(dt)) if c["pre"] else y.to(dt)


def _plain_backward(s):
    c = s["case"]
    dz = s["dy"].float()
    if s["pre"] is not None:
        dz = dz * _plain_slope(s["pre"].float(), c["act"])
    v = dz * s["svh"].float()
    # the prepared gradient is f16 too, under a power of two for each row that brings its largest value to 2^10 .. 2^11
    two = torch.exp2(11.0 - torch.frexp(v.abs().amax(1, keepdim=True)).exponent)
    u = (_plain_had(v) * two).half().float()
    dx = _plain_had(u @ _plain_weights(s["trellis"], c["codebook"]).t()) * s["suh"].float() / two
    dx = dx.to(DTYPES[c["dtype"]])
    return (dx, dz.sum(0)) if c["dbias"] else dx


def _plain_balance(s):
    E, k = s["case"]["experts"], s["case"]["topk"]
    p = _plain_softmax(s["logits"].float())
    hit = (s["inds"][..., None] == torch.arange(E, device=DEV)).sum(1)
    live = torch.full((), p.shape[0], device=DEV)
    if s["mask"] is not None:
        p, hit = p * s["mask"][:, None], hit * s["mask"][:, None]
        live = s["mask"].sum()
    counts = hit.sum(0)
    live = live.float()
    weight = s["coef"] * E * (counts.float() / (live * k).clamp(min=1)) / live.clamp(min=1)
    return dict(loss=(weight * p.sum(0)).sum(), counts=counts.int(), weight=weight)


def _plain_router_gradient(s):
    logits = s["logits"].float()
    p = _plain_softmax(logits)
    w = s["weight"]
    d = s["dloss"] * p * (w - (p * w).sum(-1, keepdim=True))
    # the scores are the softmax of the picked logits; a dropped slot has none
    kept = s["inds"] >= 0
    at = s["inds"].clamp(min=0).long()
    picked = torch.where(kept, torch.gather(logits, 1, at), -math.inf)
    sc = torch.exp(picked - picked.amax(-1, keepdim=True))
    sc = torch.where(kept, sc, 0.0)
    sc = sc / sc.sum(-1, keepdim=True)
    g = sc * (s["dscores"] - (sc * s["dscores"]).sum(-1, keepdim=True))
    d = d + ((at[..., None] == torch.arange(p.shape[1], device=DEV)) * torch.where(kept, g, 0.0)[..., None]).sum(1)
    if s["mask"] is not None:
        d = torch.where(s["mask"][:, None], d, 0.0)
    return d.to(s["logits"].dtype)


def run(s):
    if own:
        return _run_own(s)
    return {"forward": _plain_forward, "backward": _plain_backward, "balance": _plain_balance,
            "router_gradient": _plain_router_gradient}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without


def work(case):
    rows, size = case["rows"], SIZE[case["dtype"]]
    if case["kind"] in ("balance", "router_gradient"):
        E, k = case["experts"], case["topk"]
        by = rows * (E * size + 4 * k + (1 if case["mask"] else 0)) + 8 * E
        if case["kind"] == "balance":  # exp and sum for the softmax, its share into the expert's sum
            return {"bytes": by, "flops": 5 * rows * E}
        return {"bytes": by + rows * (E * size + 4 * k), "flops": 9 * rows * E}
    fin, fout = case["fin"], case["fout"]
    by = fin * fout * case["n"] // 128 + 2 * (fin + fout) + rows * (fin + fout) * size
    if case["kind"] == "forward":
        by += (fout * size if case["bias"] else 0) + rows * fout * size * (case["residual"] + case["pre"])
    else:
        by += (rows * fout * size if case["act"] != "none" else 0) + (4 * fout if case["dbias"] else 0)
    return {"bytes": by, "flops": 2 * rows * fin * fout}


# ---------------------------------------------------------------------------------------------------------------
# The same results in 64 bits, from the definitions


def _exact_codebook(codebook):
    """All 65536 codewords' values."""
    cw = np.arange(65536, dtype=np.uint64)
    low = lambda v: v & np.uint64(0xFFFFFFFF)  # noqa: E731
    if codebook == "mul1":
        total = low(cw * np.uint64(0x83DCD12D)).astype(np.uint32).view(np.uint8).reshape(-1, 4).astype(np.float64).sum(1)
        a, b = np.array([0x1EEE, 0xC931], np.uint16).view(np.float16).astype(np.float64)
        return ((1024.0 + total) * a + b).astype(np.float16).astype(np.float64)
    p = low(cw * np.uint64(89226354) + np.uint64(64248484)) if codebook == "3inst" else low(cw * np.uint64(0xCBAC1FED))
    p = ((p & np.uint64(0x8FFF8FFF)) ^ np.uint64(0x3B603B60)).astype(np.uint32)
    halves = p.view(np.uint16).reshape(-1, 2).view(np.float16).astype(np.float64)
    return halves.sum(1).astype(np.float16).astype(np.float64)


def _exact_weights(trellis, codebook):
    it, ot, n = (int(v) for v in trellis.shape[1:])
    # the stream as halfwords, first bit highest: each 32-bit word's high half comes first
    stream = trellis.reshape(it, ot, n // 2, 2).flip(-1).reshape(it, ot, n).to(torch.int32) & 0xFFFF
    r = torch.arange(16, device=DEV)[:, None]
    c = torch.arange(16, device=DEV)[None, :]
    t = 8 * (4 * (c % 8) + (r % 8) // 2) + (r % 2) + 2 * (r // 8) + 4 * (c // 8)  # the codeword of (row, column)
    begin = ((t + 1) * n) // 16 - 16
    first, off = torch.div(begin, 16, rounding_mode="floor"), begin % 16
    table = torch.from_numpy(_exact_codebook(codebook)).to(DEV)
    out = torch.empty(it * 16, ot * 16, dtype=torch.float64, device=DEV)
    for at in range(0, it, 32):  # some tile rows at a time
        part = stream[at:at + 32].long()
        span = (part[..., first % n] << 16) | part[..., (first + 1) % n]
        w = table[(span >> (16 - off)) & 0xFFFF]
        out[at * 16:at * 16 + part.shape[0] * 16] = w.permute(0, 2, 1, 3).reshape(-1, ot * 16)
    return out


def _exact_had(v):
    shape = v.shape
    for half in (64, 32, 16, 8, 4, 2, 1):
        v = v.reshape(-1, 128 // (2 * half), 2, half)
        v = torch.stack([v[:, :, 0] + v[:, :, 1], v[:, :, 0] - v[:, :, 1]], 2)
    return v.reshape(shape) / math.sqrt(128)


def _exact_normal_cdf(z):
    return 0.5 * torch.erfc(-z / math.sqrt(2))


def _exact_tanh_gate(z):
    """0.5 (1 + tanh(a (z + b z^3))) is the logistic function of twice the argument."""
    return 1 / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def _exact_linear(case, s):
    w = _exact_weights(s["trellis"], case["codebook"])
    suh, svh, act = s["suh"].double(), s["svh"].double(), case["act"]
    if case["kind"] == "forward":
        z = _exact_had(_exact_had(s["x"].half().double() * suh).half().double() @ w) * svh
        z = z if s["bias"] is None else z + s["bias"].double()
        y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z / (1 + torch.exp(-z)),
             "gelu": lambda: z * _exact_normal_cdf(z), "gelu_tanh": lambda: z * _exact_tanh_gate(z)}[act]()
        y = y if s["residual"] is None else y + s["residual"].double()
        return (y, z) if case["pre"] else y
    dz = s["dy"].double()
    if s["pre"] is not None:
        z = s["pre"].double()
        if act == "relu":
            dz = dz * (z > 0)
        elif act == "silu":
            g = 1 / (1 + torch.exp(-z))
            dz = dz * (g + z * g * (1 - g))
        elif act == "gelu":
            dz = dz * (_exact_normal_cdf(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        else:
            g = _exact_tanh_gate(z)
            dz = dz * (g + z * g * (1 - g) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z))
    v = dz * svh
    biggest = v.abs().amax(1, keepdim=True)
    scale = torch.where(biggest > 0, 2.0 ** (10 - torch.floor(torch.log2(biggest))), torch.ones_like(biggest))
    u = (_exact_had(v) * scale).half().double() / scale
    dx = _exact_had(u @ w.t().contiguous()) * suh
    return (dx, dz.sum(0)) if case["dbias"] else dx


def _exact_router(case, s):
    E, k = case["experts"], case["topk"]
    x = s["logits"].double()
    live = s["mask"] if s["mask"] is not None else torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
    if case["kind"] == "balance":
        ids = s["inds"][live].reshape(-1).long()
        counts = torch.bincount(ids[ids >= 0], minlength=E)
        T = max(int(live.sum()), 1)
        weight = s["coef"] * E * counts.double() / (T * k) / T
        return dict(loss=(p[live] @ weight).sum(), counts=counts.int(), weight=weight)
    w = s["weight"].double()
    d = float(s["dloss"]) * p * (w - p @ w[:, None])
    ds = s["dscores"].double()
    for i in range(k):  # slot by slot: its score's derivative for every other picked logit
        ei, here = s["inds"][:, i].long(), s["inds"][:, i] >= 0
        picked = torch.where(s["inds"] >= 0, x.gather(1, s["inds"].long().clamp(min=0)), -math.inf)
        sc = torch.softmax(picked, -1).nan_to_num(0.0)
        slope = sc[:, i] * (ds[:, i] - (sc * ds).sum(-1))
        d.scatter_add_(1, ei.clamp(min=0)[:, None], torch.where(here, slope, 0.0)[:, None])
    return d * live[:, None]


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_linear(case, s) if case["kind"] in ("forward", "backward") else _exact_router(case, s)
