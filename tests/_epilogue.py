"""The linear with an epilogue, its gradients and the router's balance loss in f64, each with a per-element bound of how far
an f32 evaluation of the same definition may be from it.

The bounds count roundings, worst case throughout:
  * a prepared value is f16 of an f32 FWHT: the f32 value is within d = 8 2^-24 sum|v| / sqrt(128) of the exact one (seven
    stages, each sum at most sum|v|, and the scale), so its f16 lies between those of h - d and h + d;
  * an inner product of K terms accumulates through at most K / 32 + 16 f32 additions a term passes (a matrix instruction
    sums its terms, eight waves or K / 32 instructions follow), each off by at most 2^-23 of the sum of magnitudes;
  * the output transform sums 128 of them over sqrt(128), and adds an FWHT's own roundings;
  * an activation or its slope evaluated in f32 is within 2^-17 of its argument's scale: exp's argument t reaches 25 for the
    inputs here and loses 2^-23 |t| relative, erfc and the products a few ulps; every activation's slope stays below 1.13;
  * the last rounding is half a step, finfo.eps / 2 of the value.
"""
from __future__ import annotations

import math

import numpy as np
import torch

import oracle as O
from sushi_amd import exl3

DECODES = {
    "mcg": (exl3.MCG, O.decode(O.CB_MCG)),
    "mul1": (exl3.MUL1, O.decode(O.CB_MUL1)),
    "3inst": (exl3.INST3, O.decode(O.CB_3INST)),
    "spec1": (exl3.Decode(exl3.Codebook.spec1, exl3.Window(15), 1), O.decode(O.CB_SPEC1, 15, 1)),
    "pair1": (exl3.Decode(exl3.Codebook.pair1), O.decode(O.CB_PAIR1)),
    "mcg_w12": (exl3.Decode(exl3.Codebook.mcg, exl3.Window(12)), O.decode(O.CB_MCG, 12)),
}
ACTS = list(exl3.ACTIVATIONS)
ACT_ERR = 2.0 ** -17
LIPSCHITZ = 1.13


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def had(v: torch.Tensor) -> torch.Tensor:
    h = torch.ones(1, 1, dtype=torch.float64)
    for _ in range(7):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
    return (v.reshape(*v.shape[:-1], -1, 128) @ h).reshape(v.shape) / math.sqrt(128)


def block_sum(v: torch.Tensor) -> torch.Tensor:
    """Every element replaced by the sum of its 128-block."""
    b = v.reshape(*v.shape[:-1], -1, 128)
    return b.sum(-1, keepdim=True).expand(b.shape).reshape(v.shape)


def act(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def slope(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        g = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
        return g + z * g * (1 - g) * 2 * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def weights(p: exl3.Proj, odec) -> torch.Tensor:
    """The inner weight [in, out] of a one-bank projection, f64."""
    w = O.reconstruct_inner(p.trellis.cpu().numpy().view(np.uint16), p.in_features, p.out_features, p.n, odec)
    return torch.from_numpy(w.view(np.float16).astype(np.float64))


def _prepared(v: torch.Tensor, dv: torch.Tensor):
    """(u, bound) of f16(H v) for v known to within dv."""
    h = had(v)
    d = (block_sum(dv) + 8 * 2.0 ** -24 * block_sum(v.abs())) / math.sqrt(128) + 2.0 ** -23 * h.abs()
    u = h.half().double()
    return u, torch.maximum(((h + d).half().double() - u).abs(), ((h - d).half().double() - u).abs())


def _product(u, du, w, scale):
    """(H(u w) * scale, bound)."""
    k = w.shape[0]
    inner = u @ w
    di = du @ w.abs() + (k / 32 + 16) * 2.0 ** -23 * (u.abs() @ w.abs())
    d = (block_sum(di) + 8 * 2.0 ** -24 * block_sum(inner.abs())) / math.sqrt(128)
    y = had(inner) * scale
    return y, d * scale.abs() + 2.0 ** -22 * y.abs()


def _rounded(y, dy, dtype):
    """The bound after rounding to dtype (its subnormals have a fixed step)."""
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
    return dy + half_step(dtype) * (y.abs() + dy) + tiny


def forward(x, p, odec, bias=None, act_name="none", residual=None, out_dtype=None):
    """(y, y's bound, z, z's bound), f64 on the CPU."""
    dt = out_dtype or x.dtype
    v = x.cpu().half().double() * p.suh[0].cpu().double()
    u, du = _prepared(v, 2.0 ** -24 * v.abs())
    z, dz = _product(u, du, weights(p, odec), p.svh[0].cpu().double())
    dz = dz + 63 * 2.0 ** -25  # up to 63 splits' fixed-point terms
    if bias is not None:
        z = z + bias.cpu().double()
        dz = dz + 2.0 ** -24 * z.abs()
    y = act(z, act_name)
    dy = LIPSCHITZ * dz + (ACT_ERR * z.abs() if act_name not in ("none", "relu") else 0.0)
    if residual is not None:
        y = y + residual.cpu().double()
        dy = dy + 2.0 ** -24 * y.abs()
    return y, _rounded(y, dy, dt), z, _rounded(z, dz, dt)


def backward(dy, p, odec, act_name="none", pre=None, dx_dtype=None):
    """(dx, dx's bound, dbias, dbias's bound), f64 on the CPU."""
    g = dy.cpu().double()
    dz, ddz = g, torch.zeros_like(g)
    if act_name != "none":
        dz = g * slope(pre.cpu().double(), act_name)
        ddz = g.abs() * (ACT_ERR if act_name != "relu" else 0.0) + 2.0 ** -24 * dz.abs()
    dbias = dz.sum(0)
    bound = (ddz + dz.shape[0] * 2.0 ** -24 * dz.abs()).sum(0)
    svh = p.svh[0].cpu().double()
    v = dz * svh
    top = (g * svh).abs().amax(1, keepdim=True)
    s = torch.where(top > 0, 2.0 ** (10 - torch.floor(torch.log2(top.clamp(min=1e-300)))), torch.ones_like(top))
    u, du = _prepared(v * s, (ddz * svh.abs() + 2.0 ** -24 * v.abs()) * s)
    du = du + 2.0 ** -24  # a row's scale may be the next power of two: f16's subnormal step there
    dx, ddx = _product(u, du, weights(p, odec).t().contiguous(), p.suh[0].cpu().double())
    dx, ddx = dx / s, ddx / s
    return dx, _rounded(dx, ddx, dx_dtype or dy.dtype), dbias, bound


def balance(logits, inds, mask=None, coef=1.0):
    """(loss, counts, weight) in f64 by the definition, rows of -inf alone without probabilities."""
    x, experts, k = logits.cpu().double(), logits.shape[-1], inds.shape[-1]
    x, ids = x.reshape(-1, experts), inds.cpu().long().reshape(-1, k)
    live = torch.ones(x.shape[0], dtype=torch.bool) if mask is None else mask.cpu().reshape(-1).bool()
    counts = torch.zeros(experts, dtype=torch.int64)
    ok = ids[live]
    ok = ok[(ok >= 0) & (ok < experts)]
    counts.scatter_add_(0, ok, torch.ones_like(ok))
    T = int(live.sum())
    if T == 0:
        return torch.zeros((), dtype=torch.float64), counts, torch.zeros(experts, dtype=torch.float64)
    weight = coef * experts * (counts.double() / (T * k)) / T
    return (softmax(x[live]) * weight).sum(), counts, weight


def softmax(x):
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isneginf(top), torch.zeros_like(top), top))
    s = e.sum(-1, keepdim=True)
    return torch.where(s == 0, torch.zeros_like(e), e / s)


def router_gradient(logits, inds, dscores=None, weight=None, dloss=None, mask=None):
    """dlogits in f64 by the definition."""
    x, experts, k = logits.cpu().double(), logits.shape[-1], inds.shape[-1]
    x, ids = x.reshape(-1, experts), inds.cpu().long().reshape(-1, k)
    d = torch.zeros_like(x)
    if weight is not None:
        p, w = softmax(x), weight.cpu().double()
        d = d + float(dloss) * p * (w - (p * w).sum(-1, keepdim=True))
    if dscores is not None:
        ds = dscores.cpu().double().reshape(-1, k)
        ok = (ids >= 0) & (ids < experts)
        picked = torch.where(ok, x.gather(1, ids.clamp(0, experts - 1)), torch.full((), -math.inf, dtype=torch.float64))
        s = torch.where(ok, softmax(picked), torch.zeros_like(picked))
        t = s * (ds - (s * ds).sum(-1, keepdim=True))
        d.scatter_add_(1, ids.clamp(0, experts - 1), torch.where(ok, t, torch.zeros_like(t)))
    if mask is not None:
        d = torch.where(mask.cpu().reshape(-1, 1).bool(), d, torch.zeros_like(d))
    return d.reshape(logits.shape)
