"""What stands between two routed layers, in f64 on the host: the choice of experts and its gradient, the norms around a block
and theirs, with the magnitudes that f32 roundings are relative to."""
from __future__ import annotations

import math

import torch


def probabilities(x, score):
    """p [rows, E] f64; a softmax over the finite logits (+inf and NaN are no part of it)."""
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    x = torch.where(x < math.inf, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def route(logits, k, bias=None, score="softmax", groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0, mask=None):
    """(inds, scores, bad): ids with -1 for slots without an expert, scores in f64, rows whose scores are NaN."""
    x = logits.double().cpu()
    rows, E = x.shape
    nan = x.isnan() | ((x == math.inf) if score == "softmax" else False)
    off = nan | (x == -math.inf)
    p = torch.where(nan, 0.0, probabilities(torch.where(nan, -math.inf, x), score))
    b = torch.zeros(E, dtype=torch.float64) if bias is None else bias.double().cpu()
    off = off | ~(b > -math.inf)
    by_logit = bool((b == b[0]).all()) and math.isfinite(b[0])  # the experts' order is their logits'
    c = torch.where(off, -math.inf, x if by_logit else p + b)
    if groups > 1:
        g = torch.where(off, -math.inf, x if by_logit and group_top == 1 else p + b).reshape(rows, groups, -1)
        best = g.sort(dim=-1, descending=True).values[..., :group_top]
        worth = torch.where(best > -math.inf, best, 0.0).sum(-1).where(best[..., 0] > -math.inf, torch.tensor(-math.inf, dtype=torch.float64))
        order = worth.sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        open_ = torch.zeros(rows, groups, dtype=torch.bool).scatter_(1, order, True)
        c = torch.where(open_[..., None], c.reshape(rows, groups, -1), -math.inf).reshape(rows, E)
    val, inds = c.sort(dim=-1, descending=True, stable=True)
    has = val[:, :k] > -math.inf
    inds = inds[:, :k]
    picked = torch.where(has, x.gather(1, inds), -math.inf)
    if score == "softmax" and renormalize:
        s = probabilities(picked, "softmax")
    elif renormalize:  # the ratio of far negative logits' sigmoids
        logs = -torch.log1p(torch.exp(-picked.abs())) + picked.clamp(max=0)
        s = probabilities(torch.where(has, logs, -math.inf), "softmax")
    else:
        s = p.gather(1, inds)
    s = torch.where(has, s * scale, 0.0)
    inds = torch.where(has, inds, -1)
    bad = nan.any(-1)
    if mask is not None:
        m = mask.cpu().bool()
        inds, s, bad = torch.where(m[:, None], inds, -1), torch.where(m[:, None], s, 0.0), bad & m
    return inds.int(), s, bad


def route_gradient(logits, inds, dscores, score="softmax", renormalize=True, scale=1.0, mask=None):
    """(dlogits, magnitude) in f64: the magnitude is the sum of the terms' absolute values."""
    x, ds = logits.double().cpu(), dscores.double().cpu() * scale
    rows, E = x.shape
    ids = inds.cpu().long()
    kept = (ids >= 0) & (ids < E)
    at = ids.clamp(0, E - 1)
    z = x.gather(1, at)
    p = probabilities(x, score)
    w = p.gather(1, at)
    d, mag = torch.zeros_like(x), torch.zeros_like(x)
    if renormalize:
        logs = z if score == "softmax" else -torch.log1p(torch.exp(-z.abs())) + z.clamp(max=0)
        r = torch.where(kept, probabilities(torch.where(kept, logs, -math.inf), "softmax"), 0.0)
        kds = torch.where(kept, ds, 0.0)
        t = r * (kds - (r * kds).sum(-1, keepdim=True))
        m = r * (kds.abs() + (r * kds.abs()).sum(-1, keepdim=True))
    else:
        t = torch.where(kept, w * ds, 0.0)
        m = t.abs()
    if score == "sigmoid":
        slope = 1 / (1 + torch.exp(z))
        t, m = torch.where(kept, t * slope, 0.0), torch.where(kept, m * slope, 0.0)
    d.scatter_add_(1, at, t)
    mag.scatter_add_(1, at, m)
    if score == "softmax" and not renormalize:
        d = d - p * t.sum(-1, keepdim=True)
        mag = mag + p * m.sum(-1, keepdim=True)
    if mask is not None:
        live = mask.cpu().bool()[:, None]
        d, mag = torch.where(live, d, 0.0), torch.where(live, mag, 0.0)
    return d, mag


def _f64(t):
    return None if t is None else t.double().cpu()


def norm(y, h=None, post=None, pre=None, gate=None, eps=1e-6, offset=0.0, a=1.0, b=1.0):
    """((h', x'), (their magnitudes)) in f64."""
    y, h, post, pre, gate = map(_f64, (y, h, post, pre, gate))
    n = y
    if post is not None:
        n = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (offset + post)
    n = b * n if gate is None else b * n * gate
    new, mag = n, n.abs()
    if h is not None:
        new, mag = new + a * h, mag + (a * h).abs()
    if pre is None:
        return (new, None), (mag, None)
    r = 1 / torch.sqrt((new * new).mean(-1, keepdim=True) + eps)
    # an error of h' moves its own x' and, by the factor r, every one of the row
    moved = r * r * (mag * new.abs()).mean(-1, keepdim=True)
    x = new * r * (offset + pre)
    return (new, x), (mag, (mag * r * (offset + pre).abs()) + x.abs() * (1 + moved))


def norm_gradient(dh, dx, y, h, post=None, pre=None, gate=None, eps=1e-6, offset=0.0, a=1.0, b=1.0):
    """Values and magnitudes of (dy, dresidual, dpost, dpre, dgate) in f64."""
    dh, dx, y, h, post, pre, gate = map(_f64, (dh, dx, y, h, post, pre, gate))
    H = torch.zeros_like(y) if dh is None else dh
    M = H.abs()
    dpre = dpost = dgate = (None, None)
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    if pre is not None:
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
        u = dx * (offset + pre)
        H = H + r * (u - h * r * r * (u * h).mean(-1, keepdim=True))
        M = M + r * (u.abs() + h.abs() * r * r * (u * h).abs().mean(-1, keepdim=True))
        dpre = (flat(dx * h * r).sum(0), flat(dx * h * r).abs().sum(0))
    res = (a * H, abs(a) * M)
    H, M = b * H, abs(b) * M
    q = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) if post is not None else torch.ones_like(y[..., :1])
    w = offset + post if post is not None else torch.ones(y.shape[-1], dtype=torch.float64)
    n = y * q * w
    g = torch.ones((), dtype=torch.float64) if gate is None else gate
    if gate is not None:
        full, mag = H * n, M * n.abs()
        if gate.shape == (y.shape[-1],):
            dgate = (flat(full).sum(0), flat(mag).sum(0))
        elif gate.shape[-1] == 1 and y.shape[-1] != 1 or gate.shape == (*y.shape[:-1], 1):
            dgate = (full.sum(-1, keepdim=True), mag.sum(-1, keepdim=True))
        else:
            dgate = (full, mag)
    z, Z = H * g, M * g.abs()
    if post is None:
        return (z, Z), res, dpost, dpre, dgate
    dpost = (flat(z * y * q).sum(0), flat(Z * (y * q).abs()).sum(0))
    v, V = z * w, Z * w.abs()
    dy = q * (v - y * q * q * (v * y).mean(-1, keepdim=True))
    DY = q * (V + y.abs() * q * q * (V * y.abs()).mean(-1, keepdim=True))
    return (dy, DY), res, dpost, dpre, dgate
