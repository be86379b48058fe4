"""The scale of the prepared gradient where activations are saturated: u = f16(s H(dz * svh)) with s the power of two that
brings the row's largest |dz * svh| to 2^10 .. 2^11, dz = dy act'(pre), so a row of small slopes keeps f16's eleven bits.

Bounds as tests/_epilogue.py counts them, with the slope's own error relative to its terms: the argument t of its exp comes
from at most three roundings and two constants for gelu (t = z^2 / 2), one of each for silu (t = |z|), six for gelu_tanh
(t = |u|), each 2^-24 of t and so 2^-24 t of the exp; exp2, the reciprocal and the products are a few ulps more."""
import math

import pytest
import torch

from sushi_amd import exl3, synth
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
STEP = 2.0 ** -24


def slope_bound(z, name):
    if name == "gelu":
        q = 0.5 * torch.erfc(z.abs() / math.sqrt(2))
        phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return (2.5 * z * z + 24) * STEP * (q + z.abs() * phi) + torch.where(z > 0, 4 * STEP, 0.0)
    if name in ("silu", "gelu_tanh"):
        c = 2 * math.sqrt(2 / math.pi)
        u, du, k = (z, torch.ones_like(z), 2) if name == "silu" else (c * (z + 0.044715 * z ** 3),
                                                                      c * (1 + 3 * 0.044715 * z * z), 8)
        g = torch.sigmoid(-u.abs())
        return (k * u.abs() + 32) * STEP * (g + (z * du).abs() * g) + torch.where(z > 0, 4 * STEP, 0.0)
    return torch.zeros_like(z)


def backward(dy, p, odec, name, pre):
    """(dx, its bound) in f64, u rounded under the power of two of the row's largest |dz * svh|."""
    g, z = dy.cpu().double(), pre.cpu().double()
    dz = g * E.slope(z, name)
    ddz = g.abs() * slope_bound(z, name) + 2 * STEP * dz.abs()
    svh = p.svh[0].cpu().double()
    v = dz * svh
    top = v.abs().amax(1, keepdim=True)
    s = torch.where(top > 0, 2.0 ** (10 - torch.floor(torch.log2(top.clamp(min=1e-300)))), torch.ones_like(top))
    u, du = E._prepared(v * s, (ddz * svh.abs() + STEP * v.abs()) * s)
    du = du + 2.0 ** -24  # the row's scale may be the next power of two
    dx, ddx = E._product(u, du, E.weights(p, odec).t().contiguous(), p.suh[0].cpu().double())
    return dx / s, ddx / s


@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name,at", [("gelu", -7.0), ("gelu", -9.0), ("gelu_tanh", -6.5), ("silu", -30.0), ("relu", -1.0)])
def test_rows_of_small_slopes_keep_their_bits(dev, name, at, dtype, rows):
    print(f"[gradient scale] {name} {at} {dtype} rows={rows}", flush=True)
    p = synth.proj(51, f"gs{rows}", 1, 256, 640, 48, norm=True)
    p = exl3.Proj(p.trellis.to(dev), p.suh.to(dev), p.svh.to(dev))
    dy = synth.normal(52, "dy", (rows, 640), dtype=F32)
    if name == "relu":  # one dead unit with a gradient 2^28 times the others'
        pre = synth.normal(53, "pre", (rows, 640), dtype=F32).abs() + 0.5
        pre[:, 7], dy[:, 7] = at, 2.0 ** 28
    else:
        pre = at + 0.2 * synth.normal(53, "pre", (rows, 640), dtype=F32)
    dy, pre = dy.to(dtype).to(dev), pre.to(dtype).to(dev)
    dec, odec = E.DECODES["mcg"]
    dx, _ = exl3.linear_epilogue_backward(dy, p, dec, act=name, pre=pre, dx_dtype=F32)
    torch.cuda.synchronize()
    want, bound = backward(dy, p, odec, name, pre)
    bound = bound + STEP * (want.abs() + bound)
    off = (dx.double().cpu() - want).abs()
    print(f"  worst {(off / bound).max().item():.3f} of its bound, {(off / want.abs().amax(1, keepdim=True)).max():.1e} of the row's top")
    assert torch.isfinite(dx).all() and (off <= bound).all()
