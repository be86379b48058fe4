"""The activations and their slopes from -12 to 12 at f32 output, relative to their own values: with x = 0 a linear's sums are
zeros, so z is the bias, and with one row and dy = 1 dbias is the slope.

Bounds: the exp's argument t collects at most five half steps for gelu (t = z^2 / 2), two for silu (t = |z|) and eight for
gelu_tanh (t = |u|), each 2^-24 t of the exp; the other operations (the exp2 and reciprocal an ulp each, nine coefficients of
the normal distribution's tail, the products) stay under 24 half steps."""
import math

import pytest
import torch

from sushi_amd import exl3, synth
from tests import _epilogue as E
from tests.test_gpu_gradient_scale import STEP, slope_bound

pytestmark = pytest.mark.gpu

F32 = torch.float32
WIDTH = 16384


def _sweep():
    g = torch.Generator().manual_seed(61)
    z = torch.rand(WIDTH, generator=g) * 24 - 12
    z[:7] = torch.tensor([0.0, -12.0, 12.0, -4.0, -5.0, 1e-6, -1e-6])
    return z


def _proj(dev):
    p = synth.proj(61, "act", 1, 256, WIDTH, 32, norm=True)
    return exl3.Proj(p.trellis.to(dev), p.suh.to(dev), p.svh.to(dev))


@pytest.mark.parametrize("rows", [1, 20, 600])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_activations_keep_their_small_values(dev, name, rows):
    """One row through the GEMV's finish, 20 through the split's, 600 through the 512-row tile's."""
    z = _sweep()
    x = torch.zeros(rows, 256, dtype=F32, device=dev)
    y = exl3.linear_epilogue(x, _proj(dev), exl3.MCG, bias=z.to(dev), act=name).double().cpu()
    assert torch.equal(y, y[:1].expand(rows, WIDTH))
    z = z.double()
    want = E.act(z, name)
    c = 2 * math.sqrt(2 / math.pi)
    t = {"gelu": 2.5 * z * z, "silu": 2 * z.abs(), "gelu_tanh": 8 * c * (z + 0.044715 * z ** 3).abs()}[name]
    bound = (torch.where(z < 0, t, torch.zeros_like(t)) + 24) * STEP * want.abs() + 2.0 ** -122  # (f32 flushes below)
    off = (y[0] - want).abs()
    at = (off / bound).argmax().item()
    print(f"  {name}: worst {(off / bound).max().item():.3f} of its bound at {z[at].item():.3f}", flush=True)
    assert (off <= bound).all()


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_slopes_keep_their_small_values(dev, name):
    z = _sweep()
    dy = torch.ones(1, WIDTH, dtype=F32, device=dev)
    _, got = exl3.linear_epilogue_backward(dy, _proj(dev), exl3.MCG, act=name, pre=z[None].to(dev), with_dbias=True)
    z = z.double()
    want = E.slope(z, name)
    bound = slope_bound(z, name) + 2.0 ** -116  # f32 flushes the gates below 2^-126, times z u' up to 800
    off = (got.double().cpu() - want).abs()
    at = (off / bound).argmax().item()
    print(f"  {name}: worst {(off / bound).max().item():.3f} of its bound at {z[at].item():.3f}", flush=True)
    assert (off <= bound).all()
