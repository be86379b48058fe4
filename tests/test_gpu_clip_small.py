"""The clip by scales below f32's normal range: a far norm and a tiny max_norm.  A clipped value has the scale's rounding, the
product's and its type's (as in test_gpu_clip), and half of the type's least step where it comes out denormal."""
import math

import pytest
import torch

from sushi_amd import exl3
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _check(grads, max_norm, in_place, dtype):
    norm = math.sqrt(sum((t.double() ** 2).sum().item() for t in grads))
    scale = max_norm / norm
    got = [t.clone() for t in grads]
    if in_place:
        r = exl3.clip_grad_norm(got, max_norm)
    else:
        out = [torch.full_like(t, 7, dtype=dtype) for t in grads]
        r = exl3.clip_grad_norm(got, max_norm, out=out)
        assert all(torch.equal(a, b) for a, b in zip(grads, got))
        got = out
    torch.cuda.synchronize()
    assert abs(r.scale.item() - scale) <= 2.0 ** -23 * scale + 2.0 ** -149
    for b, a in zip(grads, got):
        want = b.double() * scale
        least = 2.0 ** -133 if a.dtype == BF16 else 2.0 ** -149
        off = (a.double() - want).abs()
        assert (off <= (2.0 ** -22 + E.half_step(a.dtype)) * want.abs() + least).all(), (off.max(), want.abs().max())


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F32, BF16]], ids=str)
@pytest.mark.parametrize("max_norm", [2.0 ** k for k in (-149, -126, -113, -110, -90, -60, -30, -1)])
def test_far_norms_and_tiny_limits(dev, max_norm, dtypes):
    """Products of up to max_norm are values of f32 however small the scale is on the way."""
    for level in (2.0 ** 20, 2.0 ** 64, 2.0 ** 100, 2.0 ** 127):
        g = torch.Generator().manual_seed(7)
        grads = [(torch.randn(n, generator=g).clamp(-1.5, 1.5) * level).to(dtypes[i % len(dtypes)]).to(dev)
                 for i, n in enumerate((1, 30001, 5, 8192))]
        print(f"[clip] {max_norm} {level} {dtypes}", flush=True)
        _check(grads, max_norm, True, None)
        _check(grads, max_norm, False, F32)
        _check(grads, max_norm, False, BF16)


def test_a_scale_next_to_a_power_of_two(dev):
    """2^-130 (1 - 2^-27), whose f32 mantissa is 1: that is not a scale of 1."""
    _check([torch.tensor([2.0 ** 100], device=dev), torch.tensor([2.0 ** 87], device=dev)], 2.0 ** -30, True, None)
