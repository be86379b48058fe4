"""The choice among f32 logits whose leading bits are alike: equal ones, ones that differ in their last bits, and far ones."""
import math

import pytest
import torch

from tests.test_gpu_route import F32, _check

pytestmark = pytest.mark.gpu


def _rows(kind, rows, experts):
    g = torch.Generator().manual_seed(experts * 31 + rows)
    x = torch.randn(rows, experts, generator=g)
    if kind == "of bf16":
        return x.bfloat16().float()
    if kind == "of few values":
        return torch.randint(-3, 3, (rows, experts), generator=g).float() * 0.5
    if kind == "all equal":
        return torch.full((rows, experts), -1.25)
    if kind == "zeros of either sign":
        return torch.where(x > 0, 0.0, -0.0)
    bits = torch.randint(0, 700, (rows, experts), generator=g)
    if kind == "last bits":  # up to 700 steps of f32 above 1.5, a third of the rows' negative
        v = (torch.tensor(1.5).view(torch.int32) + bits.int()).view(F32)
        return torch.where(torch.arange(rows)[:, None] % 3 == 0, -v, v)
    if kind == "last bits behind a few":
        v = (torch.tensor(-2.5).view(torch.int32) + bits.int()).view(F32)
        return torch.where(torch.rand(rows, experts, generator=g) < 3 / experts, x.abs(), v)
    if kind == "an offset":
        return 1000 + x * 0.02
    assert kind == "denormals"
    return bits.int().view(F32) * torch.where(x > 0, 1.0, -1.0)


KINDS = ["of bf16", "of few values", "all equal", "zeros of either sign", "last bits", "last bits behind a few", "an offset", "denormals"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_f32_logits_alike(dev, kind, score):
    for rows, experts, k in ((1, 8, 8), (3, 7, 4), (67, 64, 1), (130, 60, 8), (300, 256, 8), (33, 250, 5), (2100, 128, 4), (9, 1024, 8)):
        print(f"[order] {kind} {score} {rows} {experts} {k}", flush=True)
        x = _rows(kind, rows, experts).to(dev)
        _check(x, k, score=score)
        _check(x, k, score=score, bias=torch.full((experts,), 0.25, device=dev), renormalize=False)
        mask = torch.arange(rows, device=dev) % 4 != 1
        if experts % 8 == 0 and experts > 8:
            _check(x, k, score=score, groups=8, topk_groups=3 + k // 8 * 2, group_top=1, mask=mask)
            _check(x, k, score=score, bias=torch.full((experts,), -0.5, device=dev), groups=4, topk_groups=2, group_top=2, mask=mask)


@pytest.mark.parametrize("k", [2, 8])
def test_f32_logits_far_apart_and_out(dev, k):
    """Magnitudes over all of f32's range, +inf under sigmoid, and fewer experts left than slots."""
    g = torch.Generator().manual_seed(k)
    x = torch.randn(200, 96, generator=g) * 2.0 ** torch.randint(-40, 100, (200, 96), generator=g).float()
    _check(x.to(dev), k, score="sigmoid", renormalize=False)
    x[::3, 5] = math.inf
    x[::3, 77] = math.inf
    _check(x.to(dev), k, score="sigmoid", renormalize=False)
    y = torch.randn(200, 96, generator=g)
    y[torch.rand(200, 96, generator=g) < torch.linspace(0.5, 1, 200)[:, None]] = -math.inf
    for score in ("softmax", "sigmoid"):
        _check(y.to(dev), k, score=score)
