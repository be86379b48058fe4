"""The choice of experts under biases that are far apart or take experts out, against f64 (bounds as in test_gpu_route)."""
import math

import pytest
import torch

from tests.test_gpu_route import BF16, F32, _bias, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(64, 1), (256, 1), (256, 8), (512, 16)])
def test_an_expert_out_beside_the_largest_bias(dev, score, experts, groups):
    """-inf and the largest bias among the same 64 experts: the largest still spans the range of every row's values."""
    kw = dict(groups=groups, topk_groups=max(1, groups // 2), group_top=2) if groups > 1 else {}
    for rows in (40, 5000):
        lg = _logits(experts, rows, experts, F32)
        lg[::3, 1] = 9.0
        for largest in (0.4, 5.0, 100.0):
            for at in (1, experts - 1):  # in the first and in the last 64
                bias = _bias(experts, experts)
                bias[at], bias[at - 1] = largest, -math.inf
                for k in (1, 4, 8):
                    print(f"[bias] {score} {rows}x{experts} of {groups} groups, {largest} at {at}, {k} picks", flush=True)
                    _check(lg.to(dev), k, bias=bias.to(dev), score=score, **kw)
                    _check(lg.to(BF16).to(dev), k, bias=bias.to(dev), score=score, renormalize=False, **kw)


@pytest.mark.parametrize("k", [4, 8, 11])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("fill", [-1e4, -1e9, -1e38, torch.finfo(F32).min, "far"], ids=str)
def test_fewer_ordinary_experts_than_slots(dev, fill, score, k):
    """Experts far down by a finite bias are experts: they fill the slots that the ordinary ones leave, in the order of 64-bit values."""
    for experts, groups, taken in ((8 if k <= 8 else 16, 1, 1), (64, 1, 1), (256, 1, 1), (64, 16, -(-k // 4)), (256, 8, 3)):
        for left in (1, k - 1):
            g = torch.Generator().manual_seed(experts + left)
            if fill == "far":  # apart from one another, all below -2^125
                bias = -(0.2 + 0.8 * torch.rand(experts, generator=g)) * torch.finfo(F32).max
            else:
                bias = torch.full((experts,), fill)
            ordinary = torch.randperm(experts, generator=g)[:left]
            bias[ordinary] = _bias(left, left)
            for dtype in (F32, BF16):
                lg = _logits(experts * k, 70, experts, dtype).to(dev)
                for renorm in (True, False):
                    print(f"[bias] {fill} {score} {experts} in {groups}, {left} ordinary, {k} picks", flush=True)
                    for top in ((1, 2) if groups > 1 else (1,)):
                        _check(lg, k, bias=bias.to(dev), score=score, renormalize=renorm, groups=groups, topk_groups=taken, group_top=top)
    # a row of ordinary experts beside far ones that no slot needs, and long calls
    bias = _bias(5, 256)
    bias[::5] = -3e38 if fill == "far" else fill
    for rows in (300, 3000):
        _check(_logits(rows, rows, 256, F32).to(dev), k, bias=bias.to(dev), score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_of_far_biases(dev, score):
    """A group's value is a sum of biases past 2^125: one of 0 and -3.4e38 is below two of -3e37, and one of inf and 0 above two of
    4.3e37."""
    low, high = -torch.finfo(F32).max, 4.3e37
    for rows in (60, 2500):
        for dtype in (F32, BF16):
            lg = _logits(rows, rows, 32, dtype).to(dev)
            bias = torch.full((32,), low)
            bias[0] = 0.0
            bias[8:16] = -3e37
            bias[24:] = -3.2e38
            _check(lg, 4, bias=bias.to(dev), score=score, groups=4, topk_groups=1, group_top=2)
            _check(lg, 8, bias=bias.to(dev), score=score, groups=4, topk_groups=3, group_top=2)
            bias = torch.zeros(32)
            bias[3], bias[8:10], bias[20:22] = math.inf, high, high * 1.5
            _check(lg, 4, bias=bias.to(dev), score=score, groups=4, topk_groups=1, group_top=2)
            _check(lg, 6, bias=bias.to(dev), score=score, groups=4, topk_groups=2, group_top=2, renormalize=False)
