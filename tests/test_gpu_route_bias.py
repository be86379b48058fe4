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
