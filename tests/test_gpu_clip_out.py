"""The clip into other tensors over several launches, and what an infinite limit or norm makes (bounds as in test_gpu_clip)."""
import math

import pytest
import torch

from sushi_amd import exl3
from tests.test_gpu_clip import BF16, F16, F32, _exact, _grads, _matches

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [129, 159, 160, 161, 320, 321])
@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F32, BF16, F16]], ids=str)
def test_out_of_several_launches(dev, count, dtypes):
    """A launch takes 160 tensors: one tensor in the second, empty ones between, each written type beside each read one."""
    grads = _grads(dev, [(33, 8193, 0, 77)[i % 4] if i < count - 1 else 1001 for i in range(count)], dtypes)
    norm, _ = _exact(grads, 1.0)
    for max_norm in (norm * 0.3, norm * 2):
        for shift in range(3):
            out = [torch.full_like(t, 7, dtype=(F32, BF16, F16)[(i + shift) % 3]) for i, t in enumerate(grads)]
            mine = [t.clone() for t in grads]
            _matches(grads, out, exl3.clip_grad_norm(mine, max_norm, out=out), max_norm)
            assert all(torch.equal(a, b) for a, b in zip(grads, mine))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_an_infinite_limit(dev, bad):
    """norm <= inf: the scale is 1, of an infinite norm too; NaN stays NaN."""
    grads = [torch.ones(10, device=dev), torch.ones(10, device=dev, dtype=F16)]
    grads[1][3] = bad
    out = [torch.full((10,), 7.0, device=dev, dtype=BF16) for _ in grads]
    r = exl3.clip_grad_norm([t.clone() for t in grads], math.inf, out=out)
    alone = exl3.clip_grad_norm(grads, math.inf)
    torch.cuda.synchronize()
    for q in (r, alone):
        assert math.isnan(q.norm.item()) and math.isnan(q.scale.item()) if math.isnan(bad) else math.isinf(q.norm.item()) and q.scale.item() == 1.0
    if math.isnan(bad):
        assert all(t.isnan().all() for t in out)
    else:
        assert all(torch.equal(a, b.to(BF16)) for a, b in zip(out, grads))
    assert (grads[0] == 1).all() and (grads[1][:3] == 1).all()  # the norm alone writes nothing


def test_a_norm_past_f32_s_range(dev):
    """Reported as inf; the scale is of the norm in 64 bits."""
    grads = [torch.full((64,), 3e38, device=dev)]
    r = exl3.clip_grad_norm(grads, 2.0)
    torch.cuda.synchronize()
    want = 2.0 / (8 * grads[0].new_tensor(3e38).double().item())
    assert math.isinf(r.norm.item()) and abs(r.scale.item() - want) <= 2.0 ** -23 * want + 2.0 ** -149
    assert torch.allclose(grads[0], torch.full((64,), 0.25, device=dev), rtol=2.0 ** -21, atol=0)
