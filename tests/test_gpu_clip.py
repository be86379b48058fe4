"""The clip by the global norm against f64.  The squares add in 64 bits, so the norm is its f32 rounding (2^-24, and 2^-40 for
the sums); a clipped value has the scale's rounding, the product's and its type's."""
import math

import pytest
import torch

from sushi_amd import exl3
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _grads(dev, sizes, dtypes, seed=1, level=1e-2):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * level).to(dtypes[i % len(dtypes)]).to(dev) for i, n in enumerate(sizes)]


def _exact(grads, max_norm):
    norm = math.sqrt(sum((t.double() ** 2).sum().item() for t in grads))
    return norm, 1.0 if norm <= max_norm else max_norm / norm


def _matches(before, after, r, max_norm):
    torch.cuda.synchronize()
    norm, scale = _exact(before, max_norm)
    assert r.norm.dtype == r.scale.dtype == F32 and r.norm.shape == r.scale.shape == ()
    assert abs(r.norm.item() - norm) <= (2.0 ** -24 + 2.0 ** -40) * norm
    assert abs(r.scale.item() - scale) <= (2.0 ** -23 + 2.0 ** -40) * scale  # two roundings, max_norm's and its own
    for b, a in zip(before, after):
        want = b.double() * scale
        tiny = 2.0 ** -25 if a.dtype == F16 else 2.0 ** -126
        off = (a.double() - want).abs()
        assert (off <= (2.0 ** -22 + E.half_step(a.dtype)) * want.abs() + tiny).all()


SETS = {
    "one value": [1], "small": [5, 1, 7, 0, 64], "whole chunks": [8192, 16384], "around a chunk": [8191, 8193, 24577],
    "odd": [3, 1001, 12345, 0, 7, 65521], "many": [17] * 700, "a launch's tensors and one more": [33] * 129, "empty": [0, 0],
    "large": [3_000_017, 100, 1_000_000],
}


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F16], [F32, BF16, F16]], ids=str)
@pytest.mark.parametrize("name", SETS)
def test_clip_against_f64(dev, name, dtypes):
    print(f"[clip] {name} {dtypes}", flush=True)
    grads = _grads(dev, SETS[name], dtypes)
    norm, _ = _exact(grads, 1.0)
    for max_norm in (norm * 0.3 + 1e-3, norm * 2 + 1e-3, 0.0, math.inf):
        mine = [t.clone() for t in grads]
        _matches(grads, mine, exl3.clip_grad_norm(mine, max_norm), max_norm)
        if max_norm >= norm:
            assert all(torch.equal(a, b) for a, b in zip(grads, mine))
        for shift in range(3):
            out = [torch.full_like(t, 7, dtype=(F32, BF16, F16)[(i + shift) % 3]) for i, t in enumerate(grads)]
            mine = [t.clone() for t in grads]
            _matches(grads, out, exl3.clip_grad_norm(mine, max_norm, out=out), max_norm)
            assert all(torch.equal(a, b) for a, b in zip(grads, mine))


def test_a_tensor_s_neighbours_stay_and_views_of_any_alignment(dev):
    flat = torch.full((9000,), 3.0, device=dev, dtype=BF16)
    want = flat.clone()
    cuts = [(1, 2), (5, 4000), (4003, 8999)]
    r = exl3.clip_grad_norm([flat[a:b] for a, b in cuts], 1.0)
    keep = torch.ones(9000, dtype=torch.bool, device=dev)
    for a, b in cuts:
        keep[a:b] = False
    assert torch.equal(flat[keep], want[keep])
    n = sum(b - a for a, b in cuts)
    assert abs(r.norm.item() - 3 * math.sqrt(n)) <= 2.0 ** -23 * 3 * math.sqrt(n)
    assert torch.allclose(flat[~keep].float(), torch.full((n,), 1 / math.sqrt(n), device=dev), rtol=2.0 ** -8)
    for off in range(1, 8):
        g = _grads(dev, [5003], [F16], seed=off)[0]
        base = torch.zeros(5003 + off + 9, dtype=F16, device=dev)
        base[off:off + 5003] = g
        out = torch.zeros(5003 + 16, dtype=BF16, device=dev)
        r = exl3.clip_grad_norm([base[off:off + 5003]], 0.05, out=[out[16 - off:16 - off + 5003]])
        _matches([g], [out[16 - off:16 - off + 5003]], r, 0.05)
        assert not out[:16 - off].any() and not out[16 - off + 5003:].any()


def test_shapes_and_values_that_overflow(dev):
    big = [torch.full((3, 5), 3e38, device=dev), torch.full((2, 2, 2), 1e-30, device=dev)]
    r = exl3.clip_grad_norm(big, 1.0)
    torch.cuda.synchronize()
    assert math.isinf(r.norm.item())                  # past f32's largest value
    assert torch.allclose(big[0], torch.full((3, 5), 1 / math.sqrt(15), device=dev), rtol=2.0 ** -22)
    small = [torch.full((100,), 1e-30, device=dev)]   # squares below f32's range
    r = exl3.clip_grad_norm(small, 1.0)
    assert abs(r.norm.item() - 1e-29) <= 2.0 ** -22 * 1e-29 and r.scale.item() == 1.0
    half = [torch.full((70000,), 60000.0, device=dev, dtype=F16)]
    r = exl3.clip_grad_norm(half, 1.0)
    assert abs(r.norm.item() - 60000.0 * math.sqrt(70000)) <= 2.0 ** -20 * 60000 * math.sqrt(70000)
    for bad, want in ((math.inf, 0.0), (math.nan, math.nan)):
        g = [torch.ones(10, device=dev), torch.ones(10, device=dev)]
        g[1][3] = bad
        r = exl3.clip_grad_norm(g, 1.0)
        torch.cuda.synchronize()
        assert (math.isnan(r.norm.item()) if math.isnan(bad) else math.isinf(r.norm.item()))
        assert math.isnan(r.scale.item()) if math.isnan(want) else r.scale.item() == 0.0
        assert torch.isnan(g[1][3]) and (g[0] == 0).all().item() == (bad == math.inf)


def test_clips_one_after_another_and_equal_bits(dev):
    """The workspace's counter comes back to zero, launches of other operators between."""
    grads = _grads(dev, [40001, 12, 5000] * 60, [BF16, F32])
    first = None
    for i in range(6):
        mine = [t.clone() for t in grads]
        r = exl3.clip_grad_norm(mine, 0.5)
        got = [r.norm, r.scale, *mine]
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, got))
        first = got
        exl3.moe_balance_loss(torch.randn(5000, 64, device=dev), torch.zeros(5000, 2, dtype=torch.int32, device=dev))
        exl3.clip_grad_norm([mine[0]], 0.1 * (i + 1))
