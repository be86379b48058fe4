"""The choice of experts and the gradient of its scores against f64 (tests/_block.py).  The ids are equal, near ties included:
the choice is that of 64-bit values.

f32 bounds of a score: exp of a difference d loses 2^-23 (|d| + 2) relative, |d| below 16 here, a sum one rounding a term, a
quotient one, so a renormalised score is within 2^-18 of itself and so is a softmax over up to 1024 experts (as the router's
other kernels').  Gradients: four such factors a term, and one rounding of the logits' type."""
import math

import pytest
import torch

from sushi_amd import exl3
from tests import _block as R
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
P_ERR = 2.0 ** -18


def _logits(seed, rows, experts, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, experts, generator=g) * 1.5).to(dtype)


def _bias(seed, experts):
    return torch.randint(-150, 151, (experts,), generator=torch.Generator().manual_seed(seed)).float() * 1e-3


def _check(logits, k, got=None, **kw):
    inds, scores = exl3.moe_route(logits, k, **kw) if got is None else got
    torch.cuda.synchronize()
    want, s, bad = R.route(logits.reshape(-1, logits.shape[-1]), k, **{n: v for n, v in kw.items() if n != "mask"},
                           mask=kw["mask"].reshape(-1) if kw.get("mask") is not None else None)
    assert inds.dtype == torch.int32 and scores.dtype == F32 and inds.shape == (*logits.shape[:-1], k)
    inds, scores = inds.cpu().reshape(-1, k), scores.double().cpu().reshape(-1, k)
    wrong = (inds != want).any(-1).nonzero().flatten()
    assert not len(wrong), (len(wrong), wrong[:3], inds[wrong[:3]], want[wrong[:3]])
    assert torch.isnan(scores[bad]).all()
    off = (scores - s).abs()[~bad]
    assert (off <= P_ERR * s.abs()[~bad] + 2.0 ** -126).all(), (off / s.abs()[~bad].clamp(min=1e-30)).max()


# rows, experts, k, dtype, score, bias, groups, taken, group_top, renormalize, scale, mask
CASES = [
    (1, 8, 1, F32, "softmax", False, 1, 1, 1, True, 1.0, False),
    (1, 256, 8, BF16, "sigmoid", True, 8, 4, 2, True, 2.5, False),
    (3, 5, 5, F16, "softmax", False, 1, 1, 1, False, 1.0, True),
    (5, 1, 1, F32, "sigmoid", False, 1, 1, 1, False, 3.0, False),
    (33, 60, 4, BF16, "softmax", False, 1, 1, 1, False, 1.0, False),
    (33, 60, 4, F16, "softmax", True, 4, 2, 1, True, 1.0, True),
    (64, 64, 32, F32, "sigmoid", False, 1, 1, 1, True, 1.0, False),
    (65, 100, 7, F16, "sigmoid", True, 5, 3, 2, False, 16.0, True),
    (130, 64, 6, BF16, "softmax", False, 8, 3, 1, False, 16.0, False),
    (257, 160, 6, F32, "softmax", False, 8, 3, 2, False, 16.0, True),
    (1000, 128, 6, BF16, "softmax", True, 1, 1, 1, False, 1.0, True),
    (513, 160, 8, F16, "sigmoid", True, 1, 1, 1, True, 2.5, False),
    (2047, 256, 8, BF16, "sigmoid", True, 8, 4, 2, True, 2.5, True),
    (2048, 256, 8, F32, "sigmoid", True, 8, 4, 2, True, 2.5, False),
    (700, 384, 12, BF16, "sigmoid", True, 1, 1, 1, True, 1.0, False),
    (300, 512, 8, F32, "softmax", True, 16, 5, 2, True, 1.0, True),
    (129, 1000, 10, F16, "softmax", False, 10, 9, 2, True, 1.0, False),
    (65, 1024, 32, F32, "sigmoid", True, 64, 8, 2, True, 1.0, True),
    (91, 1024, 8, BF16, "softmax", False, 1, 1, 1, True, 1.0, False),
    (77, 24, 3, F32, "sigmoid", True, 12, 2, 2, True, 1.0, False),
    (40, 33, 8, BF16, "sigmoid", False, 11, 4, 1, True, 1.0, False),
    (9001, 32, 2, BF16, "softmax", False, 1, 1, 1, True, 1.0, True),
    (20011, 16, 4, F32, "sigmoid", True, 4, 2, 2, True, 2.5, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_route_against_f64(dev, case):
    print(f"[route] {case}", flush=True)
    rows, experts, k, dtype, score, bias, groups, taken, top, renorm, scale, masked = case
    logits = _logits(rows + experts, rows, experts, dtype).to(dev)
    mask = (torch.rand(rows, generator=torch.Generator().manual_seed(3)) < 0.7).to(dev) if masked else None
    _check(logits, k, bias=_bias(experts, experts).to(dev) if bias else None, score=score, groups=groups, topk_groups=taken, group_top=top,
           renormalize=renorm, scale=scale, mask=mask)


@pytest.mark.parametrize("k", [2, 8, 20])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_values_closer_than_f32_tells(dev, score, k):
    """Logits of a billionth: their sigmoids and softmax values are equal in f32 and apart in f64; and exact ties, whose order is
    the experts'."""
    g = torch.Generator().manual_seed(5)
    lg = torch.stack([torch.randperm(96, generator=g).float() * 2.0 ** -34 for _ in range(50)]).to(dev)
    for kw in (dict(), dict(bias=torch.full((96,), 0.25, device=dev)), dict(groups=6, topk_groups=4, group_top=2)):
        _check(lg, k, score=score, **kw)
    ties = torch.randint(0, 3, (200, 96), generator=g).float().to(dev)
    bias = (torch.randint(0, 2, (96,), generator=g).float() * 0.5).to(dev)
    for dtype in (F32, BF16):
        for kw in (dict(), dict(bias=bias), dict(bias=bias * 0), dict(groups=6, topk_groups=4, group_top=2, bias=bias)):
            _check(ties.to(dtype), k, score=score, **kw)
    assert (exl3.moe_route(torch.zeros(3, 96, device=dev), k)[0].cpu() == torch.arange(k).int()).all()
    zeros = torch.tensor([[0.0, -0.0, 0.0, -0.0] * 24], device=dev)
    assert (exl3.moe_route(zeros, k, score=score)[0].cpu() == torch.arange(k).int()).all()


@pytest.mark.parametrize("k", [3, 8, 11])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("grouped", [False, True])
def test_experts_out_of_the_choice_and_odd_logits(dev, k, score, grouped):
    kw = dict(groups=4, topk_groups=2, group_top=2) if grouped else {}
    lg = _logits(7, 64, 32, F32)
    lg[:, 20:24] = -math.inf
    lg[3, 2:] = -math.inf                       # two experts left
    lg[4] = -math.inf                           # none
    lg[5] = torch.finfo(F32).min                # the type's lowest value is a value
    lg[6, :16] = torch.finfo(F32).min
    lg[7, 5] = math.nan
    lg[8, 5] = math.inf
    lg[9] = math.nan
    lg[10] = lg[10] * 60                        # far apart: sigmoids that vanish or are one
    lg[11] = lg[11] - 150                       # all of them vanish
    lg[12] = lg[12] + 80
    bias = _bias(3, 32)
    out = bias.clone()
    out[8:16], out[17] = -math.inf, math.nan
    far = bias.clone()
    far[4], far[6], far[25] = math.inf, 3e38, -3e38
    none = torch.full((32,), -math.inf)
    for b in (None, bias, out, bias * 1000, far, none):
        for renorm in (True, False):
            for dtype in (F32, BF16):
                _check(lg.to(dtype).to(dev), k, bias=None if b is None else b.to(dev), score=score, renormalize=renorm, **kw)
    # what a padded row holds is not seen
    mask = torch.ones(64, dtype=torch.bool)
    mask[3:13] = False
    _check(lg.to(dev), k, score=score, mask=mask.to(dev), **kw)
    _check(lg.to(dev), k, score=score, mask=torch.zeros(64, dtype=torch.uint8, device=dev), **kw)


def test_a_row_s_choice_does_not_depend_on_its_batch(dev):
    lg = _logits(11, 4099, 128, F32).to(dev)
    bias = _bias(1, 128).to(dev)
    kw = dict(bias=bias, score="sigmoid", groups=8, topk_groups=4, group_top=2)
    inds, scores = exl3.moe_route(lg, 8, **kw)
    for r in (0, 1, 17, 4098):
        i, s = exl3.moe_route(lg[r], 8, **kw)
        assert i.shape == (8,) and torch.equal(i, inds[r]) and torch.allclose(s, scores[r], rtol=2 * P_ERR, atol=0)
    i, s = exl3.moe_route(lg.reshape(1, 4099, 128), 8, **kw)
    assert i.shape == (1, 4099, 8) and torch.equal(i[0], inds) and torch.equal(s[0], scores)
    i, s = exl3.moe_route(lg[:0], 8, **kw)
    assert i.shape == (0, 8) and s.shape == (0, 8)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_route_of_unaligned_logits(dev, dtype):
    base = _logits(13, 1, 41 * 64 + 1, dtype)[0].to(dev)
    odd = base[1:].view(41, 64)
    whole = odd.clone()
    ds = torch.randn(41, 6, device=dev)
    for kw in (dict(), dict(score="sigmoid"), dict(renormalize=False)):
        a, b = exl3.moe_route(odd, 6, **kw), exl3.moe_route(whole, 6, **kw)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        _check(odd, 6, **kw)
        assert torch.equal(exl3.moe_route_backward(odd, a[0], ds, **kw), exl3.moe_route_backward(whole, a[0], ds, **kw))


def test_softmax_renormalised_is_the_routing_chain(dev):
    lg = _logits(17, 500, 256, F32).to(dev)
    inds, scores = exl3.moe_routing_chain(lg, 8)
    got = exl3.moe_route(lg, 8)
    assert torch.equal(got[0], inds) and torch.allclose(got[1], scores, rtol=4 * P_ERR, atol=0)


GRAD_CASES = [
    (1, 8, 1, F32, False, False), (1, 256, 8, BF16, False, False), (3, 5, 2, F16, True, True), (7, 16, 16, BF16, False, True),
    (64, 64, 32, F16, False, True), (130, 60, 6, BF16, True, True), (257, 100, 8, F32, True, True), (1000, 128, 6, BF16, True, True),
    (333, 160, 6, F16, False, False), (2048, 256, 8, F32, True, True), (700, 384, 12, BF16, True, True), (300, 512, 8, F32, False, True),
    (129, 1000, 10, F16, True, True), (65, 1024, 32, F32, True, False), (40000, 32, 2, BF16, True, True),
]
FORMS = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


def _gradient_matches(logits, inds, ds, **kw):
    got = exl3.moe_route_backward(logits, inds, ds, **kw)
    torch.cuda.synchronize()
    want, mag = R.route_gradient(logits, inds, ds, **kw)
    assert got.dtype == logits.dtype and got.shape == logits.shape
    dtype = logits.dtype
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -126
    bound = 4 * P_ERR * mag
    bound = bound + (2.0 ** -22 + E.half_step(dtype)) * want.abs() + E.half_step(dtype) * bound + tiny
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (off / bound).max()
    return got


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("case", GRAD_CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_route_gradient_against_f64(dev, case, form):
    print(f"[route gradient] {case} {form}", flush=True)
    rows, experts, k, dtype, masked, dropped = case
    logits = _logits(rows + experts, rows, experts, dtype)
    inds = torch.topk(logits.float(), k, dim=-1).indices.int()
    g = torch.Generator().manual_seed(9)
    if dropped:
        drop = torch.rand(rows, k, generator=g)
        inds = torch.where(drop < 0.1, -1, torch.where(drop < 0.15, experts + 5, inds)).int()
    mask = (torch.rand(rows, generator=g) < 0.6).to(dev) if masked else None
    ds = torch.randn(rows, k, generator=g)
    got = _gradient_matches(logits.to(dev), inds.to(dev), ds.to(dev), score=form[0], renormalize=form[1], scale=2.5, mask=mask)
    if masked:
        assert not got[~mask].any()


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_gradient_of_repeated_slots_masks_and_odd_logits(dev, form):
    kw = dict(score=form[0], renormalize=form[1])
    lg = _logits(21, 50, 64, F32)
    inds = torch.randint(0, 64, (50, 8), dtype=torch.int32, generator=torch.Generator().manual_seed(2))
    inds[:, 3] = inds[:, 1]
    inds[:, 6] = inds[:, 1]
    ds = torch.randn(50, 8, generator=torch.Generator().manual_seed(3)).to(dev)
    d = [lg.to(dev), inds.to(dev), ds]
    got = _gradient_matches(*d, **kw)
    for _ in range(3):
        assert torch.equal(got, exl3.moe_route_backward(*d, **kw))
    assert not exl3.moe_route_backward(*d, mask=torch.zeros(50, dtype=torch.bool, device=dev), **kw).any()
    assert not exl3.moe_route_backward(d[0], torch.full_like(d[1], -1), ds, **kw).any()
    assert exl3.moe_route_backward(d[0][:0], d[1][:0], ds[:0], **kw).shape == (0, 64)
    # experts out of the choice, rows of nothing else, far logits; a padded row's NaN is not seen
    lg[:, 40:] = -math.inf
    lg[5] = torch.finfo(F32).min
    lg[6] = lg[6] * 60
    lg[7] = lg[7] - 150
    inds = inds % 40
    lg[8], inds[8] = -math.inf, -1
    mask = torch.ones(50, dtype=torch.bool)
    mask[9:11] = False
    live = _gradient_matches(lg.to(dev), inds.to(dev), ds, mask=mask.to(dev), **kw)
    lg[9], lg[10, 3] = math.nan, math.inf
    assert torch.equal(live, exl3.moe_route_backward(lg.to(dev), inds.to(dev), ds, mask=mask.to(dev), **kw))


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_scores_gradient_is_moe_route_s_difference(dev, form):
    """moe_route's own scores, differenced along each logit of a row, against the gradient (first order in h: a score's third
    derivative stays below 1, its f32 error over 2 h below 2^-12 at scale 1)."""
    kw = dict(score=form[0], renormalize=form[1])
    lg = _logits(23, 6, 24, F32).to(dev)
    inds, _ = exl3.moe_route(lg, 4, **kw)
    ds = torch.randn(6, 4, device=dev, generator=torch.Generator(dev).manual_seed(8))
    got = exl3.moe_route_backward(lg, inds, ds, **kw).double()
    h = 2.0 ** -7
    for e in range(24):
        step = torch.zeros(24, device=dev)
        step[e] = h
        (ip, sp), (im, sm) = exl3.moe_route(lg + step, 4, **kw), exl3.moe_route(lg - step, 4, **kw)
        same = (ip == inds).all(1) & (im == inds).all(1)
        diff = ((sp - sm).double() / (2 * h) * ds.double()).sum(-1)
        assert ((diff - got[:, e]).abs()[same] <= (2.0 ** -12 + h * h) * ds.double().abs().sum(-1)[same]).all()
