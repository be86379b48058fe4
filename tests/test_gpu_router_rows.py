"""The gradient of the router's logits and the balance loss where a workgroup takes more than one set of rows: past 2048
workgroups of the gradient and 512 of the loss, with a ragged end, against f64 (tests/_epilogue.py; bounds as in
tests/test_gpu_router_grad.py)."""
import pytest
import torch

from sushi_amd import exl3
from tests import _epilogue as E
from tests.test_gpu_router_grad import P_ERR, _routing

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# 256 / L rows a workgroup of the gradient (L = 8, 16, 32, 64 lanes a row), 2048 workgroups; the third has several slots a
# lane, the fourth rows that are no whole vectors, the last three passes
CASES = [
    (32768 + 37, 128, 6, BF16, True, True),
    (16384 + 5, 256, 8, F32, False, True),
    (65536 + 3, 16, 12, F16, True, False),
    (32768 + 300, 100, 8, BF16, True, True),
    (8192 + 1, 512, 8, BF16, False, True),
    (2 * 8192 + 3, 300, 32, F32, True, True),
]


def _bound(logits, inds, ds, w, dl, want, dtype):
    bound = torch.zeros_like(want)
    x = logits.double().cpu()
    rows, k = inds.shape
    if w is not None:
        p, wc = E.softmax(x), w.double().cpu()
        bound += float(dl) * 4 * P_ERR * p * (wc + (p * wc).sum(-1, keepdim=True))
    if ds is not None:
        mag = (ds.double().cpu().abs().amax(-1, keepdim=True) * 2).expand(rows, k)
        ids = inds.cpu().long()
        ok = (ids >= 0) & (ids < x.shape[1])
        at = ids.clamp(0, x.shape[1] - 1)
        s = torch.where(ok, E.softmax(torch.where(ok, x.gather(1, at), float("-inf"))), 0.0)
        bound.scatter_add_(1, at, 4 * P_ERR * s * mag)
    half = E.half_step(dtype)
    return bound + (2.0 ** -22 + half) * want.abs() + half * bound + (2.0 ** -25 if dtype == F16 else 2.0 ** -126)


@pytest.mark.parametrize("parts", ["both", "scores", "balance"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_router_gradient_past_one_pass(dev, case, parts):
    rows, experts, k, dtype, masked, dropped = case
    print(f"[router gradient] {case} {parts}", flush=True)
    logits, inds, mask = _routing(dev, experts, *case)
    g = torch.Generator().manual_seed(71)
    again = torch.rand(rows, generator=g) < 0.05  # some rows name an expert twice, in any pass
    inds[:, k - 1] = torch.where(again.to(dev), inds[:, 0], inds[:, k - 1])
    ds = torch.randn(rows, k, generator=g).to(dev) if parts != "balance" else None
    _, _, weight = E.balance(logits, inds, mask, 1.0)
    w = weight.float().to(dev) if parts != "scores" else None
    dl = torch.full((), 3.0 * rows, device=dev) if parts != "scores" else None
    got = exl3.moe_router_backward(logits, inds, dscores=ds, weight=w, dloss=dl, mask=mask)
    torch.cuda.synchronize()
    want = E.router_gradient(logits, inds, ds, w, dl, mask)
    bound = _bound(logits, inds, ds, w, dl, want, dtype)
    off = (got.double().cpu() - want).abs()
    print(f"  worst {(off / bound).max().item():.3f} of its bound", flush=True)
    assert (off <= bound).all()
    assert torch.equal(got, exl3.moe_router_backward(logits, inds, dscores=ds, weight=w, dloss=dl, mask=mask))


# the loss's last rows of one workgroup and the first of several: eight sets of 512 / L rows and nine
SETS = [(512, 64, 4, BF16, True, True), (513, 64, 4, BF16, True, True), (256, 128, 6, F32, False, True),
        (257, 100, 6, F16, True, False), (128, 256, 8, F32, True, True), (129, 256, 8, F32, True, True),
        (64, 512, 8, BF16, False, False), (65, 1000, 8, F32, True, True)]


@pytest.mark.parametrize("case", CASES + SETS, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_balance_loss_past_one_pass(dev, case):
    rows = case[0]
    print(f"[balance] {case}", flush=True)
    logits, inds, mask = _routing(dev, case[1], *case)
    b = exl3.moe_balance_loss(logits, inds, mask=mask, coef=0.02)
    torch.cuda.synchronize()
    loss, counts, weight = E.balance(logits, inds, mask, 0.02)
    assert torch.equal(b.counts.cpu().long(), counts)
    assert ((b.weight.double().cpu() - weight).abs() <= 4 * 2.0 ** -24 * weight).all()
    assert abs(b.loss.item() - loss) <= (P_ERR + (rows / 4 + 1700) * 2.0 ** -24) * loss
