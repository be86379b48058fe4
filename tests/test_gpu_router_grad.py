"""The router's balance loss, the experts' counts and the gradient of its logits against f64 (tests/_epilogue.py), and a
routed block trained for one step around frozen trellis banks.

f32 bounds: a softmax of logits within 16 of each other loses exp's 2^-23 (|t| + 2) relative, its sum one rounding a term, so
p is within 2^-18 of itself for up to 1024 experts summed pairwise over lanes; sums over rows add at most rows 2^-24 of the
sum of magnitudes."""
import math

import pytest
import torch

from sushi_amd import exl3, synth
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
P_ERR = 2.0 ** -18


def _routing(dev, seed, rows, experts, k, dtype, masked, dropped):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, experts, generator=g) * 1.5).to(dtype)
    inds = torch.topk(logits.float(), k, dim=-1).indices.int()
    if dropped:
        drop = torch.rand(rows, k, generator=g)
        inds = torch.where(drop < 0.1, -1, torch.where(drop < 0.15, experts + 5, inds))
    mask = torch.rand(rows, generator=g) < 0.6 if masked else None
    return logits.to(dev), inds.int().to(dev), None if mask is None else mask.to(dev)


CASES = [
    (1, 8, 1, F32, False, False),
    (1, 256, 8, BF16, False, False),
    (3, 5, 2, F16, True, True),
    (7, 16, 16, BF16, False, True),
    (33, 24, 4, F32, True, False),
    (64, 64, 32, F16, False, True),
    (130, 60, 6, BF16, True, True),
    (257, 100, 8, F32, True, True),
    (1000, 128, 6, BF16, True, True),
    (513, 160, 8, F16, False, False),
    (2048, 256, 8, F32, True, True),
    (700, 384, 12, BF16, True, True),
    (300, 512, 8, F32, False, True),
    (129, 1000, 10, F16, True, True),
    (65, 1024, 32, F32, True, False),
    (40000, 32, 2, BF16, True, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_balance_loss_against_f64(dev, case):
    print(f"[balance] {case}", flush=True)
    rows = case[0]
    logits, inds, mask = _routing(dev, sum(case[:3]), *case)
    b = exl3.moe_balance_loss(logits, inds, mask=mask, coef=0.02)
    torch.cuda.synchronize()
    loss, counts, weight = E.balance(logits, inds, mask, 0.02)
    assert b.counts.dtype == torch.int32 and torch.equal(b.counts.cpu().long(), counts)
    assert ((b.weight.double().cpu() - weight).abs() <= 4 * 2.0 ** -24 * weight).all()
    # rows add up in a workgroup's lanes, its row groups and the workgroups: no term passes more than rows / 4 + 600 sums
    assert abs(b.loss.item() - loss) <= (P_ERR + (min(rows, rows / 4 + 600) + 1100) * 2.0 ** -24) * loss


@pytest.mark.parametrize("parts", ["both", "scores", "balance"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_router_gradient_against_f64(dev, case, parts):
    print(f"[router gradient] {case} {parts}", flush=True)
    rows, experts, k, dtype, masked, dropped = case
    logits, inds, mask = _routing(dev, sum(case[:3]) + 1, *case)
    _, counts, weight = E.balance(logits, inds, mask, 1.0)
    g = torch.Generator().manual_seed(9)
    ds = torch.randn(rows, k, generator=g).to(dev) if parts != "balance" else None
    w = weight.float().to(dev) if parts != "scores" else None
    dl = torch.full((), 3.0 * rows, device=dev) if parts != "scores" else None
    got = exl3.moe_router_backward(logits, inds, dscores=ds, weight=w, dloss=dl, mask=mask)
    torch.cuda.synchronize()
    want = E.router_gradient(logits, inds, ds, w, dl, mask)
    assert got.dtype == dtype and got.shape == logits.shape
    bound = torch.zeros_like(want)
    if parts != "scores":
        p = E.softmax(logits.double().cpu())
        wc = w.double().cpu()
        bound += 3.0 * rows * 4 * P_ERR * p * (wc + (p * wc).sum(-1, keepdim=True))
    if parts != "balance":
        # each slot's term s (ds - sum s ds), scattered
        mag = (ds.double().cpu().abs().amax(-1, keepdim=True) * 2).expand(rows, k)
        ids = inds.cpu().long()
        ok = (ids >= 0) & (ids < experts)
        picked = torch.where(ok, logits.double().cpu().gather(1, ids.clamp(0, experts - 1)), -math.inf)
        s = torch.where(ok, E.softmax(picked), 0.0)
        bound.scatter_add_(1, ids.clamp(0, experts - 1), 4 * P_ERR * s * mag)
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -126
    bound = bound + (2.0 ** -22 + E.half_step(dtype)) * want.abs() + E.half_step(dtype) * bound + tiny
    off = (got.double().cpu() - want).abs()
    print(f"  worst {(off / bound).max().item():.3f} of its bound", flush=True)
    assert (off <= bound).all()
    if mask is not None:
        assert not got[~mask].any()


def test_router_gradient_of_repeated_slots(dev):
    """A row that picks one expert several times (the same id in two slots) adds both terms, in the same bits every time."""
    logits = torch.randn(50, 64, device=dev, generator=torch.Generator(dev).manual_seed(1))
    inds = torch.randint(0, 64, (50, 8), device=dev, dtype=torch.int32, generator=torch.Generator(dev).manual_seed(2))
    inds[:, 3] = inds[:, 1]
    inds[:, 6] = inds[:, 1]
    ds = torch.randn(50, 8, device=dev, generator=torch.Generator(dev).manual_seed(3))
    got = exl3.moe_router_backward(logits, inds, dscores=ds)
    want = E.router_gradient(logits, inds, ds)
    assert (got.double().cpu() - want).abs().max() < 64 * P_ERR
    for _ in range(3):
        assert torch.equal(got, exl3.moe_router_backward(logits, inds, dscores=ds))
    b = exl3.moe_balance_loss(logits, inds)
    assert torch.equal(b.counts.cpu().long(), torch.bincount(inds.cpu().reshape(-1).long(), minlength=64))


def test_masks_that_leave_nothing_and_odd_logits(dev):
    logits = torch.randn(40, 32, device=dev, generator=torch.Generator(dev).manual_seed(4))
    inds = torch.topk(logits, 4, dim=-1).indices.int()
    none = torch.zeros(40, dtype=torch.bool, device=dev)
    dl, ds = torch.ones((), device=dev), torch.ones(40, 4, device=dev)
    b = exl3.moe_balance_loss(logits, inds, mask=none)
    assert b.loss.item() == 0 and not b.counts.any() and not b.weight.any()
    assert not exl3.moe_router_backward(logits, inds, dscores=ds, weight=b.weight, dloss=dl, mask=none).any()
    # no rows at all
    e = exl3.moe_balance_loss(logits[:0], inds[:0])
    assert e.loss.item() == 0 and not e.counts.any() and not e.weight.any()
    assert exl3.moe_router_backward(logits[:0], inds[:0], dscores=ds[:0]).shape == (0, 32)
    # NaN and inf in padded rows are never seen; in live rows they reach the loss and their own row's gradient only
    bad = logits.clone()
    bad[5], bad[6, 3], bad[7] = float("nan"), float("inf"), float("-inf")
    mask = torch.ones(40, dtype=torch.bool, device=dev)
    mask[5:8] = False
    x, y = exl3.moe_balance_loss(bad, inds, mask=mask), exl3.moe_balance_loss(logits, inds, mask=mask)
    assert all(torch.equal(u, v) for u, v in zip(x, y))
    w = y.weight
    u = exl3.moe_router_backward(bad, inds, dscores=ds, weight=w, dloss=dl, mask=mask)
    assert torch.equal(u, exl3.moe_router_backward(logits, inds, dscores=ds, weight=w, dloss=dl, mask=mask))
    assert math.isnan(exl3.moe_balance_loss(bad, inds).loss.item())
    u = exl3.moe_router_backward(bad, inds, dscores=ds, weight=w, dloss=dl)
    keep = [r for r in range(40) if r not in (5, 6)]
    assert torch.isfinite(u[keep]).all() and torch.isnan(u[5]).all()
    # experts masked by -inf, or by their type's lowest value, and a row of -inf alone
    for low in (float("-inf"), torch.finfo(F32).min):
        part = logits.clone()
        part[:, 20:] = low
        part[9] = float("-inf")
        loss, counts, weight = E.balance(part, inds, None, 1.0)
        b = exl3.moe_balance_loss(part, inds)
        assert abs(b.loss.item() - loss) <= 64 * P_ERR * loss and torch.equal(b.counts.cpu().long(), counts)
        g = exl3.moe_router_backward(part, inds, weight=b.weight, dloss=dl)
        assert not g[:, 20:].any() and not g[9].any()
        assert (g.double().cpu() - E.router_gradient(part, inds, None, b.weight, 1.0)).abs().max() < P_ERR


def test_router_of_unaligned_logits_and_leading_dims(dev):
    base = torch.randn(2 * 9 * 128 + 1, device=dev, generator=torch.Generator(dev).manual_seed(6)).to(BF16)
    odd = base[1:].view(2, 9, 128)
    assert odd.data_ptr() % 4 == 2
    whole = odd.clone()
    inds = torch.topk(whole.float(), 6, dim=-1).indices.int()
    a, b = exl3.moe_balance_loss(odd, inds), exl3.moe_balance_loss(whole, inds)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    ds = torch.randn(2, 9, 6, device=dev)
    one = torch.ones(1, device=dev)
    u = exl3.moe_router_backward(odd, inds, dscores=ds, weight=a.weight, dloss=one)
    assert u.shape == (2, 9, 128)
    assert torch.equal(u, exl3.moe_router_backward(whole, inds, dscores=ds, weight=a.weight, dloss=one))


def test_scores_gradient_is_the_routing_chain_s_difference(dev):
    """moe_routing_chain's own f32 scores, differenced along each logit of a row, against the gradient."""
    logits = torch.randn(6, 24, device=dev, generator=torch.Generator(dev).manual_seed(7))
    inds, scores = exl3.moe_routing_chain(logits, 4)
    ds = torch.randn(6, 4, device=dev, generator=torch.Generator(dev).manual_seed(8))
    got = exl3.moe_router_backward(logits, inds, dscores=ds).double()
    h = 2.0 ** -7  # the picks keep their order under it (checked), a score's f32 error over 2 h stays below 2^-14
    for e in range(24):
        step = torch.zeros(24, device=dev)
        step[e] = h
        ip, sp = exl3.moe_routing_chain(logits + step, 4)
        im, sm = exl3.moe_routing_chain(logits - step, 4)
        same = (ip == inds).all(1) & (im == inds).all(1)
        diff = ((sp - sm).double() / (2 * h) * ds.double()).sum(-1)
        # third derivatives of a softmax stay below 1: h^2 / 6 of |ds| on top
        assert ((diff - got[:, e]).abs()[same] <= (2.0 ** -14 + h * h) * ds.double().abs().sum(-1)[same]).all()


def test_balance_in_a_graph(dev):
    logits = torch.randn(3000, 64, device=dev, generator=torch.Generator(dev).manual_seed(10))
    inds = torch.topk(logits, 4, dim=-1).indices.int()
    one = torch.ones((), device=dev)

    def step():
        b = exl3.moe_balance_loss(logits, inds)
        return [*b, exl3.moe_router_backward(logits, inds, weight=b.weight, dloss=one)]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    for i in range(4):
        logits.copy_(torch.randn(3000, 64, device=dev, generator=torch.Generator(dev).manual_seed(20 + i)))
        inds.copy_(torch.topk(logits, 4, dim=-1).indices.int())
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want), i


def test_a_routed_block_trains_around_frozen_banks(dev):
    """h = x + gelu(linear(x) + b), routed experts over h, balance loss: one step's gradients of b, of the router's weight and
    of x from the operators together, against the same block in f64 on the dense weights (loss L = <y, r> + 8 balance)."""
    rows, hidden, inter, experts, k = 24, 256, 128, 8, 2
    p = synth.proj(41, "blk", 1, hidden, hidden, 48, norm=True)
    pd = exl3.Proj(p.trellis.to(dev), p.suh.to(dev), p.svh.to(dev))
    bank = synth.bank(42, "blkx", experts, hidden, inter, 48, norm=True)
    bd = exl3.Bank(*[exl3.Proj(q.trellis.to(dev), q.suh.to(dev), q.svh.to(dev)) for q in (bank.gate, bank.up, bank.down)])
    x = synth.normal(43, "x", (rows, hidden), dtype=F32).to(dev)
    b = (synth.normal(43, "b", (hidden,), dtype=F32) * 0.3).to(dev)
    wr = (synth.normal(43, "wr", (experts, hidden), dtype=F32) * 0.1).to(dev)
    r = synth.normal(43, "r", (rows, hidden), dtype=F32).to(dev)
    mask = torch.arange(rows, device=dev) % 5 != 4

    # forward through the library
    h, pre = exl3.linear_epilogue(x, pd, exl3.MCG, bias=b, act="gelu", residual=x, with_pre=True)
    logits = h @ wr.t()
    inds, scores = exl3.moe_routing_chain(logits, k)
    bal = exl3.moe_balance_loss(logits, inds, mask=mask, coef=8.0)
    y = exl3.moe(h, bd, inds, scores, exl3.MCG)
    # backward: a slot's score sees its expert's output against r (each slot's expert by itself)
    ones = torch.ones(rows, 1, device=dev)
    parts = [exl3.moe(h, bd, inds[:, i:i + 1].contiguous(), ones, exl3.MCG) for i in range(k)]
    ds = torch.stack([(q * r).sum(-1) for q in parts], -1).contiguous()
    # y is the parts' sum by their scores: f16 prepared inputs on both sides of a bank, so only sums' order differs
    mixed = sum(scores[:, i:i + 1] * q for i, q in enumerate(parts))
    assert (y - mixed).abs().max() < 1e-4 * y.abs().max()
    ds = torch.where(mask[:, None], ds, 0.0)
    dlogits = exl3.moe_router_backward(logits, inds, dscores=ds, weight=bal.weight, dloss=torch.ones((), device=dev),
                                       mask=mask)
    dwr = dlogits.t() @ h
    dh = dlogits @ wr
    dx, db = exl3.linear_epilogue_backward(dh, pd, exl3.MCG, act="gelu", pre=pre, with_dbias=True)
    dx = dx + dh  # the residual's gradient

    # the same in f64: the block up to the router by autograd over the dense weight, the experts' outputs as constants
    odec = E.DECODES["mcg"][1]
    w, suh, svh = E.weights(p, odec), p.suh[0].double(), p.svh[0].double()
    x64, b64, wr64 = (t.double().cpu().requires_grad_() for t in (x, b, wr))
    h64 = x64 + E.act(E.had(E.had(x64 * suh) @ w) * svh + b64, "gelu")
    l64 = h64 @ wr64.t()
    picked = l64.gather(1, inds.cpu().long())
    s64 = torch.softmax(picked, -1)
    m = mask.cpu()
    balance = 8.0 * experts * (bal.counts.double().cpu() / (int(m.sum()) * k) * torch.softmax(l64, -1)[m].mean(0)).sum()
    (((s64 * ds.double().cpu())[m]).sum() + balance).backward()
    assert abs(bal.loss.item() - balance.item()) < 2e-3 * balance.item()
    for name, got, want in (("dx", dx, x64.grad), ("db", db, b64.grad), ("dwr", dwr, wr64.grad)):
        # two f16 roundings (the prepared input and the prepared gradient, 2^-11 each) and f32 sums, over a chain of
        # bounded slopes: 2^-8 in the norm leaves a factor of four
        off = (got.double().cpu() - want).norm() / want.norm()
        print(f"  {name}: {off:.2e}", flush=True)
        assert off < 2.0 ** -8, name
