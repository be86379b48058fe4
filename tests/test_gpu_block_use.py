"""The choice of experts, the norms around a block and the clip as a program uses them: together in a step around frozen banks,
in captured graphs, on streams of their own, on one workspace in any order, and past 32-bit offsets and a launch's rows."""
import math

import pytest
import torch

from sushi_amd import exl3, synth
from tests import _block as R

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(dev, seed):
    return torch.Generator(dev).manual_seed(seed)


def test_a_step_around_a_routed_layer(dev):
    """norm -> router -> routed experts -> norm, its gradients, and the clip: against the same in f64 by autograd, with each slot's
    expert output held as a constant (the routed layer has no gradient here).  L = <h2, r> + <x2, s>."""
    rows, hidden, inter, experts, k = 24, 256, 128, 16, 4
    bank = synth.bank(42, "blk", experts, hidden, inter, 48, norm=True)
    bd = exl3.Bank(*[exl3.Proj(q.trellis.to(dev), q.suh.to(dev), q.svh.to(dev)) for q in (bank.gate, bank.up, bank.down)])
    n = lambda name, *shape, scale=1.0: (synth.normal(43, name, shape, dtype=F32) * scale).to(dev)  # noqa: E731
    y, h, r, s = (n(c, rows, hidden) for c in "yhrs")
    post1, pre1, post2, pre2 = (1 + n(f"w{i}", hidden, scale=0.2) for i in range(4))
    gate = 0.5 + n("g", hidden, scale=0.1)
    wr = n("wr", experts, hidden, scale=0.1)
    bias = n("bias", experts, scale=0.1)
    how = dict(score="sigmoid", renormalize=True, scale=2.5)

    h1, x1 = exl3.block_norm(y, h, post1, pre1, gate)
    logits = x1 @ wr.t()
    inds, scores = exl3.moe_route(logits, k, bias=bias, groups=4, topk_groups=2, group_top=2, **how)
    m = exl3.moe(x1, bd, inds, scores, exl3.MCG)
    h2, x2 = exl3.block_norm(m, h1, post2, pre2, block_scale=0.3)

    ones = torch.ones(rows, 1, device=dev)
    parts = [exl3.moe(x1, bd, inds[:, i:i + 1].contiguous(), ones, exl3.MCG) for i in range(k)]
    mixed = sum(scores[:, i:i + 1] * q for i, q in enumerate(parts))
    assert (m - mixed).abs().max() < 1e-4 * m.abs().max()
    two = exl3.block_norm_backward(r, s, m, h2, post2, pre2, block_scale=0.3)
    ds = torch.stack([(q * two.dy).sum(-1) for q in parts], -1).contiguous()
    dlogits = exl3.moe_route_backward(logits, inds, ds, **how)
    one = exl3.block_norm_backward(two.dresidual, dlogits @ wr, y, h1, post1, pre1, gate)
    grads = [dlogits.t() @ x1, one.dpost_weight, one.dpre_weight, one.dgate, two.dpost_weight, two.dpre_weight]
    raw = [g.clone() for g in grads]
    clip = exl3.clip_grad_norm(grads, 0.25)

    leaf = lambda t: t.double().cpu().requires_grad_()  # noqa: E731
    y6, h6, a6, b6, c6, d6, g6, w6 = (leaf(t) for t in (y, h, post1, pre1, post2, pre2, gate, wr))
    rms = lambda v, w: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    h16 = h6 + g6 * rms(y6, a6)
    x16 = rms(h16, b6)
    l6 = x16 @ w6.t()
    want, _, _ = R.route(l6.detach(), k, bias=bias, groups=4, topk_groups=2, group_top=2, **how)
    assert torch.equal(inds.cpu(), want)
    p = torch.sigmoid(l6.gather(1, inds.cpu().long()))
    sc = 2.5 * p / p.sum(-1, keepdim=True)
    m6 = sum(sc[:, i:i + 1] * q.double().cpu() for i, q in enumerate(parts))
    h26 = h16 + 0.3 * rms(m6, c6)
    ((h26 * r.double().cpu()).sum() + (rms(h26, d6) * s.double().cpu()).sum()).backward()
    near = lambda a, b: (a.double().cpu() - b).norm() <= 2.0 ** -12 * b.norm()  # noqa: E731  f32 sums over a chain of six products
    assert near(h2, h26.detach()) and near(one.dy, y6.grad) and near(one.dresidual, h6.grad)
    exact = [w6.grad, a6.grad, b6.grad, g6.grad, c6.grad, d6.grad]
    for i, (g, w) in enumerate(zip(raw, exact)):
        assert near(g, w), i
    norm = math.sqrt(sum((w ** 2).sum().item() for w in exact))
    assert abs(clip.norm.item() - norm) <= 2.0 ** -12 * norm and norm > 0.25
    for g, b in zip(grads, raw):
        assert torch.allclose(g, b * (0.25 / clip.norm), rtol=2.0 ** -20, atol=1e-30)


def _calls(dev, seed, rows=700):
    g = _gen(dev, seed)
    rand = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    lg, bias, ds = rand(rows, 64).to(BF16), 0.1 * rand(64), rand(rows, 6)
    y, h, dh, dx = (rand(rows, 328).to(BF16) for _ in range(4))
    w1, w2, gate = 1 + 0.1 * rand(328), 1 + 0.1 * rand(328), rand(rows, 1)
    grads = [rand(n) for n in (5, 40001, 128)] + [rand(3001).to(BF16)]
    out = [torch.empty_like(t) for t in grads]
    ins = [lg, bias, ds, y, h, dh, dx, w1, w2, gate, *grads]

    def run():
        inds, scores = exl3.moe_route(lg, 6, bias=bias, score="sigmoid", groups=8, topk_groups=4, group_top=2)
        d = exl3.moe_route_backward(lg, inds, ds, score="sigmoid")
        d2 = exl3.moe_route_backward(lg, inds, ds, renormalize=False)
        new = exl3.block_norm(y, h, w1, w2, gate)
        back = exl3.block_norm_backward(dh, dx, y, new.h, w1, w2, gate)
        clip = exl3.clip_grad_norm(grads, 3.0, out=out)
        return [inds, scores, d, d2, *new, *back, *clip, *out]

    return ins, run


def test_replayed_graphs(dev):
    """Captured on a stream of their own, replayed with other inputs, eager calls of the same between: the eager bits each time."""
    ins, run = _calls(dev, 1)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = run()
    torch.cuda.current_stream(dev).wait_stream(side)
    for i in range(4):
        for a, b in zip(ins, _calls(dev, 10 + i)[0]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_two_streams_at_once(dev):
    pairs = [_calls(dev, 21, 3000), _calls(dev, 22, 2500)]
    want = [[t.clone() for t in run()] for _, run in pairs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in pairs]
    for _ in range(3):
        got = []
        for st, (_, run) in zip(streams, pairs):
            st.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(st):
                got.append([t.clone() for t in run()])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_one_workspace_in_any_order(dev):
    """The linear's folds, the balance loss's counters and these operators' parts share a stream's workspace: each leaves it as the
    next expects it."""
    p = synth.proj(5, "ws", 1, 512, 256, 48, norm=True)
    pd = exl3.Proj(p.trellis.to(dev), p.suh.to(dev), p.svh.to(dev))
    x = torch.randn(3, 512, device=dev, generator=_gen(dev, 3)).to(F16)
    _, run = _calls(dev, 31)
    lg = torch.randn(5000, 64, device=dev, generator=_gen(dev, 4))
    inds = torch.topk(lg, 4, dim=-1).indices.int()
    steps = [lambda: [exl3.linear(x, pd, exl3.MCG)], run, lambda: list(exl3.moe_balance_loss(lg, inds)),
             lambda: list(exl3.clip_grad_norm([lg], math.inf)), lambda: list(exl3.linear_epilogue_backward(x[:, :256].contiguous(), pd, exl3.MCG,
                                                                                                          with_dbias=True))]
    want = [[t.clone() for t in f()] for f in steps]
    g = torch.Generator().manual_seed(6)
    for _ in range(12):
        i = int(torch.randint(0, len(steps), (1,), generator=g))
        assert all(torch.equal(a, b) for a, b in zip(steps[i](), want[i])), i


def test_offsets_past_32_bits(dev):
    """More than 2^31 values of logits, of rows to norm and of one gradient: the last rows hold what they hold by themselves."""
    rows = (1 << 31) // 256 + 9
    lg = torch.zeros(rows, 256, dtype=BF16, device=dev)
    tail = torch.randn(40, 256, device=dev, generator=_gen(dev, 1)).to(BF16)
    lg[-40:] = tail
    for kw in (dict(), dict(bias=torch.linspace(0, 0.1, 256, device=dev), score="sigmoid", groups=8, topk_groups=4, group_top=2)):
        inds, scores = exl3.moe_route(lg, 8, **kw)
        i, s = exl3.moe_route(tail, 8, **kw)
        assert torch.equal(inds[-40:], i) and torch.allclose(scores[-40:], s, rtol=2.0 ** -17, atol=0)
    ds = torch.zeros(rows, 8, device=dev)
    ds[-40:] = 1 + torch.arange(8, device=dev)
    for kw in (dict(score="sigmoid"), dict(renormalize=False)):
        d = exl3.moe_route_backward(lg, inds, ds, **kw)
        assert torch.equal(d[-40:], exl3.moe_route_backward(tail, inds[-40:].contiguous(), ds[-40:].contiguous(), **kw))
        del d
    w = 1 + 0.1 * torch.randn(256, device=dev, generator=_gen(dev, 2))
    h, x = exl3.block_norm(lg, lg, w, w)
    th, tx = exl3.block_norm(tail, tail, w, w)
    assert torch.equal(h[-40:], th) and torch.equal(x[-40:], tx)
    del x
    g = exl3.block_norm_backward(lg, lg, lg, h, w, w)
    tg = exl3.block_norm_backward(tail, tail, tail, th, w, w)
    assert torch.equal(g.dy[-40:], tg.dy) and torch.equal(g.dresidual[-40:], tg.dresidual)
    assert torch.allclose(g.dpre_weight, tg.dpre_weight, rtol=2.0 ** -16, atol=2.0 ** -16)
    del g, h
    r = exl3.clip_grad_norm([lg], 0.5)
    norm = tail.double().norm().item()
    assert abs(r.norm.item() - norm) <= 2.0 ** -22 * norm
    assert torch.equal(lg[-40:], (tail.float() * r.scale).to(BF16)) and not lg[:1000].any()


def test_more_rows_than_a_launch_takes(dev):
    rows = (1 << 24) + 77
    lg = torch.randn(4096, 8, device=dev, generator=_gen(dev, 3)).to(BF16).repeat(rows // 4096 + 1, 1)[:rows]
    mask = torch.ones(rows, dtype=torch.bool, device=dev)
    mask[-3:] = False
    inds, scores = exl3.moe_route(lg, 2, mask=mask)
    ds = torch.ones(rows, 2, device=dev)
    ds[:, 1] = -0.5
    d = exl3.moe_route_backward(lg, inds, ds, score="sigmoid", mask=mask)
    for a, b in ((0, 64), ((1 << 24) - 40, rows)):
        sl = slice(a, b)
        i, s = exl3.moe_route(lg[sl], 2, mask=mask[sl])
        assert torch.equal(inds[sl], i) and torch.equal(scores[sl], s)
        assert torch.equal(d[sl], exl3.moe_route_backward(lg[sl], i, ds[sl], score="sigmoid", mask=mask[sl]))
    gate = torch.randn(4096, 1, device=dev, generator=_gen(dev, 4)).repeat(rows // 4096 + 1, 1)[:rows]
    w = 1 + 0.1 * torch.randn(8, device=dev, generator=_gen(dev, 5))
    for g in (gate, lg):
        h, x = exl3.block_norm(lg, lg, w, w, g)
        for a, b in ((0, 64), ((1 << 21) - 40, (1 << 21) + 40), (rows - 50, rows)):
            sl = slice(a, b)
            th, tx = exl3.block_norm(lg[sl], lg[sl], w, w, g[sl])
            assert torch.equal(h[sl], th) and torch.equal(x[sl], tx)
