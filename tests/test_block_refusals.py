"""What the choice of experts, the norms around a block and the clip refuse, before any launch (no GPU: the pointers are never
dereferenced)."""
import ctypes
import math

import pytest
import torch

import sushi_amd._lib as L
from sushi_amd import exl3

B = 1 << 40
WS = dict(ws=1 << 20, wsb=1 << 36)


def _call(name, args, kw):
    args = dict(args, **kw)
    rc = getattr(L.load(), name)(*args.values(), None)
    return rc, L.last_error()


def _route(**kw):
    return _call("exl3_route", dict(lg=B, dt=2, rows=4, experts=64, k=4, bias=None, score=1, groups=8, taken=2, top=2, renorm=1,
                                    scale=1.0, mask=None, inds=2 * B, scores=3 * B), kw)


def _route_bwd(**kw):
    return _call("exl3_route_backward", dict(lg=B, dt=2, rows=4, experts=64, inds=2 * B, k=4, ds=3 * B, score=0, renorm=1,
                                             scale=1.0, mask=None, d=4 * B), kw)


def _norm(**kw):
    return _call("exl3_block_norm", dict(y=B, dt=1, h=2 * B, hdt=1, rows=4, width=128, post=5 * B, pdt=1, gate=None, gdt=1, kind=0,
                                         pre=6 * B, qdt=1, eps=1e-6, off=0.0, rs=1.0, bs=1.0, ho=3 * B, xo=4 * B), kw)


def _norm_bwd(**kw):
    return _call("exl3_block_norm_backward",
                 dict(dh=7 * B, dx=8 * B, y=B, dt=1, h=2 * B, hdt=1, rows=4, width=128, post=5 * B, pdt=1, gate=None, gdt=1, kind=0,
                      pre=6 * B, qdt=1, eps=1e-6, off=0.0, rs=1.0, bs=1.0, dy=9 * B, dres=10 * B, dpost=11 * B, dpre=12 * B,
                      dgate=None, **WS), kw)


@pytest.mark.parametrize("status,kw", [
    (-1, dict(rows=-1)), (-1, dict(experts=0)), (-1, dict(experts=1025, groups=1, taken=1)), (-1, dict(k=0)), (-1, dict(k=33)),
    (-1, dict(k=17)),                      # two groups of eight hold sixteen
    (-1, dict(groups=7)), (-1, dict(groups=0)), (-1, dict(groups=128, experts=1024)), (-1, dict(taken=0)), (-1, dict(taken=9)),
    (-1, dict(top=0)), (-1, dict(top=3)), (-1, dict(groups=64, taken=64, top=2)),
    (-2, dict(dt=3)), (-17, dict(score=2)),
    (-1, dict(lg=None)), (-1, dict(inds=None)), (-1, dict(scores=None)), (-1, dict(lg=B + 2)), (-1, dict(bias=7 * B + 2)),
    (-1, dict(inds=2 * B + 2)), (-1, dict(scores=3 * B + 1)),
    (-1, dict(inds=B)), (-1, dict(scores=B + 4 * 64 * 4 - 4)), (-1, dict(scores=2 * B + 60)), (-1, dict(bias=3 * B)), (-1, dict(mask=2 * B + 3)),
], ids=str)
def test_route_refuses(status, kw):
    rc, text = _route(**kw)
    assert rc == status and text


@pytest.mark.parametrize("status,kw", [
    (-1, dict(k=65)), (-1, dict(experts=2)), (-2, dict(dt=-1)), (-17, dict(score=-1)), (-1, dict(ds=None)), (-1, dict(inds=None)),
    (-1, dict(d=None)), (-1, dict(d=B)), (-1, dict(d=3 * B + 16)), (-1, dict(d=2 * B - 512)), (-1, dict(d=4 * B + 2)),
    (-1, dict(mask=4 * B + 1000)),
], ids=str)
def test_route_gradient_refuses(status, kw):
    rc, text = _route_bwd(**kw)
    assert rc == status and text


N = 4 * 128 * 2  # bytes of y

NORM_CASES = [
    (-1, dict(rows=-1)), (-1, dict(width=0)), (-1, dict(width=16385)), (-2, dict(dt=3)), (-2, dict(hdt=0)), (-2, dict(dt=2)),
    (-2, dict(pdt=5)), (-2, dict(qdt=3)), (-2, dict(gate=13 * B, kind=1, gdt=4)), (-2, dict(gate=13 * B, kind=3, gdt=2)),
    (-1, dict(gate=13 * B)), (-1, dict(kind=1)), (-1, dict(gate=13 * B, kind=4)), (-1, dict(kind=-1)),
    (-1, dict(eps=0.0)), (-1, dict(eps=-1e-6)), (-1, dict(eps=math.nan)), (-1, dict(eps=1e-40)), (-1, dict(eps=math.inf)), (-1, dict(y=None)), (-1, dict(y=B + 1)), (-1, dict(h=2 * B + 1)),
    (-1, dict(post=5 * B + 1)), (-1, dict(gate=13 * B + 2, kind=2, gdt=2)),
]


@pytest.mark.parametrize("status,kw", NORM_CASES + [
    (-1, dict(ho=None)), (-1, dict(xo=None)), (-1, dict(pre=None)), (-1, dict(ho=B)), (-1, dict(xo=2 * B)), (-1, dict(ho=2 * B + 2)),
    (-1, dict(xo=B + N - 2)), (-1, dict(xo=3 * B + 2)), (-1, dict(ho=5 * B)), (-1, dict(xo=6 * B + 254)),
    (-1, dict(gate=4 * B, kind=2)), (-1, dict(gate=3 * B, kind=1)),
], ids=str)
def test_norm_refuses(status, kw):
    rc, text = _norm(**kw)
    assert rc == status and text


@pytest.mark.parametrize("status,kw", NORM_CASES + [
    (-1, dict(dpost=None)), (-1, dict(dpre=None)), (-1, dict(post=None)), (-1, dict(pre=None)), (-1, dict(dgate=14 * B)),
    (-1, dict(gate=13 * B, kind=1)), (-1, dict(dx=None)), (-1, dict(h=None)), (-1, dict(dy=None)),
    (-1, dict(pre=None, dpre=None, dx=None, h=None, dh=None)),
    (-1, dict(dy=7 * B)), (-1, dict(dy=B + 2)), (-1, dict(dres=B)), (-1, dict(dres=2 * B + 2)), (-1, dict(dy=10 * B)),
    (-1, dict(dpost=12 * B + 4)), (-1, dict(dpre=9 * B)), (-1, dict(dpost=8 * B)), (-1, dict(dpost=5 * B)), (-1, dict(dpost=11 * B + 2)),
    (-1, dict(gate=13 * B, kind=3, dgate=13 * B)), (-9, dict(wsb=100)), (-9, dict(ws=None)), (-9, dict(ws=(1 << 20) + 16)),
], ids=str)
def test_norm_gradient_refuses(status, kw):
    rc, text = _norm_bwd(**kw)
    assert rc == status and text


def _clip(tensors, out=None, max_norm=1.0, result=9 * B, ws=1 << 20, wsb=1 << 36):
    """tensors and out: (address, numel, dtype)."""
    n = len(tensors)
    vps, i64s, i32s = ctypes.c_void_p * max(n, 1), ctypes.c_int64 * max(n, 1), ctypes.c_int32 * max(n, 1)
    rc = L.load().exl3_clip_grad_norm(n, vps(*[t[0] for t in tensors]), i64s(*[t[1] for t in tensors]), i32s(*[t[2] for t in tensors]),
                                      None if out is None else vps(*[t[0] for t in out]),
                                      None if out is None else i32s(*[t[2] for t in out]), max_norm, result, ws, wsb, None)
    return rc, L.last_error()


@pytest.mark.parametrize("status,tensors,kw", [
    (-1, [], {}), (-1, [(B, -1, 2)], {}), (-1, [(B, 1 << 37, 2)], {}), (-2, [(B, 4, 3)], {}), (-1, [(None, 4, 2)], {}), (-1, [(B + 2, 4, 2)], {}),
    (-1, [(B, 4, 2)], dict(max_norm=-1.0)), (-1, [(B, 4, 2)], dict(max_norm=math.nan)), (-1, [(B, 4, 2)], dict(result=None)),
    (-1, [(B, 4, 2), (B, 4, 2)], {}), (-1, [(B, 4, 2), (B + 8, 4, 1)], {}), (-1, [(9 * B - 8, 4, 2)], {}),
    (-1, [(B, 4, 2), (2 * B, 4, 2)], dict(out=[(3 * B, 4, 2), (3 * B + 12, 4, 2)])),
    (-1, [(B, 4, 2), (2 * B, 4, 2)], dict(out=[(3 * B, 4, 2), (B, 4, 2)])), (-1, [(B, 4, 2)], dict(out=[(B + 4, 4, 2)])),
    (-2, [(B, 4, 2)], dict(out=[(B, 4, 1)])), (-2, [(B, 4, 2)], dict(out=[(2 * B, 4, 7)])), (-1, [(B, 4, 2)], dict(out=[(None, 4, 2)])),
    (-9, [(B, 4, 2)], dict(wsb=4096)), (-9, [(B, 4, 2)], dict(ws=None)),
], ids=str)
def test_clip_refuses(status, tensors, kw):
    rc, text = _clip(tensors, **kw)
    assert rc == status and text


def test_what_only_looks_alike_is_taken():
    """Buffers end to end, exact replacements and empty calls: these reach the launch, which fails without a GPU, or need none."""
    assert _route(rows=0, lg=None, inds=None, scores=None)[0] == 0 and _route_bwd(rows=0, lg=None, inds=None, ds=None, d=None)[0] == 0
    assert _norm(rows=0, y=None, h=None, ho=None, xo=None)[0] == 0
    if torch.cuda.is_available():
        pytest.skip("the pointers here are no memory")
    for rc, text in (_route(), _route(scores=B + 1024), _route(groups=1, taken=1, top=1, k=32), _route_bwd(), _norm(), _norm(ho=2 * B, xo=B),
                     _norm(ho=B + N, xo=B - N), _norm(h=None), _norm_bwd(), _norm_bwd(dy=B, dres=2 * B), _norm_bwd(dy=8 * B, dres=7 * B),
                     _norm_bwd(dh=None), _norm_bwd(dres=None), _clip([(B, 4, 2)]), _clip([(B, 4, 2), (B + 16, 4, 0), (None, 0, 1)]),
                     _clip([(B, 4, 2)], out=[(B, 4, 2)]), _clip([(B, 4, 2), (B, 4, 2)], max_norm=math.inf)):
        assert rc == -8, text


def test_host_tensors_shapes_and_types_are_refused():
    lg, f = torch.zeros(3, 8), torch.zeros
    for call in (lambda: exl3.moe_route(lg, 2), lambda: exl3.moe_route_backward(lg, f(3, 2, dtype=torch.int32), f(3, 2)),
                 lambda: exl3.block_norm(lg), lambda: exl3.block_norm_backward(lg, None, lg, None), lambda: exl3.clip_grad_norm([lg], 1.0)):
        with pytest.raises(exl3.BadExl3Shape, match="device tensors"):
            call()
    with pytest.raises(exl3.Exl3ActivationUnknown):
        exl3.moe_route(lg, 2, score="tanh")
    for bad in (dict(bias=f(7)), dict(bias=f(8).half()), dict(mask=f(4, dtype=torch.bool))):
        with pytest.raises(exl3.BadExl3Shape):
            exl3.moe_route(lg, 2, **bad)
    with pytest.raises(exl3.BadExl3Dtype):
        exl3.moe_route(lg.double(), 2)
    with pytest.raises(exl3.BadExl3Dtype):
        exl3.moe_route(lg, 2, mask=f(3))
    with pytest.raises(exl3.BadExl3Dtype):
        exl3.moe_route_backward(lg, f(3, 2, dtype=torch.int32), f(3, 2).half())
    for bad in (dict(h=f(3, 7)), dict(post_weight=f(7)), dict(gate=f(3)), dict(gate=f(2, 1))):
        with pytest.raises(exl3.BadExl3Shape):
            exl3.block_norm(lg, **bad)
    for args in ((None, None, lg, None), (lg, lg[:2], lg, lg)):
        with pytest.raises(exl3.BadExl3Shape):
            exl3.block_norm_backward(*args)
    with pytest.raises(exl3.BadExl3Shape):
        exl3.block_norm_backward(lg, None, lg, lg, pre_weight=f(8))
    with pytest.raises(exl3.BadExl3Dtype):
        exl3.block_norm_backward(lg, lg.half(), lg, lg, pre_weight=f(8))
    for args in (([],), ([lg], 1.0, [f(3)])):
        with pytest.raises(exl3.BadExl3Shape):
            exl3.clip_grad_norm(*args, **({} if len(args) > 1 else dict(max_norm=1.0)))
