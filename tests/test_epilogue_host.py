"""The linear with an epilogue, its gradients and the router's balance loss without a GPU: refusals before any launch, and
the f64 forms the GPU tests compare with, held to differences and to autograd."""
import ctypes
import math

import pytest
import torch

import sushi_amd._lib as L
from sushi_amd import exl3, synth
from tests import _epilogue as E

FAKE = 0x1000  # never dereferenced: every call here is refused first


def _dec():
    return L.DecodeT(1, 16, -1)


def _fwd(**kw):
    a = dict(x=FAKE, xdt=0, rows=1, fin=128, fout=128, tr=FAKE, n=64, suh=FAKE, svh=FAKE, dec=_dec(), bias=None, bdt=0, act=0,
             res=None, y=FAKE, ydt=0, pre=None, ws=None, wsb=0)
    a.update(kw)
    return L.load().exl3_linear_epilogue(*a.values(), None)


def _bwd(**kw):
    a = dict(dy=FAKE, dt=0, rows=1, fin=128, fout=128, tr=FAKE, n=64, suh=FAKE, svh=FAKE, dec=_dec(), act=0, pre=None,
             dx=FAKE, xdt=0, dbias=None, ws=None, wsb=0)
    a.update(kw)
    return L.load().exl3_linear_epilogue_backward(*a.values(), None)


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_refusals_both_ways(call):
    assert call(fin=100) == -1
    assert call(rows=-1) == -1
    assert call(n=130) == -1
    assert call(dec=L.DecodeT(2, 15, -1)) == -3
    assert call(dec=L.DecodeT(4, 15, 3), n=16) == -10
    assert call(act=5) == -17 and call(act=-1) == -17
    assert "activation" in L.last_error()
    assert call(tr=None) == -1
    assert call() == -9  # no workspace
    assert call(ws=FAKE + 8, wsb=1 << 40) == -9  # misaligned
    assert call(rows=0) == 0


def test_forward_refusals():
    assert _fwd(xdt=9) == -2 and _fwd(ydt=3) == -2
    assert _fwd(bias=FAKE, bdt=7) == -2
    assert _fwd(bdt=7) == -9  # without a bias its dtype is not looked at
    for name in ("x", "bias", "res", "y", "pre"):
        assert _fwd(**{name: FAKE + 2}) == -1, name
        assert "4-byte" in L.last_error()


def test_backward_refusals():
    assert _bwd(dt=9) == -2
    assert _bwd(act=3) == -1 and "pre" in L.last_error()
    assert _bwd(dy=FAKE + 4) == -1 and "16-byte" in L.last_error()
    assert _bwd(act=3, pre=FAKE + 4) == -1 and _bwd(dx=FAKE + 1) == -1 and _bwd(svh=FAKE + 8) == -1
    assert _bwd(act=3, pre=FAKE + 8) == -9  # pre needs no more than 8 bytes
    assert _bwd(fin=128 * 65536 // 8) == -1


def test_router_refusals():
    lib = L.load()

    def bal(lg=FAKE, dt=2, rows=1, e=8, inds=FAKE, k=2, loss=FAKE, counts=FAKE, weight=FAKE, ws=None, wsb=0):
        return lib.exl3_balance_loss(lg, dt, rows, e, inds, k, None, 1.0, loss, counts, weight, ws, wsb, None)

    def back(lg=FAKE, dt=2, rows=1, e=8, inds=FAKE, k=2, ds=FAKE, w=None, dl=None, out=FAKE):
        return lib.exl3_router_backward(lg, dt, rows, e, inds, k, ds, w, dl, None, out, None)

    for call in (bal, back):
        assert call(e=1025) == -1 and call(e=0) == -1 and call(k=0) == -1 and call(k=33, e=64) == -1
        assert call(k=9) == -1 and call(rows=-1) == -1 and call(lg=None) == -1 and call(lg=FAKE + 2) == -1
        assert call(dt=3) == -2
        assert call(inds=None) == -1
    assert bal(loss=None) == -1 and bal(counts=None) == -1 and bal(weight=None) == -1
    assert bal() == -9
    assert back(w=FAKE) == -1 and back(dl=FAKE) == -1 and back(out=None) == -1
    assert back(rows=0, lg=None) == 0


def test_workspace_sizes_grow_with_the_rows():
    lib = L.load()
    size = lib.exl3_linear_epilogue_backward_workspace_size
    assert size(0, 128, 128) == 0
    at = [size(r, 4096, 14336) for r in (1, 64, 512, 4096, 16384, 20000, 200000)]
    assert all(v > 8 << 20 for v in at)
    # past a chunk only the rows' largest values and the partial sums grow, not the prepared gradient
    assert at[-1] - at[-2] < 180000 * 28 * 4 + (64 << 20)
    assert lib.exl3_linear_epilogue_workspace_size(100000, 4096, 4096, 64) == \
        lib.exl3_linear_epilogue_workspace_size(16384, 4096, 4096, 64)


def _cpu_proj(in_f=128, out_f=256, n=32):
    return synth.proj(1, "host", 1, in_f, out_f, n, norm=True)


def test_python_refusals():
    p, x = _cpu_proj(), torch.zeros(2, 128, dtype=torch.float16)
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue(x, p, exl3.MCG)  # host tensors
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue(x[:, :64], p, exl3.MCG)
    with pytest.raises(exl3.Exl3ActivationUnknown):
        exl3.linear_epilogue(x, p, exl3.MCG, act="tanh")
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue(x, p, exl3.MCG, bias=torch.zeros(128))
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue(x, p, exl3.MCG, residual=torch.zeros(2, 256))  # f32 beside an f16 output
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue(x, exl3.Proj(p.trellis, p.suh, p.svh[:, :128]), exl3.MCG)
    dy = torch.zeros(2, 256, dtype=torch.float16)
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue_backward(dy, p, exl3.MCG, act="gelu")
    with pytest.raises(exl3.BadExl3Shape):
        exl3.linear_epilogue_backward(dy, p, exl3.MCG, act="gelu", pre=dy.float())
    with pytest.raises(exl3.Exl3ActivationUnknown):
        exl3.linear_epilogue_backward(dy, p, exl3.MCG, act=3)
    lg, inds = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for bad in (dict(inds=inds[:3]), dict(inds=inds.long()), dict(mask=torch.ones(3, dtype=torch.bool)),
                dict(mask=torch.ones(4)), dict()):  # the last: host tensors
        with pytest.raises((exl3.BadExl3Shape, exl3.BadExl3Dtype)):
            exl3.moe_balance_loss(lg, **{"inds": inds, **bad})
    one = torch.zeros(())
    for bad in (dict(weight=torch.zeros(8)), dict(dloss=one), dict(dscores=torch.zeros(4, 3)),
                dict(dscores=torch.zeros(4, 2).half()), dict(weight=torch.zeros(7), dloss=one),
                dict(weight=torch.zeros(8), dloss=torch.zeros(2)), dict(weight=torch.zeros(8).double(), dloss=one)):
        with pytest.raises((exl3.BadExl3Shape, exl3.BadExl3Dtype)):
            exl3.moe_router_backward(lg, inds, **bad)


# ---- the f64 forms


@pytest.mark.parametrize("name", E.ACTS)
def test_activation_slopes_are_the_differences(name):
    z = torch.linspace(-8, 8, 400, dtype=torch.float64) + 1e-3
    h = 1e-6
    diff = (E.act(z + h, name) - E.act(z - h, name)) / (2 * h)
    assert (E.slope(z, name) - diff).abs().max() < 1e-8
    if name != "none":
        torch_fn = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
                    "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[name]
        assert (E.act(z, name) - torch_fn(z)).abs().max() < 1e-12
    assert E.slope(z, name).abs().max() < E.LIPSCHITZ


def test_backward_form_is_autograd_s(monkeypatch):
    """dx without its f16 rounding is autograd's through the same f64 forward."""
    p = _cpu_proj()
    odec = E.DECODES["mcg"][1]
    w, suh, svh = E.weights(p, odec), p.suh[0].double(), p.svh[0].double()
    x = synth.normal(2, "x", (3, 128), dtype=torch.float32).double().requires_grad_()
    b = synth.normal(2, "b", (256,), dtype=torch.float32).double().requires_grad_()
    dy = synth.normal(2, "dy", (3, 256), dtype=torch.float32)
    z = E.had(E.had(x * suh) @ w) * svh + b
    z.retain_grad()
    E.act(z, "gelu").backward(dy.double())
    monkeypatch.setattr(E, "_prepared", lambda v, dv: (E.had(v), dv * 0))
    dx, _, dbias, _ = E.backward(dy, p, odec, "gelu", z.detach())
    assert (dx - x.grad).abs().max() < 1e-12 * x.grad.abs().max()
    assert (dbias - b.grad).abs().max() < 1e-12


def test_router_forms_are_autograd_s():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(50, 16, dtype=torch.float64, generator=g).requires_grad_()
    top, inds = torch.topk(x, 4)
    mask = torch.rand(50, generator=g) < 0.7
    p = torch.softmax(x, -1)
    loss, counts, weight = E.balance(x.detach(), inds.int(), mask, 0.3)
    T = int(mask.sum())
    want = 0.3 * 16 * (counts.double() / (T * 4) * p[mask].mean(0)).sum()
    assert abs(want - loss) < 1e-14
    ds = torch.randn(50, 4, dtype=torch.float64, generator=g)
    scores = p.gather(1, inds)
    scores = scores / scores.sum(-1, keepdim=True)
    (2.5 * want + ((scores * ds)[mask]).sum()).backward()
    got = E.router_gradient(x.detach(), inds.int(), ds, weight, 2.5, mask)
    assert (got - x.grad).abs().max() < 1e-14
