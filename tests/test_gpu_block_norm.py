"""The norms around a block with gate and residual, and their gradient, against f64 (tests/_block.py).

f32 bounds, relative to the sums of the terms' magnitudes: a sum of squares over a row loses at most one rounding for each of
a thread's 32 values, 6 + 16 joins and the squares' own, 2^-18 with room; its root half of that; then a handful of products.  So
h' is within 2^-18 of its terms' magnitudes, x' within 2^-17 of its, the gradients (two such factors, and a mean each) within
2^-16, each plus half a step of the type that it is rounded to.  A column's sum over rows adds at most one rounding a row."""
import math

import pytest
import torch

from sushi_amd import exl3
from tests import _block as R
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _make(seed, rows, width, dtype, hdtype, post, pre, gate, wdtype, offset=0.0, lead=None):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    lead = (rows,) if lead is None else lead
    d = dict(y=(n(*lead, width) * torch.exp(0.5 * n(*lead, 1))).to(dtype), h=(2 * n(*lead, width)).to(hdtype),
             post=(1 - offset + 0.2 * n(width)).to(wdtype) if post else None, pre=(1 - offset + 0.2 * n(width)).to(wdtype) if pre else None,
             gate={"none": lambda: None, "channel": lambda: (0.5 + 0.3 * n(width)).to(wdtype), "row": lambda: n(*lead, 1).to(wdtype),
                   "full": lambda: n(*lead, width).to(dtype)}[gate](),
             dh=n(*lead, width).to(hdtype), dx=n(*lead, width).to(dtype) if pre else None)
    return d


def _near(got, want, mag, rel, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -126
    bound = rel * mag
    bound = bound + E.half_step(dtype) * (want.abs() + bound) + tiny
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (what, (off / bound).max().item())


def _kw(a, b, offset, eps):
    return dict(eps=eps, weight_offset=offset, residual_scale=a, block_scale=b)


def _forward_matches(dev, d, a=1.0, b=1.0, offset=0.0, eps=1e-6, use_h=True):
    t = {n: None if v is None else v.to(dev) for n, v in d.items()}
    got = exl3.block_norm(t["y"], t["h"] if use_h else None, post_weight=t["post"], pre_weight=t["pre"], gate=t["gate"], **_kw(a, b, offset, eps))
    torch.cuda.synchronize()
    (h, x), (mh, mx) = R.norm(d["y"], d["h"] if use_h else None, d["post"], d["pre"], d["gate"], eps, offset, a, b)
    _near(got.h, h, mh, 2.0 ** -18, d["h"].dtype if use_h else d["y"].dtype, "h")
    assert (got.x is None) == (d["pre"] is None)
    if got.x is not None:
        _near(got.x, x, mx, 2.0 ** -17, d["y"].dtype, "x")
    return got


def _backward_matches(dev, d, a=1.0, b=1.0, offset=0.0, eps=1e-6, use_dh=True, with_dresidual=True):
    """d's h is taken as the forward's h'."""
    t = {n: None if v is None else v.to(dev) for n, v in d.items()}
    got = exl3.block_norm_backward(t["dh"] if use_dh else None, t["dx"], t["y"], t["h"], post_weight=t["post"], pre_weight=t["pre"],
                                   gate=t["gate"], with_dresidual=with_dresidual, **_kw(a, b, offset, eps))
    torch.cuda.synchronize()
    want = R.norm_gradient(d["dh"] if use_dh else None, d["dx"], d["y"], d["h"], d["post"], d["pre"], d["gate"], eps, offset, a, b)
    rows = d["y"].numel() // d["y"].shape[-1]
    sums = 2.0 ** -16 + rows * 2.0 ** -24
    _near(got.dy, *want[0], 2.0 ** -16, d["y"].dtype, "dy")
    if with_dresidual:
        _near(got.dresidual, *want[1], 2.0 ** -16, d["h"].dtype, "dresidual")
    else:
        assert got.dresidual is None
    for v, w, n in ((got.dpost_weight, want[2], "dpost"), (got.dpre_weight, want[3], "dpre")):
        assert (v is None) == (w[0] is None)
        if v is not None:
            _near(v, *w, sums, F32, n)
    assert (got.dgate is None) == (d["gate"] is None)
    if got.dgate is not None:
        full = d["gate"].shape == d["y"].shape and d["gate"].dim() > 1 and d["y"].shape[-1] > 1
        _near(got.dgate, want[4][0].reshape(d["gate"].shape), want[4][1].reshape(d["gate"].shape), sums if not full else 2.0 ** -16,
              d["gate"].dtype if full else F32, "dgate")
    return got


# rows, width, dtype, hdtype, post, pre, gate, wdtype
CASES = [
    (1, 1, F32, F32, True, True, "none", F32), (2, 3, F16, F16, True, True, "channel", F16), (3, 7, BF16, F32, True, False, "row", F32),
    (5, 8, BF16, BF16, False, True, "full", BF16), (1, 64, F16, F32, True, True, "row", F16), (7, 127, BF16, BF16, True, True, "full", F32),
    (4, 128, F32, F32, True, True, "channel", F32), (9, 511, F16, F16, True, True, "none", F32), (6, 512, BF16, F32, False, True, "channel", F32),
    (5, 513, BF16, BF16, True, True, "channel", BF16), (3, 1000, F32, F32, False, False, "full", F32), (33, 2048, F16, F32, True, True, "full", F16),
    (17, 2049, BF16, BF16, True, True, "row", BF16), (1, 4096, BF16, BF16, True, True, "none", BF16), (5, 4095, F16, F16, True, False, "channel", F32),
    (600, 640, BF16, BF16, True, True, "channel", F32), (1500, 256, F16, F32, True, True, "row", F32), (12, 5120, F16, F32, False, True, "channel", F32),
    (3, 8192, F32, F32, True, True, "full", F32), (4, 8193, BF16, BF16, True, True, "channel", F32), (2, 16384, F16, F32, True, True, "row", F16),
    (1, 16381, BF16, F32, True, True, "full", BF16), (530, 16384, BF16, BF16, True, True, "channel", BF16), (0, 256, BF16, BF16, True, True, "channel", F32),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_norm_and_gradient_against_f64(dev, case):
    print(f"[norm] {case}", flush=True)
    d = _make(case[0] + case[1], *case)
    if case[0] == 0:
        t = {n: None if v is None else v.to(dev) for n, v in d.items()}
        got = exl3.block_norm(t["y"], t["h"], t["post"], t["pre"], t["gate"])
        assert got.h.shape == got.x.shape == (0, 256)
        g = exl3.block_norm_backward(t["dh"], t["dx"], t["y"], t["h"], t["post"], t["pre"], t["gate"])
        assert g.dy.shape == (0, 256) and not g.dpost_weight.any() and not g.dpre_weight.any() and not g.dgate.any()
        return
    _forward_matches(dev, d)
    _backward_matches(dev, d)


@pytest.mark.parametrize("kw", [dict(a=0.5, b=0.22), dict(offset=1.0), dict(eps=1e-2, a=-1.0), dict(a=0.0), dict(b=0.0, offset=1.0)], ids=str)
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
def test_scales_offsets_and_what_is_left_out(dev, gate, kw):
    for post, pre in ((True, True), (True, False), (False, True), (False, False)):
        d = _make(3, 37, 320, BF16, F32, post, pre, gate, F32, offset=kw.get("offset", 0.0))
        _forward_matches(dev, d, **kw)
        _backward_matches(dev, d, **kw)
        _backward_matches(dev, d, with_dresidual=False, **kw)
        if pre:
            _backward_matches(dev, d, use_dh=False, **kw)
        one = dict(d, h=d["h"].to(BF16))
        _forward_matches(dev, one, use_h=False, **kw)


def test_rows_of_zeros_extremes_and_other_rows_untouched(dev):
    d = _make(5, 40, 384, F32, F32, True, True, "channel", F32)
    d["y"][3], d["h"][3] = 0, 0
    d["y"][4], d["h"][5] = 0, 0
    d["y"][6] *= 1e15
    d["h"][7] *= 1e15
    d["y"][8] *= 1e-18          # below eps: the norm scales by 1 / sqrt(eps)
    got = _forward_matches(dev, d)
    assert not got.h[3].any() and not got.x[3].any()
    _backward_matches(dev, d)
    clean = exl3.block_norm(*(d[n].to(dev) for n in ("y", "h", "post", "pre", "gate")))
    for bad in (math.nan, math.inf):
        y = d["y"].clone()
        y[11, 5] = bad
        got = exl3.block_norm(y.to(dev), *(d[n].to(dev) for n in ("h", "post", "pre", "gate")))
        assert torch.isnan(got.x[11]).any()
        keep = [r for r in range(40) if r != 11]
        assert torch.equal(got.h[keep], clean.h[keep]) and torch.equal(got.x[keep], clean.x[keep])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width", [96, 1000, 4097])
def test_norm_at_every_alignment(dev, dtype, width):
    """Operands that begin one element into their storage, rows of odd widths: the bits of the aligned ones."""
    d = _make(7, 19, width, dtype, dtype, True, True, "full", dtype)
    def shift(v):
        base = torch.empty(v.numel() + 1, dtype=v.dtype, device=dev)
        base[1:] = v.reshape(-1).to(dev)
        return base[1:].view(v.shape)
    t = {n: v.to(dev) for n, v in d.items()}
    u = {n: shift(v) for n, v in d.items()}
    for s in (t, u):
        s["out"] = exl3.block_norm(s["y"], s["h"], s["post"], s["pre"], s["gate"])
        s["grad"] = exl3.block_norm_backward(s["dh"], s["dx"], s["y"], s["h"], s["post"], s["pre"], s["gate"])
    assert all(torch.equal(a, b) for a, b in zip((*t["out"], *t["grad"]), (*u["out"], *u["grad"])))


def test_leading_dims_a_lone_row_and_equal_bits(dev):
    d = _make(9, 0, 768, BF16, BF16, True, True, "row", F32, lead=(3, 5))
    a = _forward_matches(dev, d)
    assert a.h.shape == a.x.shape == (3, 5, 768)
    g = _backward_matches(dev, d)
    assert g.dgate.shape == (3, 5, 1)
    one = {n: None if v is None else v[1, 2] if v.dim() == 3 else v for n, v in d.items()}
    b = _forward_matches(dev, one)
    assert torch.equal(b.h, a.h[1, 2]) and torch.equal(b.x, a.x[1, 2])
    gb = _backward_matches(dev, one)
    assert gb.dy.shape == (768,) and torch.equal(gb.dy, g.dy[1, 2]) and torch.equal(gb.dresidual, g.dresidual[1, 2])
    big = {n: None if v is None else v.to(dev) for n, v in _make(10, 3000, 512, BF16, F32, True, True, "channel", F32).items()}
    call = lambda: exl3.block_norm_backward(big["dh"], big["dx"], big["y"], big["h"], big["post"], big["pre"], big["gate"])  # noqa: E731
    first = call()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, call()))


@pytest.mark.parametrize("width", [72, 640, 4100])
def test_outputs_in_their_inputs_place(dev, width):
    """Through the C ABI: h_out on h and x_out on y, dy on y or dx and dresidual on dh or h, hold what the others do."""
    from sushi_amd import _lib

    L, st = _lib.load(), torch.cuda.current_stream(dev).cuda_stream
    t = {n: None if v is None else v.to(dev) for n, v in _make(11, 700, width, BF16, BF16, True, True, "channel", F32).items()}
    want = exl3.block_norm(t["y"], t["h"], t["post"], t["pre"], t["gate"])
    y, h = t["y"].clone(), t["h"].clone()
    p = lambda v: v.data_ptr()  # noqa: E731
    mid = (p(t["post"]), 2, p(t["gate"]), 2, 1, p(t["pre"]), 2, 1e-6, 0.0, 1.0, 1.0)
    assert L.exl3_block_norm(p(y), 1, p(h), 1, 700, width, *mid, p(h), p(y), st) == 0
    torch.cuda.synchronize()
    assert torch.equal(h, want.h) and torch.equal(y, want.x)
    grads = exl3.block_norm_backward(t["dh"], t["dx"], t["y"], t["h"], t["post"], t["pre"], t["gate"])
    ws = exl3.workspace.get(dev, L.exl3_block_norm_backward_workspace_size(700, width))
    sums = [torch.empty(width, device=dev) for _ in range(3)]
    for dy_on, dres_on in (("y", "dh"), ("dx", "h")):
        c = {n: t[n].clone() for n in ("dh", "dx", "y", "h")}
        assert L.exl3_block_norm_backward(p(c["dh"]), p(c["dx"]), p(c["y"]), 1, p(c["h"]), 1, 700, width, *mid, p(c[dy_on]), p(c[dres_on]),
                                          *(p(s) for s in sums), ws.data_ptr(), ws.numel(), st) == 0
        torch.cuda.synchronize()
        assert torch.equal(c[dy_on], grads.dy) and torch.equal(c[dres_on], grads.dresidual)
        assert all(torch.equal(s, g) for s, g in zip(sums, grads[2:]))


def test_gradient_is_the_forward_s_difference(dev):
    """block_norm's own f32 outputs, differenced along random directions of every input, against the gradient: L = <h', r> +
    <x', s>.  A difference over 2 h with h = 2^-6 is off by h^2 / 6 of the third derivative and by the outputs' f32 error over h."""
    d = {n: None if v is None else v.to(dev) for n, v in _make(13, 8, 64, F32, F32, True, True, "channel", F32).items()}
    call = lambda **o: exl3.block_norm(*({**d, **o}[n] for n in ("y", "h", "post", "pre", "gate")), residual_scale=0.7, block_scale=0.3)  # noqa: E731
    new = call()
    g = exl3.block_norm_backward(d["dh"], d["dx"], d["y"], new.h, d["post"], d["pre"], d["gate"], residual_scale=0.7, block_scale=0.3)
    def loss(o):
        return ((o.h.double() * d["dh"].double()).sum() + (o.x.double() * d["dx"].double()).sum()).item()
    step = 2.0 ** -6
    for name, grad in zip(("y", "h", "post", "pre", "gate"), g):
        v = torch.randn(d[name].shape, device=dev, generator=torch.Generator(dev).manual_seed(4))
        v = v / v.norm()
        diff = (loss(call(**{name: d[name] + step * v})) - loss(call(**{name: d[name] - step * v}))) / (2 * step)
        want = (grad.double() * v.double()).sum().item()
        assert abs(diff - want) <= 2.0 ** -9 * grad.double().norm().item(), (name, diff, want)
