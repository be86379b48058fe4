"""The linear with a bias, activation and residual in its epilogue, and its gradients, against f64 with bounds that count
roundings (tests/_epilogue.py)."""
import pytest
import torch

from sushi_amd import exl3, synth
from tests import _epilogue as E

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _proj(seed, in_f, out_f, n, dev):
    p = synth.proj(seed, f"ep{in_f}.{out_f}.{n}", 1, in_f, out_f, n, norm=True)
    return exl3.Proj(p.trellis.to(dev), p.suh.to(dev), p.svh.to(dev))


def _normal(seed, name, shape, dtype, dev, scale=1.0):
    return (synth.normal(seed, name, shape, dtype=F32) * scale).to(dtype).to(dev)


def _held(got, want, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    print(f"  {what}: worst {worst:.3f} of its bound", flush=True)
    assert bool((off <= bound).all()), f"{what}: {worst} times its bound"


def _forward_case(dev, rows, in_f, out_f, n, cb, dtype, act, bias_dt, residual, pre, out_dtype=None):
    print(f"[epilogue] rows={rows} {in_f}x{out_f} n={n} {cb} {dtype} {act} bias={bias_dt} res={residual} pre={pre}",
          flush=True)
    dec, odec = E.DECODES[cb]
    p = _proj(n + rows, in_f, out_f, n, dev)
    x = _normal(rows, "x", (rows, in_f), dtype, dev)
    bias = None if bias_dt is None else _normal(rows, "bias", (out_f,), bias_dt, dev)
    dt = out_dtype or dtype
    res = _normal(rows, "res", (rows, out_f), dt, dev, 2.0) if residual else None
    got = exl3.linear_epilogue(x, p, dec, bias=bias, act=act, residual=res, out_dtype=out_dtype, with_pre=pre)
    y, z = got if pre else (got, None)
    torch.cuda.synchronize()
    wy, by, wz, bz = E.forward(x, p, odec, bias, act, res, out_dtype)
    assert y.dtype == dt and tuple(y.shape) == (rows, out_f)
    _held(y, wy, by, "y")
    if pre:
        assert z.dtype == dt
        _held(z, wz, bz, "pre")


# rows up to 16 take the decode GEMV (one split, the fold, f32 planes, row groups), wider ones the GEMM; n = 18 and 72 the
# generic readers, n = 80 .. 128 the wide lane readers
FORWARD = [
    (1, 256, 128, 64, "3inst", F16, "none", F16, True, False, None),
    (1, 1024, 384, 48, "mcg", BF16, "gelu", BF16, False, True, None),
    (1, 1024, 256, 32, "mul1", F32, "silu", F32, True, True, None),
    (2, 512, 128, 24, "spec1", F16, "relu", F32, True, True, None),
    (3, 640, 256, 40, "mcg", BF16, "gelu_tanh", F16, True, True, F32),
    (5, 1024, 256, 16, "mcg", F16, "silu", BF16, True, True, None),
    (7, 1024, 256, 48, "pair1", BF16, "none", None, True, False, None),
    (8, 512, 384, 96, "mcg", F16, "gelu", None, False, True, BF16),
    (16, 1024, 128, 128, "3inst", BF16, "gelu_tanh", BF16, True, False, None),
    (16, 256, 256, 18, "mcg", F16, "relu", F16, True, True, None),
    (13, 384, 128, 72, "mul1", F32, "gelu", F32, True, True, F16),
    (17, 256, 128, 64, "3inst", F16, "gelu", F16, True, True, None),
    (33, 512, 256, 48, "mcg", BF16, "none", None, True, False, None),
    (130, 384, 384, 32, "spec1", F32, "gelu_tanh", F32, True, True, None),
    (257, 256, 256, 40, "mcg_w12", F16, "silu", F32, False, True, None),
    (300, 256, 128, 64, "pair1", BF16, "relu", BF16, True, True, None),
    (40, 256, 256, 112, "mul1", F16, "silu", F16, True, False, F32),
    (21, 384, 128, 18, "mcg", BF16, "gelu", BF16, True, True, None),
    (35, 256, 256, 72, "3inst", F32, "silu", F32, True, True, F16),
]


@pytest.mark.parametrize("case", FORWARD, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_epilogue_against_f64(dev, case):
    _forward_case(dev, *case)


@pytest.mark.parametrize("arm", [4, 5, 6, 7])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,cb", [(48, "3inst"), (24, "spec1")])
def test_epilogue_on_every_gemm_tile(dev, arm, dtype, n, cb):
    """Every dense GEMM body, whole and ragged row tiles, with and without the residual."""
    with exl3.arm_overrides(gemm_arm=arm):
        _forward_case(dev, 530, 256, 256, n, cb, dtype, "gelu", dtype, True, True)
        _forward_case(dev, 512, 384, 128, n, cb, dtype, "silu", None, False, False)


@pytest.mark.parametrize("knobs", [dict(gemv_splits=1), dict(gemv_splits=4), dict(gemv_splits=4, gemv_fold=0),
                                   dict(gemv_splits=8, gemv_separate_finish=1), dict(gemv_rows_per_group=2)],
                         ids=lambda k: "-".join(f"{a}={b}" for a, b in k.items()))
def test_epilogue_on_every_gemv_finish(dev, knobs):
    with exl3.arm_overrides(**knobs):
        _forward_case(dev, 5, 1024, 256, 48, "mcg", F16, "gelu", F32, True, True)
        _forward_case(dev, 1, 1024, 128, 32, "mcg", BF16, "silu", BF16, True, True)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [1, 4, 11, 16, 31, 300, 700])
@pytest.mark.parametrize("n", [48, 96, 18])
def test_an_empty_epilogue_is_linear_bit_for_bit(dev, rows, n, dtype):
    """On one arm: unpinned, wider calls split k where exl3_linear does not."""
    p = _proj(3, 512, 384, n, dev)
    x = _normal(4, "x", (rows, 512), dtype, dev)
    with exl3.arm_overrides(gemm_arm=4):
        assert torch.equal(exl3.linear_epilogue(x, p, exl3.MCG), exl3.linear(x, p, exl3.MCG))
    if rows <= 16 or n == 18:
        assert torch.equal(exl3.linear_epilogue(x, p, exl3.MCG), exl3.linear(x, p, exl3.MCG))


# rows, in, out: one split through the planes, two and more with uneven parts, row tiles of 64, 128, 192 and 256 rows with
# and without a rest, row counts whose plain linear takes another tile
SPLIT = [(17, 128, 128), (17, 640, 128), (64, 256, 384), (65, 1152, 256), (128, 512, 128), (129, 896, 128),
         (256, 768, 256), (257, 640, 128), (320, 1408, 128), (384, 512, 256), (385, 512, 128), (513, 768, 256),
         (577, 512, 128)]


@pytest.mark.parametrize("n,cb,dtype", [(48, "3inst", BF16), (24, "pair1", F16), (128, "mul1", F32), (40, "spec1", BF16)])
@pytest.mark.parametrize("rows,in_f,out_f", SPLIT)
def test_epilogue_with_k_in_splits(dev, rows, in_f, out_f, n, cb, dtype):
    _forward_case(dev, rows, in_f, out_f, n, cb, dtype, "gelu", dtype, True, True)


def test_row_splits_past_the_halves_tile(dev):
    """Rows and widths where the plain linear takes k in halves or the 512-row tile keep those."""
    for rows, out_f in ((300, 10240), (520, 12288)):
        p = _proj(31, 256, out_f, 48, dev)
        x = _normal(31, "x", (rows, 256), F16, dev)
        assert torch.equal(exl3.linear_epilogue(x, p, exl3.MCG), exl3.linear(x, p, exl3.MCG))


def test_epilogue_of_unaligned_and_small_operands(dev):
    """A residual at 4 bytes past 16 (the GEMM's stores then go element by element), and no rows at all."""
    p = _proj(5, 256, 256, 48, dev)
    for dtype in (F16, BF16):
        x = _normal(6, "x", (530, 256), dtype, dev)
        res = _normal(6, "r", (530, 256), dtype, dev)
        room = torch.empty(530 * 256 + 2, dtype=dtype, device=dev)
        odd = room[2:].view(530, 256)
        odd.copy_(res)
        assert odd.data_ptr() % 16 == 4
        for arm in (4, 5, 7):
            with exl3.arm_overrides(gemm_arm=arm):
                a = exl3.linear_epilogue(x, p, exl3.MCG, act="gelu", residual=res, with_pre=True)
                b = exl3.linear_epilogue(x, p, exl3.MCG, act="gelu", residual=odd, with_pre=True)
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    none = exl3.linear_epilogue(torch.empty(0, 256, dtype=F16, device=dev), p, exl3.MCG, act="gelu", with_pre=True)
    assert tuple(none[0].shape) == (0, 256) and tuple(none[1].shape) == (0, 256)


def test_epilogue_rows_are_their_own(dev):
    """A row of inf or NaN leaves every other row's bits as they were; large sums go past the fold's range."""
    p = _proj(7, 512, 256, 48, dev)
    res = _normal(8, "r", (6, 256), F16, dev)
    x = _normal(8, "x", (6, 512), F16, dev)
    want = exl3.linear_epilogue(x, p, exl3.MCG, act="silu", residual=res)
    bad = x.clone()
    bad[1, 3], bad[4, 100] = float("nan"), float("inf")
    got = exl3.linear_epilogue(bad, p, exl3.MCG, act="silu", residual=res)
    keep = [0, 2, 3, 5]
    assert torch.equal(got[keep], want[keep])
    assert not torch.isfinite(got[1]).any() and not torch.isfinite(got[4]).any()
    big = exl3.Proj(p.trellis, p.suh, (p.svh.float() * 2000).half())
    xb = (x.float() * 1000).half()
    y = exl3.linear_epilogue(xb.to(BF16), big, exl3.MCG, act="relu", residual=res.to(BF16))
    wy, by, _, _ = E.forward(xb.to(BF16), big, E.DECODES["mcg"][1], None, "relu", res.to(BF16))
    assert wy.abs().max() > 2 ** 21  # past one term of the fold's fixed point
    _held(y, wy, by, "y past the fold's range")


def test_epilogue_of_extreme_pre_activations(dev):
    """Bias of +-inf, NaN, huge and tiny values through every activation: the limits of each, and NaN only where the
    activation has none."""
    p = _proj(9, 256, 128, 32, dev)
    x = torch.zeros(1, 256, dtype=F32, device=dev)
    vals = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 50.0, -50.0, 3e38, -3e38, float("inf"), float("nan")])
    bias = torch.zeros(128)
    bias[:10] = vals
    for act in E.ACTS:
        y, pre = exl3.linear_epilogue(x, p, exl3.MCG, bias=bias.to(dev), act=act, with_pre=True)
        y = y[0, :10].double().cpu()
        assert torch.equal(pre[0].cpu().nan_to_num(7.0), bias.nan_to_num(7.0))
        want = vals.double() if act == "none" else E.act(vals.double(), act)
        fin = torch.isfinite(want)
        # z is exact here; below 2^-126 a product of f32 may vanish
        assert ((y - want).abs()[fin] <= E.ACT_ERR * want.abs()[fin] + 2.0 ** -126).all(), (act, y, want)
        assert y[9].isnan() and y[8] == float("inf")


# ---- gradients

BACKWARD = [
    (1, 128, 256, 64, "3inst", F16, "none", True, None),
    (1, 384, 1024, 48, "mcg", BF16, "gelu", True, None),
    (5, 256, 640, 32, "mul1", F32, "silu", True, None),
    (16, 256, 512, 24, "spec1", F16, "relu", False, F32),
    (17, 384, 384, 40, "mcg", BF16, "gelu_tanh", True, F32),
    (33, 128, 128, 16, "mcg_w12", F32, "gelu", True, BF16),
    (64, 256, 1152, 48, "pair1", BF16, "silu", True, None),
    (65, 512, 256, 96, "mcg", F16, "none", False, None),
    (129, 256, 256, 128, "3inst", BF16, "relu", True, None),
    (200, 128, 512, 112, "mul1", F32, "gelu_tanh", True, None),
    (257, 256, 384, 80, "spec1", BF16, "silu", True, F16),
    (300, 384, 128, 18, "mcg", F16, "gelu", True, None),
    (40, 256, 256, 72, "3inst", BF16, "none", True, None),
    (31, 128, 384, 30, "pair1", F32, "silu", True, None),
    (515, 128, 128, 64, "mcg", F16, "gelu", True, None),
]


@pytest.mark.parametrize("case", BACKWARD, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_gradients_against_f64(dev, case):
    rows, in_f, out_f, n, cb, dtype, act, with_dbias, dx_dtype = case
    print(f"[gradient] {case}", flush=True)
    dec, odec = E.DECODES[cb]
    p = _proj(n + rows, in_f, out_f, n, dev)
    dy = _normal(rows, "dy", (rows, out_f), F32, dev)
    dy = (dy * torch.exp2(torch.arange(rows, device=dev) % 9 - 12.0)[:, None]).to(dtype)  # each row at its own scale
    pre = _normal(rows, "pre", (rows, out_f), dtype, dev, 1.5)
    dx, dbias = exl3.linear_epilogue_backward(dy, p, dec, act=act, pre=pre, with_dbias=with_dbias, dx_dtype=dx_dtype)
    torch.cuda.synchronize()
    wx, bx, wb, bb = E.backward(dy, p, odec, act, pre, dx_dtype)
    assert dx.dtype == (dx_dtype or dtype) and tuple(dx.shape) == (rows, in_f)
    _held(dx, wx, bx, "dx")
    if with_dbias:
        assert dbias.dtype == F32
        _held(dbias, wb, bb, "dbias")
    else:
        assert dbias is None


@pytest.mark.parametrize("rows,in_f,out_f", [(256, 128, 256), (320, 256, 384), (384, 128, 256), (385, 128, 256),
                                             (512, 256, 128), (513, 128, 256), (576, 384, 256), (577, 128, 256),
                                             (2089, 128, 8192)])
def test_gradients_at_the_ends_of_row_tiles(dev, rows, in_f, out_f):
    """Row tiles of 192 and 256 rows, full and with a rest, and the prepare that takes four row tiles a workgroup."""
    dec, odec = E.DECODES["mcg"]
    p = _proj(rows, in_f, out_f, 48, dev)
    dy = _normal(rows, "dy", (rows, out_f), BF16, dev)
    pre = _normal(rows, "pre", (rows, out_f), BF16, dev, 1.5)
    dx, dbias = exl3.linear_epilogue_backward(dy, p, dec, act="silu", pre=pre, with_dbias=True)
    torch.cuda.synchronize()
    wx, bx, wb, bb = E.backward(dy, p, odec, "silu", pre, None)
    _held(dx, wx, bx, "dx")
    _held(dbias, wb, bb, "dbias")


@pytest.mark.parametrize("scale", [1e-30, 1e-7, 1e4, 1e30])
def test_gradients_of_any_scale(dev, scale):
    """f16's range bounds neither small nor large gradients: every row's prepared values are rescaled."""
    p = _proj(11, 256, 384, 48, dev)
    dy = _normal(12, "dy", (20, 384), F32, dev) * scale
    dy[3] = 0.0
    dx, dbias = exl3.linear_epilogue_backward(dy, p, exl3.MCG, with_dbias=True)
    wx, bx, wb, bb = E.backward(dy, p, E.DECODES["mcg"][1])
    _held(dx, wx, bx, "dx")
    _held(dbias, wb, bb, "dbias")
    assert not dx[3].any()


def test_gradient_rows_are_their_own(dev):
    p = _proj(13, 256, 256, 32, dev)
    dy = _normal(14, "dy", (37, 256), BF16, dev)
    pre = _normal(14, "pre", (37, 256), BF16, dev)
    want, _ = exl3.linear_epilogue_backward(dy, p, exl3.MCG, act="gelu", pre=pre)
    bad = dy.clone()
    bad[2, 9], bad[20, 0] = float("nan"), float("-inf")
    got, _ = exl3.linear_epilogue_backward(bad, p, exl3.MCG, act="gelu", pre=pre)
    keep = [r for r in range(37) if r not in (2, 20)]
    assert torch.equal(got[keep], want[keep])
    assert not torch.isfinite(got[2]).any() and not torch.isfinite(got[20]).any()
    # slopes at their limits: 0 left and 1 right, whatever the gradient multiplies
    far = torch.where(torch.arange(256, device=dev) % 2 == 0, 1e30, -1e30).to(BF16).expand(37, 256).contiguous()
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        _, db = exl3.linear_epilogue_backward(dy, p, exl3.MCG, act=act, pre=far, with_dbias=True)
        _, none = exl3.linear_epilogue_backward(dy, p, exl3.MCG, with_dbias=True)
        assert torch.equal(db[::2], none[::2]) and not db[1::2].any()


def test_gradients_are_the_formula_s_differences(dev):
    """<dx, d> against the central difference of the unrounded f64 forward along d: the prepared values' f16 roundings are
    all that lies between them (2^-11 of each factor's magnitude, summed over the widths in the worst case)."""
    dec, odec = E.DECODES["3inst"]
    p = _proj(15, 256, 384, 64, dev)
    w, suh, svh = E.weights(p, odec), p.suh[0].cpu().double(), p.svh[0].cpu().double()
    x = _normal(16, "x", (9, 256), F32, dev).double().cpu()
    bias = _normal(16, "b", (384,), F32, dev)
    dy = _normal(16, "dy", (9, 384), F32, dev)
    f = lambda v: E.act(E.had(E.had(v * suh) @ w) * svh + bias.double().cpu(), "gelu")  # noqa: E731
    pre = (E.had(E.had(x * suh) @ w) * svh + bias.double().cpu()).float().to(dev)
    dx, dbias = exl3.linear_epilogue_backward(dy, p, dec, act="gelu", pre=pre, with_dbias=True)
    g = dy.double().cpu()
    v = (g * E.slope(pre.double().cpu(), "gelu") * svh)
    # |error of dx| <= (2^-11 |H v| + the scale's subnormal step, 2^-36 of the row's top) |W| through H and suh
    du = 2.0 ** -11 * E.had(v).abs() + 2.0 ** -36 * v.abs().amax(1, keepdim=True)
    room = E.block_sum(du @ w.t().abs()) / 128 ** 0.5 * suh.abs()
    for i in range(4):
        d = synth.normal(17, f"d{i}", (9, 256), dtype=F32).double()
        h = 1e-5
        diff = ((f(x + h * d) - f(x - h * d)) / (2 * h) * g).sum()
        got = (dx.double().cpu() * d).sum()
        assert abs(got - diff) <= (room * d.abs()).sum() + 1e-6 * diff.abs(), (got, diff)
    h = 1e-5
    fb = lambda s: (E.act(pre.double().cpu() + s, "gelu") * g).sum(0)  # noqa: E731
    diff = (fb(h) - fb(-h)) / (2 * h)
    assert ((dbias.double().cpu() - diff).abs() <= 1e-5 * g.abs().sum(0)).all()


def test_rows_past_a_chunk(dev):
    """16384 rows and the rest run as launches of their own: forward and gradient equal those of the slices, bit for
    bit."""
    p = _proj(19, 128, 128, 32, dev)
    rows, cut = 16384 + 21, 16384
    x = torch.randn(rows, 128, device=dev, generator=torch.Generator(dev).manual_seed(5)).to(F16)
    y, pre = exl3.linear_epilogue(x, p, exl3.MCG, act="silu", residual=x, with_pre=True)
    a = exl3.linear_epilogue(x[:cut], p, exl3.MCG, act="silu", residual=x[:cut], with_pre=True)
    b = exl3.linear_epilogue(x[cut:], p, exl3.MCG, act="silu", residual=x[cut:], with_pre=True)
    assert torch.equal(y, torch.cat([a[0], b[0]])) and torch.equal(pre, torch.cat([a[1], b[1]]))
    dx, dbias = exl3.linear_epilogue_backward(x, p, exl3.MCG, act="silu", pre=pre, with_dbias=True)
    da, ba = exl3.linear_epilogue_backward(x[:cut], p, exl3.MCG, act="silu", pre=pre[:cut], with_dbias=True)
    db, bb = exl3.linear_epilogue_backward(x[cut:], p, exl3.MCG, act="silu", pre=pre[cut:], with_dbias=True)
    assert torch.equal(dx, torch.cat([da, db]))
    total = x.double() * E.slope(pre.double().cpu(), "silu").to(dev)
    for got, part in ((dbias, total), (ba, total[:cut]), (bb, total[cut:])):
        # ceil(rows / 64) rows a tile, 4 waves, 64 tiles: under 512 additions a term passes
        bound = ((512 * 2.0 ** -24 + E.ACT_ERR) * part.abs()).sum(0) + 2.0 ** -17 * x.abs().double().sum(0)
        assert ((got.double() - part.sum(0)).abs() <= bound).all()


@pytest.mark.parametrize("rows", [1, 7, 48])
def test_epilogue_in_a_graph(dev, rows):
    """Forward and backward captured together and replayed over new inputs, with eager calls between the replays."""
    p = _proj(21, 512, 512, 48, dev)
    x = _normal(22, "x", (rows, 512), BF16, dev)
    bias = _normal(22, "b", (512,), F32, dev)
    dy = _normal(22, "dy", (rows, 512), BF16, dev)

    def step():
        y, pre = exl3.linear_epilogue(x, p, exl3.INST3, bias=bias, act="gelu_tanh", residual=x, with_pre=True)
        dx, db = exl3.linear_epilogue_backward(dy, p, exl3.INST3, act="gelu_tanh", pre=pre, with_dbias=True)
        return y, pre, dx, db

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    for i in range(4):
        x.copy_(_normal(30 + i, "x", (rows, 512), BF16, dev))
        dy.copy_(_normal(30 + i, "dy", (rows, 512), BF16, dev))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want), i


def test_streams_have_their_own_scratch(dev):
    p = _proj(23, 1024, 512, 48, dev)
    xs = [_normal(24 + i, "x", (9, 1024), F16, dev) for i in range(2)]
    want = [exl3.linear_epilogue_backward(exl3.linear_epilogue(x, p, exl3.MCG, act="silu"), p, exl3.MCG)[0] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = exl3.linear_epilogue_backward(exl3.linear_epilogue(xs[i], p, exl3.MCG, act="silu"), p, exl3.MCG)[0]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i], want[i])


def test_operators_share_a_workspace_and_streams_do_not(dev):
    """The fold's words, the joins' counters and the splits' planes on one buffer, call after call in any order, and on two
    streams at once: every result as when it ran alone."""
    p = _proj(41, 1024, 512, 48, dev)
    one, many = _normal(42, "a", (3, 1024), F16, dev), _normal(42, "b", (77, 1024), F16, dev)
    dy = _normal(42, "d", (77, 512), F16, dev)
    logits = _normal(42, "l", (9000, 64), BF16, dev)
    inds = torch.randint(0, 64, (9000, 4), dtype=torch.int32, device=dev, generator=torch.Generator(dev).manual_seed(7))
    calls = [lambda: exl3.moe_balance_loss(logits, inds), lambda: (exl3.linear(one, p, exl3.MCG),),
             lambda: (exl3.linear_epilogue(many, p, exl3.MCG, act="silu"),),
             lambda: exl3.linear_epilogue_backward(dy, p, exl3.MCG, with_dbias=True),
             lambda: (exl3.linear_epilogue(one, p, exl3.MCG, act="gelu", residual=dy[:3]),)]
    want = []
    for call in calls:
        want.append(call())
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for step in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                got += [(k, calls[k]()) for k in ((step + 2 * i + j) % 5 for j in range(5))]
    torch.cuda.synchronize()
    for k, outs in got:
        for a, b in zip(outs, want[k]):
            assert torch.equal(a, b), k
