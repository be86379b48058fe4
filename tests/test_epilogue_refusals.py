"""Buffers that must not share memory, refused before any launch (no GPU: the pointers are never dereferenced)."""
import pytest

import sushi_amd._lib as L

BASE = 1 << 40
WS = dict(ws=1 << 20, wsb=1 << 36)


def _dec():
    return L.DecodeT(1, 16, -1)


def _fwd(**kw):
    a = dict(x=BASE, xdt=0, rows=4, fin=256, fout=512, tr=1 << 30, n=64, suh=1 << 31, svh=1 << 32, dec=_dec(), bias=None,
             bdt=0, act=0, res=None, y=2 * BASE, ydt=0, pre=None, **WS)
    a.update(kw)
    return L.load().exl3_linear_epilogue(*a.values(), None), L.last_error()


def _bwd(**kw):
    a = dict(dy=BASE, dt=0, rows=4, fin=256, fout=512, tr=1 << 30, n=64, suh=1 << 31, svh=1 << 32, dec=_dec(), act=0,
             pre=None, dx=2 * BASE, xdt=0, dbias=None, **WS)
    a.update(kw)
    return L.load().exl3_linear_epilogue_backward(*a.values(), None), L.last_error()


Y = 4 * 512 * 2  # bytes of y, residual and pre
X = 4 * 256 * 2
DX = 4 * 256 * 2


@pytest.mark.parametrize("kw", [
    dict(res=2 * BASE), dict(res=2 * BASE + Y - 4), dict(res=2 * BASE - Y + 4),
    dict(pre=2 * BASE), dict(pre=2 * BASE + 16), dict(pre=3 * BASE, res=3 * BASE + Y - 16),
    dict(y=BASE), dict(y=BASE + X - 4), dict(y=BASE - Y + 4), dict(pre=BASE),
    dict(bias=2 * BASE + 64), dict(bias=2 * BASE - 1024 + 4), dict(bias=3 * BASE, bdt=2, pre=3 * BASE + 2044),
], ids=str)
def test_forward_outputs_overlap_nothing(kw):
    rc, text = _fwd(**kw)
    assert rc == -1 and "overlap" in text


@pytest.mark.parametrize("kw", [
    dict(dbias=BASE), dict(dbias=BASE + 4 * 512 * 2 - 4), dict(dbias=2 * BASE + DX - 4), dict(dbias=2 * BASE - 2048 + 4),
    dict(act=3, pre=3 * BASE, dbias=3 * BASE),
    # past a chunk of rows a later chunk's dy would hold an earlier one's dx
    dict(rows=20000, dx=BASE), dict(rows=20000, act=1, pre=3 * BASE, dx=3 * BASE),
    dict(rows=20000, fin=512, dx=BASE + 1024), dict(rows=20000, fin=512, dx=BASE, xdt=2),
], ids=str)
def test_backward_outputs_overlap_no_input_still_to_be_read(kw):
    rc, text = _bwd(**kw)
    assert rc == -1 and "overlap" in text


def test_neighbours_are_no_overlap():
    """Buffers end to end, and what only looks alike: these reach the launch, which fails without a GPU."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("the pointers here are no memory")
    for rc, text in (_fwd(), _fwd(res=2 * BASE + Y, pre=2 * BASE - Y), _fwd(res=BASE), _fwd(y=BASE + X, bias=BASE + X + Y),
                     _bwd(), _bwd(dbias=2 * BASE + DX), _bwd(dx=BASE), _bwd(act=3, pre=BASE + 4 * 512 * 2),
                     _bwd(rows=20000, fin=512, dx=BASE), _bwd(rows=20000, dx=BASE + 20000 * 1024)):
        assert rc != 0 and "overlap" not in text, text
