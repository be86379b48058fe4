"""The paths of the linears with an epilogue and of their gradients that only larger calls take, against the f64 forms of
tests/_epilogue.py: the split finish with four rows a wave, its loop over more splits than it loads at once, rows past a
chunk, and the gradient's order of tiles over the XCDs."""
import pytest
import torch

from sushi_amd import exl3
from tests import _epilogue as E
from tests.test_gpu_epilogue import _forward_case, _held, _normal, _proj

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# rows x blocks of 128 columns from 16384 on: four rows a wave.  One split, two, three and four of them (as many as such a
# call can have: its tiles are 64 or more), a last group of three rows and of one
FOUR_ROWS = [
    (203, 256, 10496, 48, "mcg", BF16, F32, "gelu", True),
    (203, 512, 10496, 32, "3inst", F32, F16, "silu", True),
    (253, 896, 8320, 96, "mul1", F16, F16, "gelu_tanh", False),
    (256, 1024, 8192, 64, "mcg", BF16, BF16, "relu", True),
    (4097, 768, 512, 24, "mcg", F32, F32, "gelu", True),
]


@pytest.mark.parametrize("case", FOUR_ROWS, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_split_finish_of_four_rows_a_wave(dev, case):
    rows, in_f, out_f, n, cb, dtype, bias_dt, act, residual = case
    assert rows * (out_f // 128) >= 16384
    _forward_case(dev, rows, in_f, out_f, n, cb, dtype, act, bias_dt, residual, True)


@pytest.mark.parametrize("rows,in_f,dtype", [(17, 2560, BF16), (17, 4352, F32), (19, 2304, F16), (130, 4096, F32)])
def test_split_finish_of_many_splits(dev, rows, in_f, dtype):
    """10, 17, 9 and 16 splits, eight of them loaded at once."""
    _forward_case(dev, rows, in_f, 128, 48, "mcg", dtype, "gelu", dtype, True, True)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_past_a_chunk_against_f64(dev, dtype):
    _forward_case(dev, 16384 + 21, 128, 128, 32, "mcg", dtype, "silu", dtype, True, True)


# rows, in, out: 1, 2, 4 and 8 row tiles whose column blocks divide among the XCDs, one block of them an XCD and more, one
# split and several, the last row tile whole and ragged
MAPPED = [(5, 1024, 128), (5, 2048, 1152), (64, 1024, 512), (300, 512, 128), (300, 1024, 768), (512, 512, 1024),
          (800, 256, 128), (1000, 512, 640), (2048, 128, 128), (2047, 256, 768)]


@pytest.mark.parametrize("rows,in_f,out_f", MAPPED)
def test_gradients_over_the_xcds(dev, rows, in_f, out_f):
    nm, nib = (rows + 255) // 256, in_f // 128
    assert 8 % nm == 0 and nib % (8 // nm) == 0
    print(f"[gradient] {rows} {in_f} {out_f}", flush=True)
    dec, odec = E.DECODES["3inst"]
    p = _proj(rows + out_f, in_f, out_f, 48, dev)
    dy = _normal(rows, "dy", (rows, out_f), BF16, dev)
    pre = _normal(rows, "pre", (rows, out_f), BF16, dev, 1.5)
    dx, dbias = exl3.linear_epilogue_backward(dy, p, dec, act="gelu", pre=pre, with_dbias=True, dx_dtype=F32)
    torch.cuda.synchronize()
    wx, bx, wb, bb = E.backward(dy, p, odec, "gelu", pre, F32)
    _held(dx, wx, bx, "dx")
    _held(dbias, wb, bb, "dbias")
