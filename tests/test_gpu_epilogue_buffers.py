"""The gradient with dx in the place of dy (the C entry reads a chunk's dy whole before it writes the chunk's dx), and with
pre at the least alignment that is documented."""
import pytest
import torch

import sushi_amd._lib as L
from sushi_amd import exl3
from tests.test_gpu_epilogue import _normal, _proj

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width", [(3, 1024), (300, 256), (16384 + 21, 128)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_dx_in_place_of_dy(dev, rows, width, act):
    p = _proj(81, width, width, 48, dev)
    dy, pre = (_normal(82, n, (rows, width), torch.bfloat16, dev) for n in ("dy", "pre"))
    want, db = exl3.linear_epilogue_backward(dy, p, exl3.MCG, act=act, pre=pre, with_dbias=True)
    lib = L.load()
    ws = exl3.workspace.get(dev, lib.exl3_linear_epilogue_backward_workspace_size(rows, width, width))
    got = torch.empty_like(db)
    rc = lib.exl3_linear_epilogue_backward(dy.data_ptr(), 1, rows, width, width, p.trellis.data_ptr(), 48, p.suh.data_ptr(),
                                           p.svh.data_ptr(), exl3.MCG.c(), exl3.ACTIVATIONS[act], pre.data_ptr(),
                                           dy.data_ptr(), 1, got.data_ptr(), ws.data_ptr(), ws.numel(),
                                           torch.cuda.current_stream(dev).cuda_stream)
    assert rc == 0, L.last_error()
    torch.cuda.synchronize()
    assert torch.equal(dy, want) and torch.equal(got, db)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_pre_at_eight_bytes(dev, dtype):
    """pre needs no more than 8-byte alignment, also where a row is read 16 bytes at a time."""
    p = _proj(83, 256, 640, 32, dev)
    dy, pre = (_normal(84, n, (70, 640), dtype, dev) for n in ("dy", "pre"))
    skip = 8 // pre.element_size()
    odd = torch.empty(70 * 640 + skip, dtype=dtype, device=dev)[skip:].view(70, 640)
    odd.copy_(pre)
    assert odd.data_ptr() % 16 == 8
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        a = exl3.linear_epilogue_backward(dy, p, exl3.MCG, act=act, pre=pre, with_dbias=True)
        b = exl3.linear_epilogue_backward(dy, p, exl3.MCG, act=act, pre=odd, with_dbias=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
