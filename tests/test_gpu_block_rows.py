"""Norms around a block and their gradient where a row ends inside a thread's vector, and where several rows share a workgroup
whose last set is not full."""
import pytest
import torch

from sushi_amd import _lib, exl3
from tests.test_gpu_block_norm import BF16, F16, F32, _backward_matches, _forward_matches, _make

pytestmark = pytest.mark.gpu

TYPES = [(BF16, BF16), (F16, F32), (F32, F32)]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
def test_every_row_end(dev, types, gate):
    for width in [*range(1, 18), 505, 507, 519, 1017, 1025, 1031, 2041, 2055, 4089, 4103, 6139, 6147, 8185, 8195]:
        print(f"[rows] {types} {gate} {width}", flush=True)
        d = _make(width, 3, width, *types, True, True, gate, types[0])
        _forward_matches(dev, d)
        _backward_matches(dev, d)


@pytest.mark.parametrize("width", [33, 512, 680, 1023, 1536, 2048])
def test_sets_of_rows_that_are_not_full(dev, width):
    for rows in (1, 2, 3, 4, 5, 7, 8, 9, 2047, 2057):
        print(f"[rows] {rows} of {width}", flush=True)
        d = _make(rows, rows, width, BF16, F32 if rows % 2 else BF16, True, rows % 4 != 0, ("none", "channel", "row", "full")[rows % 4], F32)
        _backward_matches(dev, d)


@pytest.mark.parametrize("width", [15, 499, 679, 1001, 1999, 4093])
def test_gradient_in_place_and_repeated(dev, width):
    """dy on y, dresidual on h: the bits of outputs of their own, and of the first call at every call."""
    rows = 1 + 8 * 257
    d = {n: None if v is None else v.to(dev) for n, v in _make(width, rows, width, BF16, BF16, True, True, "full", F32).items()}
    L, p, st = _lib.load(), lambda v: v.data_ptr(), torch.cuda.current_stream().cuda_stream
    args = (d["dh"], d["dx"], d["y"], d["h"], d["post"], d["pre"], d["gate"])
    first = exl3.block_norm_backward(*args)
    for _ in range(3):
        again = exl3.block_norm_backward(*args)
        for a, b in zip(first, again):
            assert torch.equal(a, b)
    ws = exl3.workspace.get(dev, L.exl3_block_norm_backward_workspace_size(rows, width))
    y, h = d["y"].clone(), d["h"].clone()
    dpost, dpre, dgate = torch.empty(width, device=dev), torch.empty(width, device=dev), torch.empty_like(d["gate"])
    rc = L.exl3_block_norm_backward(p(d["dh"]), p(d["dx"]), p(y), 1, p(h), 1, rows, width, p(d["post"]), 2, p(d["gate"]), 1, 3, p(d["pre"]), 2,
                                    1e-6, 0.0, 1.0, 1.0, p(y), p(h), p(dpost), p(dpre), p(dgate), p(ws), ws.numel(), st)
    assert rc == 0
    for a, b in zip(first, (y, h, dpost, dpre, dgate)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("width", [200, 680, 1500, 2561])
def test_a_row_of_nan_stays_in_its_row(dev, width):
    rows = 603
    d = {n: None if v is None else v.to(dev) for n, v in _make(2, rows, width, F16, F16, True, True, "row", F32).items()}
    clean = exl3.block_norm_backward(d["dh"], d["dx"], d["y"], d["h"], d["post"], d["pre"], d["gate"])
    for at in (0, 300, rows - 1):
        y = d["y"].clone()
        y[at, width // 2] = float("nan")
        got = exl3.block_norm_backward(d["dh"], d["dx"], y, d["h"], d["post"], d["pre"], d["gate"])
        keep = [r for r in range(rows) if r != at]
        assert torch.isnan(got.dy[at]).all() and torch.equal(got.dy[keep], clean.dy[keep])
        assert torch.equal(got.dresidual, clean.dresidual) and torch.equal(got.dgate.reshape(-1)[keep], clean.dgate.reshape(-1)[keep])
        assert torch.isnan(got.dpost_weight).all() and torch.equal(got.dpre_weight, clean.dpre_weight)
