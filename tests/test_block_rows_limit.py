"""Rows past what the library counts are refused, not counted modulo 2^32 (no GPU: the tensors are views of one value)."""
import pytest
import torch

from sushi_amd import exl3

ROWS = (1 << 32) + 4


def _view(*shape, dtype=torch.float32):
    return torch.zeros((), dtype=dtype).expand(*shape)


def test_rows_past_31_bits_are_refused():
    lg, y, inds = _view(ROWS, 8), _view(4, ROWS // 4, 2), _view(ROWS, 2, dtype=torch.int32)
    for call in (lambda: exl3.moe_route(lg, 2), lambda: exl3.moe_route_backward(lg, inds, _view(ROWS, 2)),
                 lambda: exl3.moe_balance_loss(lg, inds), lambda: exl3.moe_router_backward(lg, inds, _view(ROWS, 2)),
                 lambda: exl3.block_norm(y), lambda: exl3.block_norm_backward(y, None, y, None),
                 lambda: exl3.moe_route(_view(1 << 31, 8), 2)):
        with pytest.raises(exl3.BadExl3Shape, match="rows"):
            call()
    with pytest.raises(exl3.BadExl3Shape, match="device tensors"):  # as many as there may be
        exl3.moe_route(_view((1 << 31) - 1, 8), 2)
