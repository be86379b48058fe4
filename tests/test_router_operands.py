"""One token's logits without a leading dimension: what moe_routing_chain takes, the balance loss and the gradient of the
logits take too.  Without a GPU: host tensors are refused for being that, not for their shape."""
import pytest
import torch

from sushi_amd import exl3


def test_one_token_s_logits_have_a_shape():
    lg, inds, ds, one = torch.zeros(8), torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(())
    for mask in (None, torch.ones((), dtype=torch.bool)):
        with pytest.raises(exl3.BadExl3Shape, match="device tensors"):
            exl3.moe_balance_loss(lg, inds, mask=mask)
        with pytest.raises(exl3.BadExl3Shape, match="device tensors"):
            exl3.moe_router_backward(lg, inds, dscores=ds, mask=mask)
    for bad in (dict(inds=inds[None]), dict(inds=torch.zeros((), dtype=torch.int32)), dict(mask=torch.ones(1, dtype=torch.bool))):
        with pytest.raises(exl3.BadExl3Shape, match="logits"):
            exl3.moe_balance_loss(lg, **{"inds": inds, **bad})
    with pytest.raises(exl3.BadExl3Shape, match="logits"):
        exl3.moe_balance_loss(one, one.int())


@pytest.mark.gpu
def test_one_token_is_a_row_of_one(dev):
    lg = torch.randn(32, device=dev, generator=torch.Generator(dev).manual_seed(1))
    inds, scores = exl3.moe_routing_chain(lg, 4)
    ds, dl = torch.randn(4, device=dev, generator=torch.Generator(dev).manual_seed(2)), torch.ones((), device=dev)
    a, b = exl3.moe_balance_loss(lg, inds), exl3.moe_balance_loss(lg[None], inds[None])
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    got = exl3.moe_router_backward(lg, inds, dscores=ds, weight=a.weight, dloss=dl)
    want = exl3.moe_router_backward(lg[None], inds[None], dscores=ds[None], weight=a.weight, dloss=dl)
    assert got.shape == (32,) and torch.equal(got, want[0])
    dead = torch.zeros((), dtype=torch.bool, device=dev)
    assert not exl3.moe_router_backward(lg, inds, dscores=ds, mask=dead).any()
