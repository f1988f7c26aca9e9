"""The differentiable operators have no forward-mode derivative: a tensor with a
tangent is refused (on the host, before any device work), with or without
requires_grad, since its output would come without one."""

import pytest
import torch
from torch.autograd import forward_ad

from flow2surf_b200.losses import dcd_loss, velocity_loss
from flow2surf_b200.ops import nearest_squared_distances, offset_attention_aggregate, reduce_neighbor_messages

B, N, K, D, H, C = 1, 6, 2, 6, 8, 4


def messages(first):
    rest = [torch.ones(B, N, K, D), torch.zeros(B, N, K, dtype=torch.int32), torch.ones(H, D), torch.ones(H),
            torch.ones(C, H), torch.ones(C), torch.ones(H), torch.ones(H), torch.ones(C), torch.ones(C)]
    return reduce_neighbor_messages(first, *rest)


CALLS = {
    "offset_attention_aggregate": ((B, N, C), lambda q: offset_attention_aggregate(q, torch.ones(B, C, N), torch.ones(B, N, 3))),
    "offset_attention_aggregate value": ((B, N, 3), lambda v: offset_attention_aggregate(torch.ones(B, N, C), torch.ones(B, C, N), v)),
    "reduce_neighbor_messages": ((B, 2 * C, N), messages),
    "nearest_squared_distances": ((B, N, 3), lambda x: nearest_squared_distances(torch.ones(B, 5, 3), x)),
    "dcd_loss": ((B, N, 3), lambda x: dcd_loss(x, torch.ones(B, 5, 3), 40.0)),
    "velocity_loss": ((B, N, 3), lambda x: velocity_loss(torch.ones(B, N, 3), x)),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, grad):
    shape, call = CALLS[name]
    plain = torch.ones(shape)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(plain.clone().requires_grad_(grad), plain)
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            call(dual)
        with pytest.raises(ValueError, match="CUDA tensors"):  # an ordinary tensor gets further
            call(plain)
    with pytest.raises(ValueError, match="CUDA tensors"):
        call(plain)
