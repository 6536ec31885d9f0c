"""route_backward returns gradients without a graph of their own: under grad mode it
refuses what would ask for one, as the forward-only operators do."""

import pytest
import torch

from moe_dispatch import route_backward


def arguments():
    return dict(x=torch.zeros(4, 16, dtype=torch.bfloat16), router_weight=torch.zeros(8, 16),
                expert_ids=torch.zeros(4, 2, dtype=torch.int32), weights=torch.zeros(4, 2),
                grad_weights=torch.zeros(4, 2), grad_logits=torch.zeros(4, 8))


@pytest.mark.parametrize("name", ["x", "router_weight", "weights", "grad_weights", "grad_logits"])
def test_inputs_that_require_gradients_are_refused(name):
    args = arguments()
    args[name].requires_grad_()
    with pytest.raises(ValueError, match="detach"):
        route_backward(**args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):  # past the check
        route_backward(**args)
    args[name] = args[name].detach()
    with pytest.raises(RuntimeError, match="CUDA"):
        route_backward(**args)
