"""What surrounds the balance loss: its counts in the caller's hands, its checked entries."""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]


def problem(tokens=300, experts=24, topk=3):
    g = torch.Generator().manual_seed(tokens)
    logits = torch.randn(tokens, experts, generator=g).cuda()
    ids = torch.topk(logits, topk, dim=-1).indices.to(torch.int32)
    return logits, ids


def test_counts_may_be_changed_before_the_backward_pass():
    """As by a sum over ranks in place: the gradient is still that of the shares of this call."""
    from moe_dispatch import balance_loss

    logits, ids = problem()
    leaf = logits.requires_grad_()
    loss, counts = balance_loss(leaf, ids, coefficient=3.0)
    kept = counts.clone()
    (want,) = torch.autograd.grad(loss, leaf)
    for change in (lambda c: c.add_(7), lambda c: c.data.zero_()):
        loss, counts = balance_loss(leaf, ids, coefficient=3.0)
        assert torch.equal(counts, kept) and not counts.requires_grad
        change(counts)
        (grad,) = torch.autograd.grad(loss, leaf)
        assert torch.equal(grad, want)
