"""One gradient of the router's backward pass alone: the bits that both together give,
in every kernel, and nothing written past its end."""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]


@pytest.mark.parametrize("tokens,hidden,experts,topk", [
    (1, 8, 1, 1), (37, 72, 3, 2), (600, 520, 8, 2), (3001, 1032, 8, 8), (777, 520, 9, 3), (4000, 2056, 16, 4),
    (333, 264, 24, 4), (5000, 520, 80, 8), (50, 72, 81, 2), (3000, 1032, 130, 8), (700, 264, 256, 8)])
@pytest.mark.parametrize("with_logits", [True, False])
def test_one_gradient_alone(tokens, hidden, experts, topk, with_logits):
    from moe_dispatch import get_extension, route_backward

    g = torch.Generator().manual_seed(tokens + experts)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16).cuda()
    weight = torch.randn(experts, hidden, generator=g).cuda()
    top, ids = torch.topk(torch.randn(tokens, experts, generator=g), topk, dim=-1)
    ids, weights = ids.to(torch.int32).cuda(), torch.softmax(top, -1).cuda()
    grad_weights = torch.randn(tokens, topk, generator=g).cuda()
    grad_logits = torch.randn(tokens, experts, generator=g).cuda() if with_logits else None
    problem = (x, weight, ids, weights, grad_weights, grad_logits)
    dx, dw = route_backward(*problem)
    ext = get_extension()

    def guarded(like):  # 64 more elements behind the gradient keep their value
        buffer = torch.full((like.numel() + 64,), -77.0, dtype=like.dtype, device="cuda")
        return buffer, buffer[:like.numel()].view_as(like)

    buffer, out = guarded(dx)
    ext.route_backward_out(*problem, out, None)
    assert torch.equal(out, dx) and bool((buffer[dx.numel():] == -77.0).all())
    buffer, out = guarded(dw)
    ext.route_backward_out(*problem, None, out)
    assert torch.equal(out, dw) and bool((buffer[dw.numel():] == -77.0).all())
    assert ext.device_status() == 0


@pytest.mark.parametrize("experts", [8, 40, 200])
def test_route_of_no_tokens(experts):
    from moe_dispatch import balance_loss, route

    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    weight = torch.randn(experts, 64, device="cuda", requires_grad=True)
    ids, weights, logits = route(x, weight, topk=2)
    loss, counts = balance_loss(logits, ids)
    grad_x, grad_weight = torch.autograd.grad(weights.sum() + loss, (x, weight))
    assert ids.shape == (0, 2) and grad_x.shape == (0, 64) and loss.item() == 0.0
    assert not counts.any() and grad_weight.shape == (experts, 64) and not grad_weight.any()
