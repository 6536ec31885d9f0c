"""dx of the router's backward pass is an fp32 product, rounded once.

d and W are three bf16 parts each (every part within half a step, 2^-8, of the
rest), so a value is its parts' sum to 2^-24.  Six of the nine products are made;
those left out (mid lo, lo mid, lo lo) are at most (2 + 2^-8) 2^-24 |d W|.  With the
two splits that is below 2.1 * 2^-23 |d W|.  Every MMA cuts its sum off at most
2^-23 below the running sum, which never exceeds (1 + 2^-6) sum |d W|; an MMA whose
products are all zero cuts nothing.  So with d not zero in `blocks` groups of 16
experts dx is within (6 blocks + 4) 2^-23 sum |d W| before it is rounded to bf16
(2^-8 of the value).
"""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]


@pytest.mark.parametrize("experts", [2, 8, 9, 16, 17, 24, 64, 65, 100, 256])
@pytest.mark.parametrize("apart", [False, True], ids=["neighbours", "apart"])
@pytest.mark.parametrize("tokens,hidden", [(40, 1032), (300, 264)])
def test_products_that_cancel_keep_fp32_accuracy(experts, apart, tokens, hidden):
    """d = (s, -s v), W = (v w rounded to fp32, w): dx is what that rounding leaves."""
    from moe_dispatch import route_backward

    g = torch.Generator().manual_seed(experts + hidden)
    other = experts - 1 if apart else 1
    v = 1.0 + 2.0**-8 - 2.0**-13              # bf16 leaves 2^-8 of it, nearly the most
    w = (1.0 + torch.rand(hidden, generator=g)) * torch.exp2(torch.randint(-3, 4, (hidden,), generator=g).float())
    w[::7] = 1.0 + 2.0**-8 - 2.0**-13
    weight = torch.zeros(experts, hidden)
    weight[0], weight[other] = v * w, w
    s = torch.exp2((torch.arange(tokens) % 5).float())
    grad_logits = torch.zeros(tokens, experts)
    grad_logits[:, 0], grad_logits[:, other] = s, -v * s
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    ids = torch.zeros(tokens, 1, dtype=torch.int32)
    nothing = torch.zeros(tokens, 1)          # of the routing weights' gradient

    dx, _ = route_backward(x.cuda(), weight.cuda(), ids.cuda(), torch.ones(tokens, 1, device="cuda"),
                           nothing.cuda(), grad_logits.cuda())
    d, wd = grad_logits.double(), weight.double()
    exact = d @ wd
    blocks = 2 if other >= 16 else 1
    bound = (6 * blocks + 4) * 2.0**-23 * (d.abs() @ wd.abs()) + 2.0**-8 * exact.abs()
    error = (dx.double().cpu() - exact).abs()
    assert bool((error <= bound).all()), float((error / bound).max())
