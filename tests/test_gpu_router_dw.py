"""dW of the router's backward pass over many tokens.

The tensor cores cut a sum off below the accumulator's last bit (2^-23 of it at
most), so an accumulator may only take a bounded number of products: 256 tokens, 16
MMAs of each part of d.  What follows are fp32 additions, half a step (2^-24) each.
"""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]


@pytest.mark.parametrize("tokens,hidden,experts", [
    (4096, 65536, 3), (4096, 65536, 8), (4096, 65536, 16), (2048, 18944, 17), (2048, 18944, 40),
    (2048, 18944, 80), (2048, 18944, 96)])
def test_small_terms_of_many_tokens_are_not_lost(tokens, hidden, experts):
    """x = 1, d = 2^k at the first token and 7/8 of 2^(k-23) per 16 tokens after it: an accumulator that
    stands at 2^k loses all of them.

    The first accumulator loses its 15 later MMAs (one cut each, and one more in its first); the
    others are exact.  Additions in fp32: one per 256 tokens, and at most 40 over ranges of tokens."""
    from moe_dispatch import route_backward

    small = 7 * 2.0**-30
    scale = torch.exp2((torch.arange(experts) % 5 - 2).double())
    d = (small * scale).repeat(tokens, 1)
    d[0] = scale
    x = torch.ones(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    zeros = torch.zeros(tokens, 1, device="cuda")
    _, dw = route_backward(x, torch.zeros(experts, hidden, device="cuda"), zeros.to(torch.int32), zeros + 1,
                           zeros, d.float().cuda())
    exact = d.sum(0)
    bound = (16 * 2.0**-23 + (tokens // 256 + 40) * 2.0**-24) * exact
    error = (dw.double().cpu() - exact[:, None]).abs().amax(1)
    assert bool((error <= bound).all()), float((error / bound).max())
