"""Values of the adapters where a rounding, an infinity or a sign would show.

Rows: 60 take the form that reads A and B per row, 700 the form over tiles.
"""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]

BF16 = torch.bfloat16
ROWS = [60, 700]


def bits(t):
    return t.view(torch.int16)


@pytest.mark.parametrize("rows", ROWS)
def test_rows_without_an_adapter_keep_the_sign_of_zero(rows):
    from moe_dispatch import adapter_add, adapter_swiglu, get_extension

    g = torch.Generator().manual_seed(rows)
    base = torch.randn(rows, 144, generator=g).to(BF16)
    base[:, ::3] = -0.0
    base[:, 1::3] = 0.0
    base[:, 80::2] = -0.0
    base = base.cuda()
    x = torch.randn(rows, 64, generator=g).to(BF16).cuda()
    a = torch.randn(3, 1, 16, 64, generator=g).to(BF16).cuda()
    b = torch.randn(3, 1, 144, 16, generator=g).to(BF16).cuda()
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(bits(adapter_add(base, x, a, b, ids)), bits(base))
    want = torch.empty(rows, 72, dtype=BF16, device="cuda")
    get_extension().swiglu_out(base, torch.tensor([rows], dtype=torch.int32, device="cuda"), want)
    assert torch.equal(bits(adapter_swiglu(base, x, a, b, ids)), bits(want))
