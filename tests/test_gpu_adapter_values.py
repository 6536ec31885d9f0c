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


@pytest.mark.parametrize("rows", ROWS)
def test_swiglu_of_gates_whose_exponential_is_near_the_largest_number(rows):
    """Every bf16 gate from -88.5 (e^88.5 is below the largest fp32 number) to 90.

    Rows with an adapter whose product is zero; 2^-8 of the value for the rounding to
    bf16 and (|g| + 8) 2^-23 for g log2 e rounded once, the exponential, the
    reciprocal and the products."""
    from moe_dispatch import adapter_swiglu

    patterns = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16)
    gates = patterns.view(BF16)
    gates = gates[(gates.float() >= -88.5) & (gates.float() <= 90.0)]
    half = (gates.numel() + rows * 8 - 1) // (rows * 8) * 8
    gate = torch.zeros(rows * half, dtype=BF16)
    gate[:gates.numel()] = gates
    gate = gate.view(rows, half)
    for up in (1.0, -3.0, 2.0**20):
        projection = torch.cat([gate, torch.full_like(gate, up)], 1).cuda()
        x = torch.ones(rows, 8, dtype=BF16, device="cuda")
        a = torch.ones(1, 1, 8, 8, dtype=BF16, device="cuda")
        b = torch.zeros(1, 1, 2 * half, 8, dtype=BF16, device="cuda")
        out = adapter_swiglu(projection, x, a, b, torch.zeros(rows, dtype=torch.int32, device="cuda"))
        g = gate.double()
        exact = g / (1.0 + torch.exp(-g)) * up
        # half a step of bf16 is 2^-134 at least
        bound = (2.0**-8 + 1.01 * (g.abs() + 8) * 2.0**-23) * exact.abs() + 2.0**-134
        error = (out.double().cpu() - exact).abs()
        assert bool((error <= bound).all()), (up, float((error / bound).max()))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("rank", [8, 16, 24, 64, 128])
def test_the_inner_product_enters_in_fp32(rows, rank):
    """s = (1 + 2^-9 + 2^-18, 1 + 2^-9, 0, ...) and B = (1, -1, ...): 2^-18 is left.

    Every product and partial sum is a multiple of 2^-18 below 4 (times a power of
    two that the row and the column share), so nothing is ever rounded."""
    from moe_dispatch import adapter_add, adapter_swiglu

    k, n = 136, 80
    row = torch.exp2((torch.arange(rows) % 3).float())
    column = torch.exp2((torch.arange(n) % 4).float())
    x = torch.zeros(rows, k)
    x[:, 1], x[:, 50], x[:, 135] = row, 2.0**-9 * row, 2.0**-18 * row
    a = torch.zeros(1, 1, rank, k)
    a[0, 0, 0], a[0, 0, 1, :135] = 1.0, 1.0
    b = torch.zeros(1, 1, n, rank)
    b[0, 0, :, 0], b[0, 0, :, 1] = column, -column
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    x, a, b = (t.to(BF16).cuda() for t in (x, a, b))
    want = 2.0**-18 * row[:, None] * column
    out = adapter_add(torch.zeros(rows, n, dtype=BF16, device="cuda"), x, a, b, ids)
    assert torch.equal(out.float().cpu(), want)

    base = torch.zeros(rows, 2 * n, dtype=BF16, device="cuda")
    base[:, :n] = 4.0
    b = torch.cat([torch.zeros_like(b), b], 2)
    out = adapter_swiglu(base, x, a, b, ids)
    exact = 4.0 / (1.0 + torch.exp(torch.tensor(-4.0, dtype=torch.float64))) * want.double()
    assert bool(((out.double().cpu() - exact).abs() <= (2.0**-8 + 12 * 2.0**-23) * exact).all())


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 72, 128])
def test_infinite_and_very_large_inner_products(rows, rank):
    """An infinite s gives the infinity of the formula (a, b, up > 0: no inf - inf, no 0 inf), and an s
    past the largest bf16 value is still a number."""
    from moe_dispatch import adapter_add, adapter_swiglu

    g = torch.Generator().manual_seed(rank)
    k, n = 264, 72
    x = torch.rand(rows, k, generator=g)
    x[7, 5] = float("inf")
    x[20, 5] = -float("inf")
    x[33] = 0.0
    x[33, 0], x[33, 1] = 2.0**127, 2.0**127
    a = torch.rand(2, 1, rank, k, generator=g) + 0.5
    a[:, :, :, 0], a[:, :, :, 1] = 0.0, 0.0
    a[:, :, 0, 0], a[:, :, 0, 1] = 1.0, 1.0 - 2.0**-8  # s[33] = (2^127 (2 - 2^-8), 0, ...): a tie, up to infinity in bf16
    b = torch.rand(2, 1, n, rank, generator=g) + 0.5
    b[:, :, :, 0] = 2.0**-20
    ids = (torch.arange(rows) % 2).to(torch.int32)
    x, a, b = (t.to(BF16).cuda() for t in (x, a, b))
    out = adapter_add(torch.ones(rows, n, dtype=BF16, device="cuda"), x, a, b, ids.cuda()).cpu()
    assert bool((out[7] == float("inf")).all()) and bool((out[20] == -float("inf")).all())
    assert bool((out[33] == 2.0**108).all())  # 2^107 (2 - 2^-8), rounded to bf16
    rest = torch.ones(rows, dtype=torch.bool)
    rest[[7, 20]] = False
    assert bool(torch.isfinite(out[rest]).all())

    base = torch.ones(rows, 2 * n, dtype=BF16, device="cuda")
    b = torch.cat([b, torch.full_like(b, 2.0**-20)], 2)
    out = adapter_swiglu(base, x, a, b, ids.cuda()).cpu()
    rest[33] = False                             # its gate times its up is past the largest number
    assert bool((out[7] == float("inf")).all()) and bool(torch.isfinite(out[rest]).all())


@pytest.mark.parametrize("rows", ROWS + [12000])
def test_small_terms_of_a_long_inner_product_are_not_lost(rows):
    """s = 1 + (K - 1) 7 2^-30, base = -1, b = 1: what is left are the small terms, 7/8 of 2^-23 per 16.

    A sum that stands at 1 may lose the terms of 256 elements (16 cuts of at most 2^-23); then
    half a step (2^-24) for each of at most K / 256 + 8 additions, and three cuts of 2^-23 for the
    parts of s in the second product."""
    from moe_dispatch import adapter_add

    k, rank = 14336, 16
    a = torch.zeros(1, 1, rank, k)
    a[0, 0, 0] = 7 * 2.0**-30
    a[0, 0, 0, 0] = 1.0
    b = torch.zeros(1, 1, 8, rank)
    b[..., 0] = 1.0
    x = torch.ones(rows, k, dtype=BF16, device="cuda")
    base = torch.full((rows, 8), -1.0, dtype=BF16, device="cuda")
    out = adapter_add(base, x, a.to(BF16).cuda(), b.to(BF16).cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda"))
    exact = (k - 1) * 7 * 2.0**-30
    bound = 19 * 2.0**-23 + (k // 256 + 8) * 2.0**-24 + 2.0**-8 * exact
    error = float((out.double() - exact).abs().max())
    assert error <= bound, error / bound


@pytest.mark.parametrize("rows", [5500, 6500, 7300, 8190, 8192, 8193])
def test_every_size_of_the_sorting_cluster(rows):
    """6 to 8 chunks of rows in one cluster, the most adapters, and the first size past it: x A^T B^T of
    small whole numbers, so every sum is exact."""
    from moe_dispatch import adapter_add

    g = torch.Generator().manual_seed(rows)
    adapters, k, n, rank = 512, 16, 8, 8
    x = torch.randint(-2, 3, (rows, k), generator=g).float()
    a = torch.randint(-1, 2, (adapters, 1, rank, k), generator=g).float()
    b = torch.randint(-1, 2, (adapters, 1, n, rank), generator=g).float()
    base = torch.randint(-4, 5, (rows, n), generator=g).float()
    ids = torch.randint(-1, adapters, (rows,), generator=g)
    s = torch.einsum("rk,rjk->rj", x, a[ids.clamp_min(0), 0])
    want = base + (ids >= 0)[:, None] * torch.einsum("rj,rnj->rn", s, b[ids.clamp_min(0), 0])
    out = adapter_add(*(t.to(BF16).cuda() for t in (base, x, a, b)), ids.cuda())
    assert torch.equal(out.cpu(), want.to(BF16))  # integers below 2^24, rounded once
