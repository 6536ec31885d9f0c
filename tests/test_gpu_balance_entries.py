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


def entries(logits, ids, **changes):
    """Arguments of the checked forward and backward entries, and what they write."""
    experts, device = logits.shape[1], logits.device
    out = dict(loss=torch.full((), -1.0, device=device),
               counts=torch.full((experts,), -1, dtype=torch.int32, device=device),
               counted=torch.full((1,), -1, dtype=torch.int32, device=device),
               grad=torch.full_like(logits, -1.0))
    args = dict(logits=logits, ids=ids, bias=None, mask=None, coefficient=2.0,
                upstream=torch.ones((), device=device), **out)
    args.update(changes)
    return args, out


def forward_entry(a):
    from moe_dispatch import get_extension

    get_extension().balance_loss_out(a["logits"], a["ids"], a["bias"], a["mask"], a["coefficient"],
                                     a["loss"], a["counts"], a["counted"])


def backward_entry(a):
    from moe_dispatch import get_extension

    get_extension().balance_loss_backward_out(a["logits"], a["bias"], a["mask"], a["counts"],
                                              a["counted"], a["upstream"], a["coefficient"],
                                              a["ids"].shape[1], a["grad"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_options", [False, True])
def test_the_checked_entries_give_the_public_calls_bits(dtype, with_options):
    from moe_dispatch import balance_loss

    logits, ids = problem()
    logits = logits.to(dtype)
    options = {}
    if with_options:
        options = dict(bias=torch.linspace(-1, 1, 24, device="cuda"),
                       mask=torch.arange(300, device="cuda") % 3 != 0)
    leaf = logits.clone().requires_grad_()
    loss, counts = balance_loss(leaf, ids, bias=options.get("bias"), token_mask=options.get("mask"),
                                coefficient=2.0)
    (grad,) = torch.autograd.grad(loss, leaf)
    args, out = entries(logits, ids, **options)
    forward_entry(args)
    backward_entry(args)
    assert torch.equal(out["loss"], loss.detach()) and torch.equal(out["counts"], counts)
    assert out["counted"].item() == (200 if with_options else 300)
    assert torch.equal(out["grad"], grad)


def refused():
    logits, ids = problem(12, 8, 2)
    return logits, ids, [
        (forward_entry, dict(logits=logits.double()), "logits"),
        (forward_entry, dict(logits=logits.t()), "logits"),
        (forward_entry, dict(ids=ids.long()), "ids"),
        (forward_entry, dict(ids=ids[:5].contiguous()), "ids"),
        (forward_entry, dict(ids=ids[:, 0].contiguous()), "ids"),
        (forward_entry, dict(ids=ids.cpu()), "balance_loss"),
        (forward_entry, dict(counts=torch.zeros(7, dtype=torch.int32, device="cuda")), "counts"),
        (forward_entry, dict(counted=torch.zeros(2, dtype=torch.int32, device="cuda")), "counted"),
        (forward_entry, dict(loss=torch.zeros(2, device="cuda")), "loss"),
        (forward_entry, dict(bias=torch.zeros(7, device="cuda")), "bias"),
        (forward_entry, dict(mask=torch.ones(12, device="cuda")), "token_mask"),
        (backward_entry, dict(grad=None), "grad"),
        (backward_entry, dict(grad=torch.zeros(12, 8, dtype=torch.float16, device="cuda")), "grad"),
        (backward_entry, dict(grad=torch.zeros(8, 12, device="cuda").t()), "balance_loss"),
        (backward_entry, dict(upstream=torch.ones(2, device="cuda")), "grad_loss"),
        (backward_entry, dict(counts=torch.zeros(8, device="cuda")), "counts"),
    ]


@pytest.mark.parametrize("case", range(16))
def test_the_checked_entries_refuse(case):
    logits, ids, cases = refused()
    assert len(cases) == 16
    call, changes, message = cases[case]
    args, _ = entries(logits, ids)
    args.update(changes)
    with pytest.raises(RuntimeError, match=message):
        call(args)
