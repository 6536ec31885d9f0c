"""What the router training operators refuse, before anything reaches a GPU."""

import pytest
import torch

from moe_dispatch import balance_loss, route, route_backward
from moe_dispatch._extension import load_library


def balance_args(**changes):
    args = dict(logits=torch.zeros(4, 8), expert_ids=torch.zeros(4, 2, dtype=torch.int32), bias=None,
                token_mask=None)
    args.update(changes)
    return args


@pytest.mark.parametrize("changes, error, message", [
    (dict(logits=torch.zeros(4)), ValueError, "logits"),
    (dict(logits=torch.zeros(4, 8, dtype=torch.float64)), TypeError, "FP32"),
    (dict(logits=torch.zeros(4, 300)), ValueError, "experts"),
    (dict(logits=torch.zeros(4, 0)), ValueError, "experts"),
    (dict(logits=torch.zeros(8, 4).t()), ValueError, "contiguous"),
    (dict(expert_ids=torch.zeros(5, 2, dtype=torch.int32)), ValueError, "expert_ids"),
    (dict(expert_ids=torch.zeros(4, dtype=torch.int32)), ValueError, "expert_ids"),
    (dict(expert_ids=torch.zeros(4, 2)), TypeError, "int32 or int64"),
    (dict(expert_ids=torch.zeros(4, 33, dtype=torch.int32)), ValueError, "topk"),
    (dict(expert_ids=torch.zeros(4, 0, dtype=torch.int32)), ValueError, "topk"),
    (dict(bias=torch.zeros(7)), ValueError, "bias"),
    (dict(bias=torch.zeros(8, dtype=torch.float64)), ValueError, "bias"),
    (dict(bias=torch.zeros(8, requires_grad=True)), ValueError, "no gradient"),
    (dict(token_mask=torch.ones(3, dtype=torch.bool)), ValueError, "token_mask"),
    (dict(token_mask=torch.ones(4)), ValueError, "token_mask"),
    (dict(), RuntimeError, "requires CUDA"),
])
def test_balance_loss_refuses(changes, error, message):
    with pytest.raises(error, match=message):
        balance_loss(**balance_args(**changes))


def route_args(**changes):
    args = dict(x=torch.zeros(4, 16, dtype=torch.bfloat16), router_weight=torch.zeros(8, 16), bias=None, topk=2)
    args.update(changes)
    return args


@pytest.mark.parametrize("changes, error, message", [
    (dict(x=torch.zeros(4, 16)), TypeError, "BF16"),
    (dict(x=torch.zeros(4, 24, dtype=torch.bfloat16)), ValueError, "expected x"),
    (dict(x=torch.zeros(4, 12, dtype=torch.bfloat16), router_weight=torch.zeros(8, 12)), ValueError, "multiple of 8"),
    (dict(x=torch.zeros(16, 4, dtype=torch.bfloat16).t()), ValueError, "contiguous"),
    (dict(router_weight=torch.zeros(300, 16)), ValueError, "experts"),
    (dict(router_weight=torch.zeros(8, 16, dtype=torch.bfloat16)), TypeError, "FP32"),
    (dict(bias=torch.zeros(8, requires_grad=True)), ValueError, "no gradient"),
    (dict(topk=9), ValueError, "topk"),
    (dict(topk=0), ValueError, "topk"),
    (dict(topk=2.0), ValueError, "topk"),
    (dict(), RuntimeError, "requires CUDA"),
])
def test_route_refuses(changes, error, message):
    args = route_args(**changes)
    with pytest.raises(error, match=message):
        route(args.pop("x"), args.pop("router_weight"), **args)


def backward_args(**changes):
    args = dict(x=torch.zeros(4, 16, dtype=torch.bfloat16), router_weight=torch.zeros(8, 16),
                expert_ids=torch.zeros(4, 2, dtype=torch.int32), weights=torch.zeros(4, 2),
                grad_weights=torch.zeros(4, 2), grad_logits=torch.zeros(4, 8))
    args.update(changes)
    return args


@pytest.mark.parametrize("changes, error, message", [
    (dict(weights=torch.zeros(4, 3)), ValueError, "weights"),
    (dict(weights=torch.zeros(4, 2, dtype=torch.bfloat16)), ValueError, "weights"),
    (dict(grad_weights=torch.zeros(2, 4).t()), ValueError, "contiguous"),
    (dict(grad_logits=torch.zeros(4, 9)), ValueError, "grad_logits"),
    (dict(grad_logits=torch.zeros(8, 4).t()), ValueError, "contiguous"),
    (dict(expert_ids=torch.zeros(3, 2, dtype=torch.int32)), ValueError, "expert_ids"),
    (dict(), RuntimeError, "requires CUDA"),
])
def test_route_backward_refuses(changes, error, message):
    with pytest.raises(error, match=message):
        route_backward(**backward_args(**changes))


@pytest.mark.parametrize("call, message", [
    (lambda lib: lib.moe_balance_loss(None, 9, None, None, None, 1.0, None, None, None, 4, 8, 2, None, 0, None), "FP32"),
    (lambda lib: lib.moe_balance_loss(None, 0, None, None, None, 1.0, None, None, None, 4, 300, 2, None, 0, None), "experts"),
    (lambda lib: lib.moe_balance_loss(None, 0, None, None, None, 1.0, None, None, None, 4, 8, 33, None, 0, None), "topk"),
    (lambda lib: lib.moe_balance_loss(None, 0, None, None, None, 1.0, None, None, None, 2**31, 8, 2, None, 0, None), "int32"),
    (lambda lib: lib.moe_balance_loss(None, 0, None, None, None, 1.0, None, None, None, 4, 8, 2, None, 0, None), "null"),
    (lambda lib: lib.moe_balance_loss(None, 0, None, None, None, 1.0, 64, 64, 64, 0, 8, 2, None, 0, None), "scratch"),
    (lambda lib: lib.moe_balance_loss_backward(None, 0, None, None, None, None, None, 1.0, None, 0, 8, 2, None), "null"),
    (lambda lib: lib.moe_route_backward(None, None, None, None, None, None, 16, None, 4, 12, 8, 2, None, 0, None), "hidden"),
    (lambda lib: lib.moe_route_backward(None, None, None, None, None, None, 16, None, 4, 16, 0, 2, None, 0, None), "experts"),
    (lambda lib: lib.moe_route_backward(None, None, None, None, None, None, 16, None, 4, 16, 8, 0, None, 0, None), "topk"),
    (lambda lib: lib.moe_route_backward(None, None, None, None, None, None, 16, None, 2**30, 16, 8, 2, None, 0, None), "int32"),
    (lambda lib: lib.moe_route_backward(None, None, None, None, None, None, 16, None, 4, 16, 8, 2, None, 0, None), "null"),
    (lambda lib: lib.moe_route_backward(16, 16, 16, 16, 16, None, 24, None, 4, 16, 8, 2, None, 0, None), "aligned"),
])
def test_library_refuses(call, message):
    lib = load_library()
    assert call(lib) == 1
    assert message in lib.moe_last_error().decode()


def test_scratch_queries_refuse_bad_shapes():
    lib = load_library()
    assert lib.moe_balance_loss_scratch_bytes(0) == -1 and lib.moe_balance_loss_scratch_bytes(257) == -1
    assert lib.moe_balance_loss_scratch_bytes(8) > 0
    assert lib.moe_route_backward_scratch_bytes(4, 12, 8, 1, 1) == -1
    assert lib.moe_route_backward_scratch_bytes(-1, 16, 8, 1, 1) == -1
