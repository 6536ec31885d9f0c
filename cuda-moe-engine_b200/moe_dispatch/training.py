"""Differentiable router: routing weights, load-balance loss, and their gradients.

The reference's block is forward-only; these operators are what fine-tuning its
router needs beside it.  They take the block's own tensors (bf16 tokens, fp32
router weight and logits, int32 expert ids) and run kernels from libmoe_b200.so.

Every call launches on the current stream of its tensors' device, allocates its
scratch from torch's caching allocator for itself alone and never synchronises,
so calls on several streams may overlap and each can be captured in a CUDA
graph.  To capture a backward pass, use ``torch.autograd.grad`` or call
``route_backward`` inside the capture, with the forward pass captured as well and
no other live autograd graph over the same leaf tensors.
"""

import torch
from torch.autograd.function import once_differentiable

from ._extension import get_extension
from .layer import MAX_EXPERTS, MAX_TOPK


def _check_ids(expert_ids, tokens, like):
    if expert_ids.ndim != 2 or expert_ids.shape[0] != tokens:
        raise ValueError("expected expert_ids[T,K] with one row per token")
    if expert_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("expert_ids must be int32 or int64")
    if not 1 <= expert_ids.shape[1] <= MAX_TOPK:
        raise ValueError(f"topk must be 1..{MAX_TOPK}")
    if expert_ids.device != like.device:
        raise ValueError("all tensors must be on the same device")


def _ids32(expert_ids):
    """Contiguous int32 ids; int64 values past int32 stay out of range."""
    if expert_ids.dtype == torch.int64:
        expert_ids = expert_ids.clamp(-1, 2**31 - 1).to(torch.int32)
    return expert_ids.contiguous()


def _check_bias(bias, experts, like):
    if bias is None:
        return
    if bias.requires_grad:
        raise ValueError("the routing bias gets no gradient; detach it")
    if bias.shape != (experts,) or bias.dtype != torch.float32 or not bias.is_contiguous():
        raise ValueError("expected contiguous fp32 bias[E]")
    if bias.device != like.device:
        raise ValueError("all tensors must be on the same device")


def _require_cuda(tensor, name):
    if not tensor.is_cuda:
        raise RuntimeError(f"{name} requires CUDA")


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, expert_ids, bias, token_mask, coefficient):
        extension = get_extension()
        experts = logits.shape[1]
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        counts = torch.empty(experts, dtype=torch.int32, device=logits.device)
        counted = torch.empty(1, dtype=torch.int32, device=logits.device)
        # kept begins with counts and counted: the caller may sum its own counts over ranks in
        # place before the backward pass
        kept = extension.launch_balance_loss(logits, expert_ids, bias, token_mask, coefficient, loss,
                                             counts, counted)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, bias, token_mask, kept)
        ctx.coefficient, ctx.topk = coefficient, expert_ids.shape[1]
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        if grad_loss is None or not ctx.needs_input_grad[0]:
            return None, None, None, None, None
        logits, bias, token_mask, kept = ctx.saved_tensors
        grad = torch.empty_like(logits)
        counts = kept.data_ptr()
        get_extension().launch_balance_loss_backward(
            logits, bias, token_mask, counts, counts + 4 * logits.shape[1], grad_loss.contiguous(),
            ctx.coefficient, ctx.topk, grad)
        return grad, None, None, None, None


def balance_loss(logits, expert_ids, *, bias=None, token_mask=None, coefficient=1.0):
    """Load-balance loss of a router and how many assignments each expert got.

    logits [T,E] (fp32, fp16 or bf16) and the expert ids [T,K] chosen from them;
    ``bias`` [E] fp32 is added to the logits first, as in routing; ``token_mask``
    [T] bool leaves out the tokens where it is False (padding): they are neither
    read nor counted and their gradient is 0.  With p = softmax(logits + bias),
    V tokens that count and f[e] the share of their V*K assignments that expert e
    got,

        loss = coefficient * E * sum_e f[e] * mean_t p[t,e]

    which is ``coefficient`` when every expert gets its share.  Returns the fp32
    scalar loss, differentiable in ``logits`` (f is a constant), and counts [E]
    int32, the caller's own: what is written there does not change the gradient.  Ids outside 0..E-1 (dropped assignments) count for nothing; without
    a token that counts the loss is 0.
    """
    if logits.ndim != 2:
        raise ValueError("expected logits[T,E]")
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError("logits must be FP32, FP16, or BF16")
    tokens, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be 1..{MAX_EXPERTS}")
    if not logits.is_contiguous():
        raise ValueError("logits must be contiguous")
    _check_ids(expert_ids, tokens, logits)
    _check_bias(bias, experts, logits)
    if token_mask is not None:
        if token_mask.shape != (tokens,) or token_mask.dtype != torch.bool:
            raise ValueError("expected bool token_mask[T]")
        if token_mask.device != logits.device:
            raise ValueError("all tensors must be on the same device")
        token_mask = token_mask.contiguous()
    _require_cuda(logits, "balance_loss")
    return _BalanceLoss.apply(logits, _ids32(expert_ids), bias, token_mask,
                              float(coefficient))


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, router_weight, bias, topk):
        tokens, experts = x.shape[0], router_weight.shape[0]
        if bias is None:
            bias = torch.zeros(experts, dtype=torch.float32, device=x.device)
        ids32 = torch.empty((tokens, topk), dtype=torch.int32, device=x.device)
        ids64 = torch.empty((tokens, topk), dtype=torch.int64, device=x.device)
        weights = torch.empty((tokens, topk), dtype=torch.float32, device=x.device)
        logits = torch.empty((tokens, experts), dtype=torch.float32, device=x.device)
        get_extension().route_out(x, router_weight, bias, logits, ids32, ids64, weights)
        ctx.mark_non_differentiable(ids32)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, router_weight, ids32, weights)
        return ids32, weights, logits

    @staticmethod
    @once_differentiable
    def backward(ctx, _, grad_weights, grad_logits):
        want_x, want_weight = ctx.needs_input_grad[:2]
        if grad_weights is None and grad_logits is None:
            return None, None, None, None
        x, router_weight, ids, weights = ctx.saved_tensors
        grad_weights = torch.zeros_like(weights) if grad_weights is None else grad_weights.contiguous()
        if grad_logits is not None:
            grad_logits = grad_logits.contiguous()
        return (*_route_backward(x, router_weight, ids, weights, grad_weights, grad_logits, want_x,
                                 want_weight), None, None)


def _route_backward(x, router_weight, ids, weights, grad_weights, grad_logits, want_x, want_weight):
    grad_x = torch.empty_like(x) if want_x else None
    grad_weight = torch.empty_like(router_weight) if want_weight else None
    get_extension().launch_route_backward(x, router_weight, ids, weights, grad_weights, grad_logits,
                                          grad_x, grad_weight)
    return grad_x, grad_weight


def _check_router(x, router_weight):
    if x.ndim != 2 or router_weight.ndim != 2 or x.shape[1] != router_weight.shape[1]:
        raise ValueError("expected x[T,H] and router_weight[E,H]")
    if x.dtype != torch.bfloat16 or router_weight.dtype != torch.float32:
        raise TypeError("x must be BF16 and router_weight FP32")
    if x.shape[1] < 8 or x.shape[1] % 8:
        raise ValueError("hidden must be a positive multiple of 8")
    if not 1 <= router_weight.shape[0] <= MAX_EXPERTS:
        raise ValueError(f"experts must be 1..{MAX_EXPERTS}")
    if x.device != router_weight.device:
        raise ValueError("all tensors must be on the same device")
    if not x.is_contiguous() or not router_weight.is_contiguous():
        raise ValueError("x and router_weight must be contiguous")


def route(x, router_weight, *, bias=None, topk=2):
    """The block's routing, differentiable in ``x`` and ``router_weight``.

    x [T,H] bf16, router_weight [E,H] fp32, bias [E] fp32 (no gradient).  Returns
    expert ids [T,K] int32, routing weights [T,K] fp32 (softmax over the selected
    scores) and logits [T,E] fp32 (without the bias): the bits of
    ``MoEBlock.route`` and ``MoEBlock.logits``.  Gradients of the weights and of
    the logits (of ``balance_loss``, say) reach x as bf16 and router_weight as
    fp32 through ``route_backward``.  The experts and the combine are forward-only:
    the gradient of the routing weights comes from the caller's own combination of
    expert outputs.
    """
    _check_router(x, router_weight)
    experts = router_weight.shape[0]
    if not isinstance(topk, int) or not 1 <= topk <= min(experts, MAX_TOPK):
        raise ValueError(f"topk must be an integer in 1..min(experts, {MAX_TOPK})")
    _check_bias(bias, experts, x)
    _require_cuda(x, "route")
    return _Route.apply(x, router_weight, bias, topk)


def route_backward(x, router_weight, expert_ids, weights, grad_weights, grad_logits=None):
    """Gradients (grad_x [T,H] bf16, grad_router_weight [E,H] fp32) of ``route``.

    ``expert_ids`` and ``weights`` [T,K] are what it returned, ``grad_weights``
    [T,K] and ``grad_logits`` [T,E] (optional) the fp32 gradients of its outputs:
    with ds = weights * (grad_weights - sum_k weights * grad_weights) and
    d = grad_logits + ds at the ids, grad_x = d router_weight (rounded once) and
    grad_router_weight = d^T x, both products to fp32 accuracy.  The results carry no
    graph: with gradients enabled, inputs that require them are refused.
    """
    _check_router(x, router_weight)
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad
            for t in (x, router_weight, weights, grad_weights, grad_logits)):
        raise ValueError("route_backward has no gradient of its own; detach inputs or use no_grad")
    tokens, experts = x.shape[0], router_weight.shape[0]
    _check_ids(expert_ids, tokens, x)
    for name, tensor, shape in (("weights", weights, expert_ids.shape),
                                ("grad_weights", grad_weights, expert_ids.shape),
                                ("grad_logits", grad_logits, (tokens, experts))):
        if tensor is None and name == "grad_logits":
            continue
        if tuple(tensor.shape) != tuple(shape) or tensor.dtype != torch.float32:
            raise ValueError(f"expected fp32 {name}{list(shape)}")
        if tensor.device != x.device:
            raise ValueError("all tensors must be on the same device")
        if not tensor.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    _require_cuda(x, "route_backward")
    with torch.no_grad():
        return _route_backward(x, router_weight, _ids32(expert_ids), weights,
                               grad_weights, grad_logits, True, True)
