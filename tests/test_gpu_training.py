"""Load-balance loss, differentiable routing and its backward pass on the GPU.

Every result is compared with the definition in float64.  Tolerances follow from
the arithmetic (U = 2^-24, half a step of fp32):

* softmax: a score is rounded once when the bias is added (U |z|) and once when
  the row's maximum is subtracted (2 U max|z|); expf is good to 2 U * 2, the sum
  of at most 256 terms over 5 shuffle levels and 8 per lane to 13 U, and three
  more roundings follow.  With |z| <= 16: p is within (3 * 16 + 20) U = 68 U.
* loss: positive terms only, so p's error carries over, plus the additions over
  tokens: per lane at most tokens / (148 * 16) + 1 (<= 16 here), 16 warps, 148
  CTAs, and 16 more operations: (68 + 200) U of the loss.
* d loss / d logits = factor p (f - f.p): (68 + 68 + 20) U of factor p (f + f.p),
  plus half a step of the output type (and of fp16's subnormals, 2^-25).
* dW: d is within 2^-24 of its parts' sum and the tensor cores' fp32 additions cut
  off at most 2^-23 of the running sum: one per 16 tokens of a range (<= 4096) for
  each of the two accumulators or three column groups, then at most 16 ranges:
  (2 * min(T, 4096) / 16 + 24) * 2^-23 * sum_t |d x|.
* dx: (3 * 2^-16 + (3 * 256 / 16 + 2) * 2^-23) * sum_e |d W|, plus half a bf16 step.
* d itself: ds = w (g - sum w g), within (topk + 4) U w (|g| + sum |w g|).
"""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]

U = 2.0**-24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def balance_reference(logits, ids, bias=None, mask=None, coefficient=1.0):
    """(loss, counts, gradient, |gradient| terms) in float64 on the CPU."""
    z = logits.detach().double().cpu()
    tokens, experts = z.shape
    if bias is not None:
        z = z + bias.double().cpu()
    keep = torch.ones(tokens, dtype=torch.bool) if mask is None else mask.cpu()
    ids = ids.cpu().long()
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isinf(top) & (top < 0), 0.0, top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total == 0, 0.0, e / total)
    counts = torch.zeros(experts, dtype=torch.int64)
    for row in ids[keep].tolist():
        for i in row:
            if 0 <= i < experts:
                counts[i] += 1
    valid = int(keep.sum())
    grad = torch.zeros_like(z)
    terms = torch.zeros_like(z)
    if valid == 0:
        return 0.0, counts, grad, terms
    f = counts.double() / (valid * ids.shape[1])
    factor = coefficient * experts / valid
    loss = factor * float((f * p[keep].sum(0)).sum())
    dot = (p * f).sum(-1, keepdim=True)
    grad[keep] = (factor * p * (f - dot))[keep]
    terms[keep] = (abs(factor) * p * (f + dot))[keep]
    return loss, counts, grad, terms


def check_gradient(got, grad, terms, upstream=1.0):
    half_step = torch.finfo(got.dtype).eps / 2
    floor = 2.0**-25 if got.dtype == torch.float16 else 0.0
    error = (got.double().cpu() - upstream * grad).abs()
    bound = abs(upstream) * (156 * U * terms + half_step * grad.abs()) + floor
    assert bool((error <= bound).all()), float((error - bound).max())


def make_logits(tokens, experts, topk, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    logits = (2 * torch.randn(tokens, experts, generator=g)).clamp(-8, 8).to(dtype)
    ids = torch.topk(logits.float(), topk, dim=-1).indices.to(torch.int32)
    return logits, ids, g


@pytest.mark.parametrize("tokens,experts,topk", [
    (1, 1, 1), (1, 8, 2), (2, 3, 3), (63, 8, 2), (64, 9, 2), (65, 16, 4), (100, 17, 3), (513, 32, 8),
    (700, 33, 6), (1000, 60, 4), (255, 64, 6), (129, 65, 1), (4099, 128, 8), (300, 200, 8), (9001, 256, 8)])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d).split(".")[1])
def test_balance_loss_matches_the_definition(tokens, experts, topk, dtype):
    from moe_dispatch import balance_loss

    logits, ids, g = make_logits(tokens, experts, topk, dtype, seed=tokens + experts)
    bias = torch.randn(experts, generator=g).clamp(-4, 4) if tokens % 2 else None
    mask = torch.rand(tokens, generator=g) < 0.7 if experts % 2 else None
    leaf = logits.cuda().requires_grad_()
    loss, counts = balance_loss(leaf, ids.cuda(), bias=None if bias is None else bias.cuda(),
                                token_mask=None if mask is None else mask.cuda(), coefficient=0.3)
    (grad,) = torch.autograd.grad(loss, leaf, torch.tensor(2.5, device="cuda"))
    want, want_counts, want_grad, terms = balance_reference(logits, ids, bias, mask, 0.3)
    assert counts.dtype == torch.int32 and counts.cpu().tolist() == want_counts.tolist()
    assert loss.dtype == torch.float32 and abs(loss.item() - want) <= 268 * U * abs(want)
    assert grad.dtype == dtype
    check_gradient(grad, want_grad, terms, 2.5)


def test_balance_loss_of_rows_and_batches_that_hold_nothing():
    from moe_dispatch import balance_loss

    logits, ids, _ = make_logits(40, 12, 2, torch.float32, 3)
    logits[5] = -float("inf")                      # a row whose mask leaves no expert
    logits[6, 1:] = -float("inf")                  # one expert left
    logits[7] = torch.finfo(torch.float32).min     # the type's lowest value everywhere: uniform
    logits[8, :3] = torch.finfo(torch.float32).min
    mask = torch.ones(40, dtype=torch.bool)
    mask[9:12] = False
    logits[9] = float("nan")                       # behind the mask nothing is read
    logits[10] = float("inf")
    ids[11] = -7
    ids[12] = torch.tensor([-1, 12])               # dropped assignments
    ids[13] = 4                                    # the same id twice
    clean = logits.clone()
    clean[9:11] = 0.0
    leaf = logits.cuda().requires_grad_()
    loss, counts = balance_loss(leaf, ids.cuda(), token_mask=mask.cuda())
    (grad,) = torch.autograd.grad(loss, leaf)
    want, want_counts, want_grad, terms = balance_reference(clean, ids, None, mask)
    assert counts.cpu().tolist() == want_counts.tolist()
    assert abs(loss.item() - want) <= 268 * U * want
    check_gradient(grad, want_grad, terms)
    assert not grad[9:12].any() and not grad[5].any()

    # no token counts, and no token at all
    for rows in (40, 0):
        leaf = logits[:rows].cuda().requires_grad_()
        loss, counts = balance_loss(leaf, ids[:rows].cuda(),
                                    token_mask=torch.zeros(rows, dtype=torch.bool, device="cuda"))
        (grad,) = torch.autograd.grad(loss, leaf)
        assert loss.item() == 0.0 and not counts.any() and not grad.any() and grad.shape == (rows, 12)

    # what is not finite and counts shows
    leaf = logits.cuda().requires_grad_()
    loss, _ = balance_loss(leaf, ids.cuda())
    (grad,) = torch.autograd.grad(loss, leaf)
    assert torch.isnan(loss) and torch.isnan(grad[9]).all() and torch.isnan(grad[10]).all()
    assert torch.isfinite(grad[:9]).all()


def test_balance_loss_gradient_matches_differences():
    from moe_dispatch import balance_loss

    logits, ids, g = make_logits(37, 10, 3, torch.float32, 8)
    leaf = logits.cuda().requires_grad_()
    loss, _ = balance_loss(leaf, ids.cuda(), coefficient=7.0)
    (grad,) = torch.autograd.grad(loss, leaf)
    way = torch.randn(37, 10, generator=g, dtype=torch.float64)
    step = 1e-5
    up = balance_reference(logits.double() + step * way, ids, coefficient=7.0)[0]
    down = balance_reference(logits.double() - step * way, ids, coefficient=7.0)[0]
    slope = float((grad.double().cpu() * way).sum())
    # central differences: step^2 in truncation (third derivatives of O(loss)), float64 rounding / step
    scale = float((grad.double().cpu() * way).abs().sum())
    assert abs(slope - (up - down) / (2 * step)) <= 200 * U * scale + 1e-8


def router_problem(tokens, hidden, experts, topk, seed, with_logits=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    weight = torch.randn(experts, hidden, generator=g) / hidden**0.5
    scores = torch.randn(tokens, experts, generator=g)
    top, ids = torch.topk(scores, topk, dim=-1)
    weights = torch.softmax(top, -1)
    grad_weights = torch.randn(tokens, topk, generator=g)
    grad_logits = torch.randn(tokens, experts, generator=g) if with_logits else None
    return x, weight, ids.to(torch.int32), weights, grad_weights, grad_logits


def check_router(problem, grad_x, grad_weight):
    x, weight, ids, weights, grad_weights, grad_logits = problem
    tokens, experts = x.shape[0], weight.shape[0]
    w, g = weights.double(), grad_weights.double()
    dot = (w * g).sum(-1, keepdim=True)
    d = grad_logits.double().clone() if grad_logits is not None else torch.zeros(tokens, experts).double()
    d_error = torch.zeros(tokens, experts).double()
    d_abs = d.abs()
    for k in range(ids.shape[1]):
        i = ids[:, k].long()
        ok = ((i >= 0) & (i < experts)).double()
        at = i.clamp(0, experts - 1)[:, None]
        term = (w[:, k] * (g[:, k] - dot[:, 0]) * ok)[:, None]
        d.scatter_add_(1, at, term)
        d_abs.scatter_add_(1, at, term.abs())
        size = (w[:, k] * (g[:, k].abs() + (w * g).abs().sum(-1)) * ok)[:, None]
        d_error.scatter_add_(1, at, (ids.shape[1] + 4) * U * size)
    d_error += ids.shape[1] * U * d_abs  # its additions
    xd, wd = x.double(), weight.double()
    if grad_weight is not None:
        assert grad_weight.dtype == torch.float32
        steps = 2 * min(tokens, 4096) / 16 + 24
        bound = steps * 2.0**-23 * (d.abs().T @ xd.abs()) + d_error.T @ xd.abs()
        error = (grad_weight.double().cpu() - d.T @ xd).abs()
        assert bool((error <= bound).all()), float((error - bound).max())
    if grad_x is not None:
        assert grad_x.dtype == torch.bfloat16
        exact = d @ wd
        bound = ((3 * 2.0**-16 + 50 * 2.0**-23) * (d.abs() @ wd.abs()) + d_error @ wd.abs()
                 + 2.0**-8 * exact.abs())
        error = (grad_x.double().cpu() - exact).abs()
        assert bool((error <= bound).all()), float((error - bound).max())


ROUTER_SHAPES = [
    (1, 8, 1, 1), (1, 64, 8, 2), (3, 72, 5, 2), (31, 136, 80, 8), (33, 128, 81, 3), (128, 512, 8, 2),
    (257, 520, 96, 6), (500, 2056, 200, 8), (1000, 1032, 256, 8), (5000, 256, 64, 6), (9000, 136, 16, 32),
    (4097, 264, 33, 1), (2111, 128, 128, 4), (64, 7168, 256, 8), (700, 4104, 8, 3), (3001, 1032, 9, 9),
    (70000, 64, 4, 2), (1, 2056, 16, 16), (1000, 520, 17, 17), (129, 264, 32, 20),
    (40, 8, 20, 2), (40, 8, 100, 2), (70, 24, 40, 3), (2, 16, 256, 1), (35, 8, 8, 2)]


@pytest.mark.parametrize("shape", ROUTER_SHAPES, ids=str)
@pytest.mark.parametrize("with_logits", [True, False])
def test_route_backward_matches_the_definition(shape, with_logits):
    from moe_dispatch import route_backward

    tokens, hidden, experts, topk = shape
    topk = min(topk, experts)
    problem = router_problem(tokens, hidden, experts, topk, seed=sum(shape), with_logits=with_logits)
    grads = route_backward(*(None if t is None else t.cuda() for t in problem))
    check_router(problem, *grads)
    again = route_backward(*(None if t is None else t.cuda() for t in problem))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_route_backward_with_dropped_and_repeated_ids_and_wide_values():
    from moe_dispatch import route_backward

    x, weight, ids, weights, gw, gl = router_problem(300, 264, 24, 4, seed=5)
    ids[7] = torch.tensor([-1, 24, 3, 2**31 - 1])
    ids[8] = 5                                   # the same id four times
    gl *= torch.exp2(torch.randint(-20, 20, gl.shape, generator=torch.Generator().manual_seed(1)).float())
    weights[9], gw[10] = 0.0, 0.0
    problem = (x, weight, ids, weights, gw, gl)
    check_router(problem, *route_backward(*(t.cuda() for t in problem)))


def test_route_backward_of_no_tokens():
    from moe_dispatch import route_backward

    problem = router_problem(0, 64, 8, 2, seed=1)
    grad_x, grad_weight = route_backward(*(t.cuda() for t in problem))
    assert grad_x.shape == (0, 64) and grad_weight.shape == (8, 64) and not grad_weight.any()


def test_one_wanted_gradient_is_the_same_as_both():
    from moe_dispatch import get_extension, route_backward

    problem = [t.cuda() for t in router_problem(777, 520, 40, 4, seed=2)]
    both = route_backward(*problem)
    ext = get_extension()
    grad_x, grad_weight = torch.empty_like(both[0]), torch.empty_like(both[1])
    ext.route_backward_out(*problem, grad_x, None)
    ext.route_backward_out(*problem, None, grad_weight)
    ext.route_backward_out(*problem, None, None)
    assert torch.equal(grad_x, both[0]) and torch.equal(grad_weight, both[1])


def block_like(tokens, hidden, experts, topk, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16).cuda()
    weight = (torch.randn(experts, hidden, generator=g) / hidden**0.5).cuda()
    bias = (0.3 * torch.randn(experts, generator=g)).cuda()
    return x, weight, bias, g


@pytest.mark.parametrize("tokens,hidden,experts,topk", [(50, 64, 8, 2), (333, 256, 64, 6), (200, 128, 256, 8)])
def test_training_step_of_the_router(tokens, hidden, experts, topk):
    """route, a loss on the routing weights, the balance loss, and their gradients together."""
    from moe_dispatch import MoEBlock, MoEConfig, MoEWeights, balance_loss, route

    x, weight, bias, g = block_like(tokens, hidden, experts, topk, 11)
    x.requires_grad_()
    weight.requires_grad_()
    target = torch.randn(tokens, topk, generator=g).cuda()
    ids, weights, logits = route(x, weight, bias=bias, topk=topk)
    balance, counts = balance_loss(logits, ids, bias=bias, coefficient=50.0)
    ((weights * target).sum() + balance).backward()

    # the block's own routing, bit for bit
    block = MoEBlock(MoEConfig(hidden, 64, experts, topk), weights=MoEWeights(
        weight.detach(), torch.zeros(experts, 128, hidden, device="cuda"),
        torch.zeros(experts, hidden, 64, device="cuda")))
    block.routing_bias.copy_(bias)
    block_ids, _, block_weights = block.route(x.detach())
    assert torch.equal(ids, block_ids) and torch.equal(weights, block_weights)
    assert torch.equal(logits, block.logits(x.detach()))
    assert counts.sum().item() == tokens * topk

    # float64 on the CPU, from the logits that the kernel computed
    want_loss, _, want_grad, _ = balance_reference(logits.detach(), ids, bias, None, 50.0)
    assert abs(balance.item() - want_loss) <= 268 * U * want_loss
    problem = (x.detach().cpu(), weight.detach().cpu(), ids.cpu(), weights.detach().cpu(), target.cpu(),
               torch.autograd.grad(balance_loss(leaf := logits.detach().requires_grad_(), ids, bias=bias,
                                                coefficient=50.0)[0], leaf)[0].cpu())
    check_gradient(problem[-1], want_grad, balance_reference(logits.detach(), ids, bias, None, 50.0)[3])
    check_router(problem, x.grad, weight.grad)


def test_router_gradient_matches_differences():
    """The whole step against central differences in float64 with the selection held."""
    from moe_dispatch import balance_loss, route

    x, weight, bias, g = block_like(60, 72, 12, 3, 4)
    weight.requires_grad_()
    target = torch.randn(60, 3, generator=g)
    ids, weights, logits = route(x, weight, bias=bias, topk=3)
    loss = (weights * target.cuda()).sum() + balance_loss(logits, ids, bias=bias, coefficient=20.0)[0]
    (grad,) = torch.autograd.grad(loss, weight)
    xd, chosen = x.double().cpu(), ids.long().cpu()

    def value(w):
        scores = xd @ w.T
        picked = torch.softmax((scores + bias.double().cpu()).gather(1, chosen), -1)
        return float((picked * target.double()).sum()) + balance_reference(scores, ids, bias, None, 20.0)[0]

    way = torch.randn(12, 72, generator=g, dtype=torch.float64)
    step = 1e-5
    base = weight.detach().double().cpu()
    slope = (value(base + step * way) - value(base - step * way)) / (2 * step)
    got = float((grad.double().cpu() * way).sum())
    # fp32 logits: 72 products of O(1) summed, so weights and p are off by ~1e-5 at most, and d with them
    assert abs(got - slope) <= 1e-4 * float((grad.double().cpu() * way).abs().sum())


def test_only_the_wanted_leaves_get_gradients():
    from moe_dispatch import balance_loss, route

    x, weight, bias, _ = block_like(40, 64, 8, 2, 9)
    weight.requires_grad_()
    ids, weights, logits = route(x, weight, topk=2)
    (from_weights,) = torch.autograd.grad(weights.square().sum(), weight, retain_graph=True)
    (from_logits,) = torch.autograd.grad(logits.sum(), weight, retain_graph=True)
    (both,) = torch.autograd.grad(weights.square().sum() + logits.sum(), weight)
    size = float(from_weights.abs().max() + from_logits.abs().max())
    assert float((from_weights + from_logits - both).abs().max()) <= 1e-5 * size
    with torch.no_grad():
        assert not route(x, weight, topk=2)[1].requires_grad
        assert not balance_loss(logits, ids)[0].requires_grad


def test_captured_steps_do_not_share_scratch():
    """Forward and backward captured in two graphs, replayed at once on two streams."""
    from moe_dispatch import balance_loss, route

    def step(x, weight):
        leaf = weight.detach().requires_grad_()
        ids, weights, logits = route(x, leaf, topk=4)
        loss, counts = balance_loss(logits, ids, coefficient=3.0)
        (grad,) = torch.autograd.grad(loss + weights.square().sum(), leaf)
        return loss.detach(), counts, grad

    problems = [block_like(3000, 256, 48, 4, seed)[:2] for seed in (1, 2)]
    eager = [step(*p) for p in problems]
    graphs, outputs, streams = [], [], []
    for p in problems:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(*p)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outputs.append(step(*p))
        graphs.append(graph)
        streams.append(stream)
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outputs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outputs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_overlap_on_two_streams():
    from moe_dispatch import balance_loss, route_backward

    problems = [[t.cuda() for t in router_problem(4000, 512, 32, 4, seed=s)] for s in (1, 2)]
    want = [(*route_backward(*p), *balance_loss(p[5], p[2])) for p in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for p, stream in zip(problems, streams):
            with torch.cuda.stream(stream):
                got.append((*route_backward(*p), *balance_loss(p[5], p[2])))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_device_status_stays_clear():
    from moe_dispatch import get_extension

    assert get_extension().device_status() == 0


@pytest.mark.parametrize("experts", [1, 2, 3, 4, 8, 40])
def test_balance_loss_with_every_expert_chosen(experts):
    """topk = E: every share is 1 / E, and the gradient vanishes but for roundings."""
    from moe_dispatch import balance_loss

    logits, ids, _ = make_logits(70, experts, min(experts, 32), torch.float32, 6)
    ids = torch.arange(experts, dtype=torch.int32).repeat(70, 1)[:, :32].contiguous()
    leaf = logits.cuda().requires_grad_()
    loss, counts = balance_loss(leaf, ids.cuda())
    (grad,) = torch.autograd.grad(loss, leaf)
    want, want_counts, want_grad, terms = balance_reference(logits, ids)
    assert counts.cpu().tolist() == want_counts.tolist()
    assert abs(loss.item() - want) <= 268 * U * want
    check_gradient(grad, want_grad, terms)


@pytest.mark.parametrize("shape", [(33, 264, 40, 12), (50, 136, 100, 20), (29, 72, 130, 17), (300, 2312, 66, 3),
                                   (70, 64, 252, 32), (5, 40, 64, 8)], ids=str)
def test_route_backward_of_repeated_ids_and_unaligned_logit_gradients(shape):
    from moe_dispatch import route_backward

    tokens, hidden, experts, topk = shape
    x, weight, ids, weights, gw, gl = router_problem(tokens, hidden, experts, topk, seed=sum(shape))
    ids[1] = ids[1, 0]                           # one expert topk times
    ids[2, 1:] = -1
    ids[3, :2] = torch.tensor([experts, experts - 1])
    buffer = torch.empty(tokens * experts + 1, device="cuda")
    shifted = buffer[1:].view(tokens, experts)   # contiguous rows off every 16-byte boundary
    shifted.copy_(gl)
    aligned = [t.cuda() for t in (x, weight, ids, weights, gw, gl)]
    got = route_backward(*aligned[:5], shifted)
    check_router((x, weight, ids, weights, gw, gl), *got)
    assert all(torch.equal(a, b) for a, b in zip(got, route_backward(*aligned)))


def test_balance_loss_of_strided_ids_and_masks():
    from moe_dispatch import balance_loss

    logits, ids, _ = make_logits(500, 12, 3, torch.float32, 9)
    mask = torch.arange(500) % 3 != 1
    want = balance_loss(logits.cuda(), ids.to(torch.int32).cuda(), token_mask=mask.cuda())
    wide_ids = torch.stack([ids.long(), -ids.long()], -1).cuda()[..., 0]
    wide_mask = torch.stack([mask, ~mask], -1).cuda()[:, 0]
    assert not wide_ids.is_contiguous() and not wide_mask.is_contiguous()
    got = balance_loss(logits.cuda(), wide_ids, token_mask=wide_mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inference_mode_gives_the_same_values():
    from moe_dispatch import balance_loss, route, route_backward

    problem = [t.cuda() for t in router_problem(300, 264, 24, 4, seed=5)]
    x, weight, ids, _, _, logits = problem
    want = (*route(x, weight, topk=4), *route_backward(*problem), *balance_loss(logits, ids))
    with torch.inference_mode():
        got = (*route(x, weight, topk=4), *route_backward(*problem), *balance_loss(logits, ids))
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))


@pytest.mark.parametrize("shape", [(20000, 1032, 40, 4), (12001, 2056, 130, 4), (40000, 520, 256, 8)], ids=str)
def test_route_backward_of_several_tiles_per_sm(shape):
    from moe_dispatch import route_backward

    problem = router_problem(*shape, seed=3)
    check_router(problem, *route_backward(*(t.cuda() for t in problem)))


@pytest.mark.parametrize("experts", [12, 24, 96])
def test_route_backward_passes_32_bit_offsets(experts):
    """x and dx of more than 2^31 elements: rows around that border, and dW of all tokens."""
    from moe_dispatch import route_backward

    tokens, hidden, topk = 300_100, 7168, 2
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(tokens, hidden, device="cuda", generator=g, dtype=torch.bfloat16)
    _, weight, ids, weights, gw, gl = router_problem(tokens, 8, experts, topk, seed=4)
    weight = torch.randn(experts, hidden, generator=torch.Generator().manual_seed(8)) / hidden**0.5
    grad_x, grad_weight = route_backward(x, *(t.cuda() for t in (weight, ids, weights, gw, gl)))
    border = 2**31 // hidden
    rows = torch.tensor([0, 1, border - 1, border, border + 1, tokens - 1])
    check_router((x[rows.cuda()].cpu(), weight, ids[rows], weights[rows], gw[rows], gl[rows]), grad_x[rows.cuda()], None)
    w, u = weights.double(), gw.double()
    ds = w * (u - (w * u).sum(-1, keepdim=True))
    d = gl.double().scatter_add_(1, ids.long(), ds).cuda()
    # d itself is within (topk + 4) U of |ds| and |w| sum |w u|, and topk U of its sum
    slack = gl.double().abs().scatter_add_(1, ids.long(), ds.abs() + w * (u.abs() + (w * u).abs().sum(-1, keepdim=True))).cuda()
    want = torch.zeros(experts, hidden, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for first in range(0, tokens, 50_000):
        part = x[first:first + 50_000].double()
        want += d[first:first + 50_000].T @ part
        size += slack[first:first + 50_000].T @ part.abs()
    bound = (2 * 4096 / 16 + 24 + topk + 4) * 2.0**-23 * size
    assert bool(((grad_weight.double() - want).abs() <= bound).all())
