"""Workloads of the block's router training operators and of its adapters.

Three operators: the load-balance loss of a router with its per-expert counts
and gradient, the router's backward pass, and low-rank adapters of many
requests added to the experts' grouped projections.  ``run`` computes one pass
in elementary torch operations, or (``own``) through the framework's calls.
"""

import functools
import math
import sys
from pathlib import Path

import torch

own = False

# Sizes: the framework's block workloads small (T 128, H 512, I 1024, E 8, top-2), mixtral (4096, 4096, 14336, 8,
# top-2), fine_grained (16384, 2048, 1408, 64, top-6) and expert_parallel (32768, 7168, 2048, 256, top-8).


def listed():
    return [
        # the small block's router: launch latency decides
        dict(name="balance_small", op="balance", tokens=128, experts=8, topk=2, dtype="float32", masked=False, bias=False),
        # a bf16 router with an odd number of experts over a padded batch
        dict(name="balance_ragged_bf16", op="balance", tokens=5003, experts=60, topk=4, dtype="bfloat16", masked=True, bias=False),
        # 256 experts, a padded batch, a routing bias: the largest logits
        dict(name="balance_e256", op="balance", tokens=32768, experts=256, topk=8, dtype="float32", masked=True, bias=True),
        # backward passes of the four blocks' routers
        dict(name="router_small", op="router", tokens=128, hidden=512, experts=8, topk=2, balance=True),
        dict(name="router_mixtral", op="router", tokens=4096, hidden=4096, experts=8, topk=2, balance=True),
        dict(name="router_fine_grained", op="router", tokens=16384, hidden=2048, experts=64, topk=6, balance=False),
        dict(name="router_e256", op="router", tokens=32768, hidden=7168, experts=256, topk=8, balance=True),
        # one token being decoded: two expert rows of the gate/up projection
        dict(name="adapter_one_token", op="adapter", tokens=1, k=4096, n=14336, experts=8, topk=2, adapters=16, rank=16,
             requests=1, swiglu=True, scaled=True),
        # 67 requests decoded together, each token with an adapter of its own choice, down projection
        dict(name="adapter_decode", op="adapter", tokens=67, k=14336, n=4096, experts=8, topk=2, adapters=64, rank=16,
             requests=67, swiglu=False, scaled=True),
        # prefill of 9 requests, gate/up
        dict(name="adapter_prefill", op="adapter", tokens=4096, k=4096, n=14336, experts=8, topk=2, adapters=8, rank=16,
             requests=9, swiglu=True, scaled=True),
        # prefill over 64 small experts with 32 adapters: many short runs of rows
        dict(name="adapter_fine_grained", op="adapter", tokens=16384, k=2048, n=1408, experts=64, topk=6, adapters=32, rank=32,
             requests=48, swiglu=True, scaled=False),
        # one projection shared by every row (no experts), rows of the requests interleaved
        dict(name="adapter_interleaved", op="adapter", tokens=5003, k=2048, n=2048, experts=1, topk=1, adapters=24, rank=64,
             requests=5003, swiglu=False, scaled=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["balance", "router", "adapter", "adapter"])
    if op == "balance":
        experts = _log_int(rng, 2, 256)
        return dict(op=op, tokens=_log_int(rng, 1, 32768), experts=experts, topk=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]), masked=rng.random() < 0.5,
                    bias=rng.random() < 0.5)
    if op == "router":
        experts = _log_int(rng, 2, 256)
        return dict(op=op, tokens=_log_int(rng, 1, 32768), hidden=8 * _log_int(rng, 8, 896), experts=experts,
                    topk=rng.randint(1, min(8, experts)), balance=rng.random() < 0.7)
    experts = rng.choice([1, 8, _log_int(rng, 2, 64)])
    topk = rng.randint(1, min(6, experts))
    swiglu = rng.random() < 0.5
    k, n = 8 * _log_int(rng, 8, 1024), 8 * _log_int(rng, 8, 1024)
    adapters, rank = _log_int(rng, 1, 64), 8 * rng.choice([1, 2, 2, 3, 4, 8, 16])
    while adapters * experts * rank * (k + 2 * n) > 300e6:
        adapters = max(1, adapters // 2)
        experts = max(topk, experts // 2)
    most = max(64, min(16384, int(250e6 / (topk * (k + 4 * n)))))
    tokens = _log_int(rng, 1, most)
    requests = tokens if rng.random() < 0.4 else rng.randint(1, min(64, tokens))
    return dict(op=op, tokens=tokens, k=k, n=n, experts=experts, topk=topk, adapters=adapters, rank=rank, requests=requests,
                swiglu=swiglu, scaled=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    out = torch.randn(*shape, device="cuda", generator=g, dtype=dtype)
    return out if scale == 1.0 else out.mul_(scale)


def _selection(scores, topk):
    top, ids = torch.topk(scores, topk, dim=-1)
    return ids.to(torch.int32).contiguous(), torch.softmax(top, dim=-1).contiguous()


def _prepare_balance(case, g):
    dtype = getattr(torch, case["dtype"])
    t, e = case["tokens"], case["experts"]
    logits = _randn(g, t, e).to(dtype)
    # popularity falls with the expert's rank, as it does before a router is balanced
    bias = -0.5 * torch.log(torch.randperm(e, device="cuda", generator=g).float() + 1.0) if case["bias"] else None
    ids, _ = _selection(logits.float() + (bias if bias is not None else 0.0), case["topk"])
    # a padded batch: the tokens behind each sequence's end count for nothing
    mask = None
    if case["masked"]:
        length = max(1, min(t, 512))
        ends = torch.randint(0, length + 1, ((t + length - 1) // length,), device="cuda", generator=g)
        at = torch.arange(t, device="cuda")
        mask = (at % length) < ends[at // length]
    return dict(logits=logits.requires_grad_(True), ids=ids, bias=bias, mask=mask, coefficient=0.01)


def _prepare_router(case, g):
    t, h, e, k = case["tokens"], case["hidden"], case["experts"], case["topk"]
    x = _randn(g, t, h, dtype=torch.bfloat16)
    weight = _randn(g, e, h, scale=1.0 / math.sqrt(h))
    ids, weights = _selection(_randn(g, t, e), k)
    # what comes back through the combine, and through a balance loss on the logits
    grad_weights = _randn(g, t, k, scale=0.1)
    grad_logits = _randn(g, t, e, scale=0.01 / e) if case["balance"] else None
    return dict(x=x, weight=weight, ids=ids, weights=weights, grad_weights=grad_weights, grad_logits=grad_logits)


def _prepare_adapter(case, g):
    t, k, experts, topk = case["tokens"], case["k"], case["experts"], case["topk"]
    n = case["n"] * (2 if case["swiglu"] else 1)
    adapters, rank = case["adapters"], case["rank"]
    # tokens of one request are neighbours and share an adapter; -1: a request without one
    of_request = torch.randint(-1, adapters, (case["requests"],), device="cuda", generator=g)
    cuts = torch.sort(torch.randperm(t, device="cuda", generator=g)[: case["requests"] - 1]).values
    request = torch.searchsorted(cuts, torch.arange(t, device="cuda"), right=True)
    token_adapter = of_request[request]
    if experts == 1:
        rows, used, offsets = t, t, None
        row_adapters = token_adapter.to(torch.int32).contiguous()
    else:  # the block's packed rows: by expert, each span a multiple of 8, token order within
        align = 8
        ids = torch.topk(torch.rand(t, experts, device="cuda", generator=g), topk, dim=-1).indices.flatten()
        order = torch.sort(ids, stable=True).indices
        counts = (ids[:, None] == torch.arange(experts, device="cuda")).sum(0)
        spans = (counts + align - 1) // align * align
        offsets = torch.cat([spans.new_zeros(1), spans.cumsum(0)])
        starts = counts.cumsum(0) - counts
        place = torch.arange(t * topk, device="cuda") - starts[ids[order]] + offsets[ids[order]]
        rows = (t * topk + experts * (align - 1) + 1 + align - 1) // align * align
        row_adapters = torch.full((rows,), -1, device="cuda", dtype=torch.int32)
        row_adapters[place] = token_adapter[order // topk].to(torch.int32)
        used = int(offsets[-1])
        offsets = offsets.to(torch.int32)
    return dict(
        base=_randn(g, rows, n, dtype=torch.bfloat16),
        x=_randn(g, rows, k, dtype=torch.bfloat16),
        a=_randn(g, adapters, experts, rank, k, dtype=torch.bfloat16, scale=1.0 / math.sqrt(k)),
        b=_randn(g, adapters, experts, n, rank, dtype=torch.bfloat16, scale=0.25 / math.sqrt(rank)),
        scale=(torch.rand(adapters, device="cuda", generator=g) + 0.5) if case["scaled"] else None,
        row_adapters=row_adapters, offsets=offsets, used=used, swiglu=case["swiglu"],
        out=torch.zeros(rows, case["n"], device="cuda", dtype=torch.bfloat16))


_PREPARE = dict(balance=_prepare_balance, router=_prepare_router, adapter=_prepare_adapter)


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, _generator(seed))
    state["op"] = case["op"]
    return state


# ------------------------------------------------------------- plain forms


def _plain_balance(s):
    with torch.no_grad():
        z = s["logits"].float()
        if s["bias"] is not None:
            z = z + s["bias"]
        t, e = z.shape
        keep = s["mask"] if s["mask"] is not None else torch.ones(t, dtype=torch.bool, device=z.device)
        top = z.max(-1, keepdim=True).values
        p = torch.exp(z - top.masked_fill(top == -math.inf, 0.0))
        total = p.sum(-1, keepdim=True)
        p = p / total.masked_fill(total == 0, 1.0)
        p = torch.where(keep[:, None], p, 0.0)
        valid = keep.sum().float().clamp_min(1.0)
        place = torch.where(keep[:, None], s["ids"], e).flatten()
        counts = torch.zeros(e + 1, dtype=torch.int32, device=z.device)
        counts = counts.index_add_(0, place, torch.ones_like(place))[:e]
        f = counts.float() / (valid * s["ids"].shape[1])
        loss = s["coefficient"] * e * (f * (p.sum(0) / valid)).sum()
        grad = (s["coefficient"] * e / valid) * p * (f - (p * f).sum(-1, keepdim=True))
        return loss, counts, grad.to(s["logits"].dtype)


def _plain_router(s):
    w, gw = s["weights"], s["grad_weights"]
    ds = w * (gw - (w * gw).sum(-1, keepdim=True))
    d = s["grad_logits"].clone() if s["grad_logits"] is not None else torch.zeros(
        w.shape[0], s["weight"].shape[0], device=w.device)
    d.scatter_add_(1, s["ids"].long(), ds)
    return (d @ s["weight"]).to(torch.bfloat16), d.t() @ s["x"].float()


def _plain_adapter(s):
    rows, experts = s["x"].shape[0], s["a"].shape[1]
    at = torch.arange(rows, device="cuda")
    expert = torch.zeros_like(at) if s["offsets"] is None else torch.searchsorted(s["offsets"][1:].long(), at, right=True)
    pair = torch.where((s["row_adapters"] >= 0) & (expert < experts), s["row_adapters"].long() * experts + expert, -1)
    y = s["base"].float()
    order = torch.sort(pair, stable=True).indices
    found, sizes = torch.unique_consecutive(pair[order], return_counts=True)
    first = 0
    for group, size in zip(found.tolist(), sizes.tolist()):
        if group >= 0:
            r = order[first:first + size]
            p, e = divmod(group, experts)
            delta = (s["x"][r].float() @ s["a"][p, e].float().t()) @ s["b"][p, e].float().t()
            y[r] += delta if s["scale"] is None else delta * s["scale"][p]
        first += size
    if s["swiglu"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    out = s["out"]
    out[:s["used"]] = y[:s["used"]].to(torch.bfloat16)
    return out


# ---------------------------------------------------------- framework calls


@functools.lru_cache(maxsize=1)
def _framework():
    path = str(Path.cwd() / "cuda-moe-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import moe_dispatch

    return moe_dispatch


def _own_balance(s, moe):
    loss, counts = moe.balance_loss(s["logits"], s["ids"], bias=s["bias"], token_mask=s["mask"],
                                    coefficient=s["coefficient"])
    (grad,) = torch.autograd.grad(loss, s["logits"])
    return loss.detach(), counts, grad


def _own_router(s, moe):
    return moe.route_backward(s["x"], s["weight"], s["ids"], s["weights"], s["grad_weights"], s["grad_logits"])


def _own_adapter(s, moe):
    call = moe.adapter_swiglu if s["swiglu"] else moe.adapter_add
    return call(s["base"], s["x"], s["a"], s["b"], s["row_adapters"], offsets=s["offsets"], scale=s["scale"], out=s["out"])


_PLAIN = dict(balance=_plain_balance, router=_plain_router, adapter=_plain_adapter)
_OWN = dict(balance=_own_balance, router=_own_router, adapter=_own_adapter)


def run(state):
    if own:
        return _OWN[state["op"]](state, _framework())
    return _PLAIN[state["op"]](state)


# ---------------------------------------------------------- work and values


def work(case):
    if case["op"] == "balance":
        t, e = case["tokens"], case["experts"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * t * e * size + 4 * t * case["topk"] + (t if case["masked"] else 0) + 8 * e, "flops": 12 * t * e}
    if case["op"] == "router":
        t, h, e, k = case["tokens"], case["hidden"], case["experts"], case["topk"]
        return {"bytes": 4 * t * h + 8 * e * h + 12 * t * k + (4 * t * e if case["balance"] else 0), "flops": 4 * t * e * h}
    rows, experts, rank = case["tokens"] * case["topk"], case["experts"], case["rank"]
    n = case["n"] * (2 if case["swiglu"] else 1)
    pairs = experts * case["adapters"]
    # (adapter, expert) pairs that some row has, in expectation over requests and routing
    present_adapters = case["adapters"] * (1 - (1 - 1 / (case["adapters"] + 1)) ** case["requests"])
    served = rows * case["adapters"] / (case["adapters"] + 1)
    present = max(1.0, present_adapters * experts)
    present = min(pairs, present * (1 - (1 - 1 / present) ** served)) if served else 0.0
    return {"bytes": 2 * served * case["k"] + 2 * rows * (n + case["n"]) + 2 * present * rank * (case["k"] + n) + 4 * rows,
            "flops": 2 * served * rank * (case["k"] + n)}


def exact(case, seed):
    """What run() returns, from the definitions in float64."""
    s = prepare(case, seed)
    if case["op"] == "balance":
        t, e = case["tokens"], case["experts"]
        with torch.no_grad():
            z = s["logits"].double() + (s["bias"].double() if s["bias"] is not None else 0.0)
            if s["mask"] is not None:
                kept, ids = z[s["mask"]], s["ids"][s["mask"]].long()
            else:
                kept, ids = z, s["ids"].long()
            v = kept.shape[0]
            counts = torch.stack([(ids == j).sum() for j in range(e)]).to(torch.int32)
            grad = torch.zeros(t, e, dtype=torch.float64, device="cuda")
            if v == 0:
                return torch.zeros((), dtype=torch.float64), counts, grad
            p = torch.exp(kept - torch.logsumexp(kept, -1, keepdim=True))
            share = counts.double() / (v * case["topk"])
            c = s["coefficient"] * e
            loss = c * torch.dot(share, p.mean(0))
            g = c / v * (p * share - p * (p @ share)[:, None])
            if s["mask"] is not None:
                grad[s["mask"]] = g
            else:
                grad = g
            return loss, counts, grad
    if case["op"] == "router":
        t, e = case["tokens"], case["experts"]
        w, gw = s["weights"].double(), s["grad_weights"].double()
        centre = torch.einsum("tk,tk->t", w, gw)
        d = torch.zeros(t, e, dtype=torch.float64, device="cuda") if s["grad_logits"] is None else s["grad_logits"].double()
        rows = torch.arange(t, device="cuda")
        for j in range(case["topk"]):  # a token's ids are distinct
            d[rows, s["ids"][:, j].long()] += w[:, j] * (gw[:, j] - centre)
        weight, h = s["weight"].double(), case["hidden"]
        dx = torch.empty(t, h, dtype=torch.float64, device="cuda")
        dw = torch.zeros(e, h, dtype=torch.float64, device="cuda")
        for a in range(0, t, 4096):
            dx[a:a + 4096] = torch.einsum("te,eh->th", d[a:a + 4096], weight)
            dw += torch.einsum("te,th->eh", d[a:a + 4096], s["x"][a:a + 4096].double())
        return dx, dw
    experts, n = case["experts"], case["n"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    bounds = [0, s["x"].shape[0]] if s["offsets"] is None else s["offsets"].tolist()
    owner = s["row_adapters"].cpu()
    for e in range(experts):
        low, high = bounds[e], bounds[e + 1]
        if high == low:
            continue
        y = s["base"][low:high].double()
        here = owner[low:high]
        for p in here.unique().tolist():
            if p < 0:
                continue
            r = (here == p).nonzero().flatten().cuda()
            low_rank = torch.einsum("rk,jk->rj", s["x"][low:high][r].double(), s["a"][p, e].double())
            factor = 1.0 if s["scale"] is None else float(s["scale"][p])
            y.index_add_(0, r, factor * torch.einsum("rj,nj->rn", low_rank, s["b"][p, e].double()))
        if case["swiglu"]:
            y = torch.nn.functional.silu(y[:, :n]) * y[:, n:]
        out[low:high] = y
    return out
