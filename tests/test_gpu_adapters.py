"""Low-rank adapters beside the grouped projections, on the GPU.

Every output is compared with the definition in float64.  Tolerances:

* s = x A^T: fp32 sums, cut off at most 2^-23 of the running sum per 16 products on
  the tensor cores (the plain form rounds 64 + 16 times at 2^-24, which is less):
  (K / 16 + 20) 2^-23 sum_k |x a|; used as two bf16 parts: 2^-16 |s|.
* delta = scale s B^T: (2 * 128 / 16 + 6) 2^-23 of scale sum_j |s b|; adding base:
  2^-24 |y|.
* SwiGLU: |silu'| <= 1.1, so 1.1 |u| dg + |silu(g)| du, and 8 * 2^-23 of the value
  for expf, the division and the product (expf: 2^-22).
* one rounding to bf16: 2^-8 of the value.
"""

import pytest
import torch

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA GPU required"),
]

SENTINEL = -77.0


def make_problem(spans, k, n, adapters, rank, swiglu, seed, behind=0, grouped=False, scaled=True):
    """Rows of the given expert spans and `behind` more; adapter ids in -1..adapters-1, per
    row or (grouped) in long stretches.  spans None: one expert without offsets."""
    g = torch.Generator().manual_seed(seed)
    experts = 1 if isinstance(spans, int) else len(spans)
    used = spans if isinstance(spans, int) else sum(spans)
    rows = used + behind
    width = 2 * n if swiglu else n
    ids = torch.randint(-1, adapters, (rows,), generator=g)
    if grouped:
        ids = ids[torch.arange(rows) // 37]
    offsets = None if isinstance(spans, int) else torch.tensor([0] + list(torch.tensor(spans).cumsum(0)))
    return dict(
        base=torch.randn(rows, width, generator=g).bfloat16(),
        x=torch.randn(rows, k, generator=g).bfloat16(),
        a=(torch.randn(adapters, experts, rank, k, generator=g) / k**0.5).bfloat16(),
        b=(torch.randn(adapters, experts, width, rank, generator=g) / rank**0.5).bfloat16(),
        row_adapters=ids.to(torch.int32),
        offsets=None if offsets is None else offsets.to(torch.int32),
        scale=torch.rand(adapters, generator=g) + 0.5 if scaled else None), used


def reference(p, used, swiglu):
    """(values, bounds) of the used rows in float64."""
    x, a, b = p["x"][:used].double(), p["a"].double(), p["b"].double()
    y = p["base"][:used].double()
    dy = 2.0**-24 * y.abs()
    k, experts = x.shape[1], a.shape[1]
    bounds = [0, used] if p["offsets"] is None else p["offsets"].tolist()
    for e in range(experts):
        lo, hi = bounds[e], bounds[e + 1]
        ids = p["row_adapters"][lo:hi]
        for q in ids.unique().tolist():
            if not 0 <= q < a.shape[0]:
                continue
            r = (ids == q).nonzero().flatten() + lo
            f = 1.0 if p["scale"] is None else float(p["scale"][q])
            s = x[r] @ a[q, e].T
            ds = (k / 16 + 20) * 2.0**-23 * (x[r].abs() @ a[q, e].abs().T) + 2.0**-16 * s.abs()
            y[r] += f * (s @ b[q, e].T)
            dy[r] += f * (ds @ b[q, e].abs().T + 22 * 2.0**-23 * (s.abs() @ b[q, e].abs().T))
    dy += 2.0**-24 * y.abs()
    if swiglu:
        half = y.shape[1] // 2
        g, u, dg, du = y[:, :half], y[:, half:], dy[:, :half], dy[:, half:]
        silu = g * torch.sigmoid(g)
        y = silu * u
        dy = 1.01 * (1.1 * u.abs() * dg + silu.abs() * du) + 8 * 2.0**-23 * y.abs()
    return y, dy + 2.0**-8 * y.abs()


def run(p, swiglu, out=None, **changes):
    from moe_dispatch import adapter_add, adapter_swiglu

    call = adapter_swiglu if swiglu else adapter_add
    args = {k: None if v is None else v.cuda() for k, v in {**p, **changes}.items()}
    return call(args["base"], args["x"], args["a"], args["b"], args["row_adapters"],
                offsets=args["offsets"], scale=args["scale"], out=out)


def check(p, used, swiglu):
    cols = p["base"].shape[1] // (2 if swiglu else 1)
    out = torch.full((p["x"].shape[0], cols), SENTINEL, dtype=torch.bfloat16, device="cuda")
    assert run(p, swiglu, out) is out
    want, bound = reference(p, used, swiglu)
    got = out.cpu()
    assert bool((got[used:] == SENTINEL).all())
    error = (got[:used].double() - want).abs()
    assert bool((error <= bound).all()), float((error - bound).max())
    return out


CASES = [
    # spans, k, n, adapters, rank
    (1, 64, 64, 1, 8),
    (3, 8, 8, 2, 8),
    ([1, 0, 0, 1], 4096, 520, 16, 16),
    ([0, 0, 5, 0, 0, 3, 0], 2056, 136, 3, 24),
    ([8] * 8, 264, 72, 12, 64),
    (200, 72, 1032, 7, 128),
    ([40, 0, 100, 116], 136, 200, 4, 40),        # 256 rows
    ([40, 0, 101, 116], 136, 200, 4, 40),        # 257: the sorted form
    (300, 8, 8, 5, 8),
    ([64, 64, 64, 65], 72, 136, 1, 16),
    ([0, 700, 0, 0, 300, 1, 0, 63], 520, 264, 9, 32),
    (1500, 200, 72, 300, 16),                    # runs of a few rows
    ([512] * 5, 136, 264, 3, 128),
    (5003, 64, 128, 24, 64),
    ([9] * 64, 328, 88, 512, 8),                 # every row its own pair, few-rows form
    ([20] * 60, 328, 88, 512, 8),                # and sorted: 1200 rows
    ([100] * 9, 72, 136, 80, 16),                # 913 rows, scattered over 720 pairs
    ([3000, 0, 1096], 1096, 1160, 6, 96),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0] if isinstance(c[0], int) else len(c[0])}-{c[1]}-{c[2]}-{c[3]}-{c[4]}")
@pytest.mark.parametrize("swiglu", [False, True], ids=["add", "swiglu"])
@pytest.mark.parametrize("grouped", [False, True], ids=["mixed", "grouped"])
def test_adapters_match_the_definition(case, swiglu, grouped):
    spans, k, n, adapters, rank = case
    behind = 0 if isinstance(spans, int) else 13
    p, used = make_problem(spans, k, n, adapters, rank, swiglu, seed=k + n, behind=behind,
                           grouped=grouped, scaled=rank != 16)
    check(p, used, swiglu)


@pytest.mark.parametrize("rows", [130, 1030])
@pytest.mark.parametrize("swiglu", [False, True])
def test_ids_outside_the_adapters_pick_none(rows, swiglu):
    p, used = make_problem([rows // 2, 0, rows - rows // 2], 136, 72, 4, 16, swiglu, 1)
    p["row_adapters"][::3] = torch.tensor([4, -1, 2**31 - 1, -2**31, 7]).repeat(rows)[: len(p["row_adapters"][::3])].to(torch.int32)
    check(p, used, swiglu)
    wide = p["row_adapters"].long()
    wide[wide == 4] = 2**32  # would be adapter 0 in 32 bits
    assert torch.equal(run(p, swiglu), run(p, swiglu, row_adapters=wide))
    p["row_adapters"][:] = -1
    out = check(p, used, swiglu)
    if not swiglu:
        assert torch.equal(out.cpu(), p["base"])


@pytest.mark.parametrize("rows", [100, 2000])
def test_add_in_place(rows):
    p, used = make_problem([rows // 4, rows // 2, rows // 4], 264, 136, 5, 16, False, 2, behind=9)
    want = run(p, False)
    base = p["base"].cuda()
    assert run({**p, "base": base}, False, base) is base
    assert torch.equal(base[:used], want[:used]) and torch.equal(base[used:].cpu(), p["base"][used:])


@pytest.mark.parametrize("rows", [60, 700])
@pytest.mark.parametrize("swiglu", [False, True])
def test_what_is_not_finite_stays_in_its_rows(rows, swiglu):
    p, used = make_problem([rows // 2, rows // 2], 136, 72, 6, 16, swiglu, 3)
    clean = run(p, swiglu)
    p["a"][1, :, 3] = float("nan")
    p["b"][2, :, 5] = float("inf")
    p["x"][7] = float("inf")
    p["base"][9, 4] = float("nan")
    out = run(p, swiglu)
    touched = (p["row_adapters"] == 1) | (p["row_adapters"] == 2)
    touched[7] = touched[9] = True
    assert torch.equal(out[~touched.cuda()], clean[~touched.cuda()])
    if bool((p["row_adapters"] == 1).any()):
        assert not torch.isfinite(out[(p["row_adapters"] == 1).cuda()]).any()


def test_rows_do_not_depend_on_the_batch_around_them():
    p, used = make_problem([600, 500], 264, 200, 5, 32, True, 4)
    want = run(p, True)
    order = torch.cat([torch.randperm(600, generator=torch.Generator().manual_seed(1)),
                       600 + torch.randperm(500, generator=torch.Generator().manual_seed(2))])
    shuffled = {**p, **{k: p[k][order] for k in ("base", "x", "row_adapters")}}
    assert torch.equal(run(shuffled, True), want[order.cuda()])
    assert torch.equal(run(p, True), want)


def test_long_projections_pass_32_bit_offsets():
    """base and out of more than 2^31 elements."""
    rows, n, rank, adapters = 70000, 32768, 8, 2
    g = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(rows, n, device="cuda", generator=g, dtype=torch.bfloat16)
    x = torch.randn(rows, 8, device="cuda", generator=g, dtype=torch.bfloat16)
    a = torch.randn(adapters, 1, rank, 8, device="cuda", generator=g, dtype=torch.bfloat16)
    b = torch.randn(adapters, 1, n, rank, device="cuda", generator=g, dtype=torch.bfloat16)
    ids = torch.randint(0, adapters, (rows,), device="cuda", generator=g, dtype=torch.int32)
    from moe_dispatch import adapter_add

    out = adapter_add(base, x, a, b, ids)
    for r in (0, 65535, 65536, rows - 1):
        p = dict(base=base[r:r + 1].cpu(), x=x[r:r + 1].cpu(), a=a.cpu(), b=b.cpu(), offsets=None,
                 row_adapters=ids[r:r + 1].cpu(), scale=None)
        want, bound = reference(p, 1, False)
        assert bool(((out[r].double().cpu() - want[0]).abs() <= bound[0]).all())


@pytest.mark.parametrize("rows", [60, 700])
def test_extreme_base_values_pass_through(rows):
    """A product of zero leaves every base value as it is: subnormals, the largest, infinities."""
    p, used = make_problem([rows // 2, rows // 2], 136, 200, 3, 24, False, 8)
    p["b"].zero_()
    values = torch.tensor([2.0**-133, -2.0**-130, 2.0**-126, 3.3895e38, -3.3895e38, float("inf"), -float("inf"), 1.0])
    p["base"].copy_(values.repeat(25).to(torch.bfloat16))
    p["base"][5, 17] = float("nan")
    out = run(p, False).cpu()
    same = out == p["base"]
    assert not bool(same[5, 17]) and bool(torch.isnan(out[5, 17]))
    same[5, 17] = True
    assert bool(same.all())


@pytest.mark.parametrize("rows", [60, 700])
@pytest.mark.parametrize("swiglu", [False, True])
def test_inference_mode_gives_the_same_rows(rows, swiglu):
    p, used = make_problem([rows // 2, rows // 2], 136, 72, 6, 16, swiglu, 3)
    want = run(p, swiglu)
    with torch.inference_mode():
        assert torch.equal(run(p, swiglu), want)


def test_no_rows():
    p, _ = make_problem([0, 0], 64, 64, 2, 8, True, 6)
    assert run(p, True).shape == (0, 64)
    p, used = make_problem([0, 0], 64, 64, 2, 8, False, 6, behind=300)
    check(p, used, False)


def test_calls_on_two_streams_and_in_two_graphs():
    problems = [make_problem([700, 800], 264, 136, 7, 16, swiglu, s)[0] for s, swiglu in ((1, True), (2, False))]
    problems = [{k: None if v is None else v.cuda() for k, v in p.items()} for p in problems]
    want = [run(p, s) for p, s in zip(problems, (True, False))]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    for _ in range(4):
        got = []
        for p, swiglu, stream in zip(problems, (True, False), streams):
            with torch.cuda.stream(stream):
                got.append(run(p, swiglu))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for p, swiglu, stream in zip(problems, (True, False), streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(run(p, swiglu))
        graphs.append(graph)
    for _ in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ------------------------------------------------------------------ the block


def make_block(config, implementation="cuda_fused", expert_dtype="bf16", seed=1):
    from moe_dispatch import MoEBlock

    return MoEBlock(config, implementation=implementation, expert_dtype=expert_dtype, seed=seed)


def make_adapters(config, count, ranks, seed, scaled=True):
    from moe_dispatch import MoEAdapters

    g = torch.Generator().manual_seed(seed)
    h, i, e = config.hidden, config.intermediate, config.experts
    r1, r2 = ranks

    def pair(r, k, n):
        if not r:
            return None, None
        return ((torch.randn(count, e, r, k, generator=g) / k**0.5).bfloat16().cuda(),
                (0.5 * torch.randn(count, e, n, r, generator=g) / r**0.5).bfloat16().cuda())

    return MoEAdapters(*pair(r1, h, 2 * i), *pair(r2, i, h),
                       (torch.rand(count, generator=g) + 0.5).cuda() if scaled else None)


@pytest.mark.parametrize("tokens", [1, 5, 67, 400])
@pytest.mark.parametrize("ranks", [(16, 16), (8, 0), (0, 24)], ids=str)
def test_block_with_adapters(tokens, ranks):
    """Against the float64 definition from the block's own stages, and bit for bit against the
    block without adapters where a token has none."""
    from moe_dispatch import MoEConfig

    config = MoEConfig(256, 512, 8, 2)
    block = make_block(config)
    adapters = make_adapters(config, 5, ranks, 3)
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, 256, generator=g).bfloat16().cuda()
    ids = torch.randint(-1, 5, (tokens,), generator=g)
    plain = block(x).clone()
    block.set_adapters(adapters)
    assert torch.equal(block(x), plain)  # adapters are used only where ids are given
    out = block(x, adapter_ids=ids.to(torch.int32).cuda()).clone()
    assert torch.equal(out[(ids < 0).cuda()], plain[(ids < 0).cuda()])
    assert torch.equal(block(x, adapter_ids=ids.cuda()), out)  # int64 ids
    assert torch.equal(block(x, adapter_ids=torch.full_like(ids, -1).cuda()), plain)
    assert torch.equal(block(x), plain)

    # the "cuda" implementation walks the same kernels
    unfused = make_block(config, "cuda")
    unfused.set_adapters(adapters)
    assert torch.equal(unfused(x, adapter_ids=ids.cuda()), out)

    # float64: W + scale B A per token and expert
    choice, _, weights = block.route(x)
    expected = torch.zeros(tokens, 256, dtype=torch.float64)
    scale = adapters.scale.double().cpu()
    for t in range(tokens):
        q = int(ids[t])
        for j in range(2):
            e = int(choice[t, j])
            up = block.gate_up_weight[e].double().cpu()
            down = block.down_weight[e].double().cpu()
            if q >= 0 and ranks[0]:
                up = up + scale[q] * adapters.gate_up_b[q, e].double().cpu() @ adapters.gate_up_a[q, e].double().cpu()
            if q >= 0 and ranks[1]:
                down = down + scale[q] * adapters.down_b[q, e].double().cpu() @ adapters.down_a[q, e].double().cpu()
            y = up @ x[t].double().cpu()
            act = torch.nn.functional.silu(y[:512]) * y[512:]
            expected[t] += float(weights[t, j]) * (down @ act)
    # bf16 roundings: the projection (2^-8 of each half), the activation, the down product, its
    # sum with the adapters' part, the output: in the norm sqrt(2 + 4) half steps at most
    error = float((out.double().cpu() - expected).norm() / expected.norm())
    assert error <= 6**0.5 * 2.0**-8


def test_block_adapters_in_a_graph_follow_their_ids():
    from moe_dispatch import MoEConfig

    config = MoEConfig(256, 256, 16, 4)
    block = make_block(config)
    block.set_adapters(make_adapters(config, 3, (16, 8), 4))
    g = torch.Generator().manual_seed(2)
    x = torch.randn(300, 256, generator=g).bfloat16().cuda()
    batches = [torch.randint(-1, 3, (300,), generator=g, dtype=torch.int32).cuda() for _ in range(3)]
    want = [block(x, adapter_ids=b).clone() for b in batches]
    ids = batches[0].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(x, adapter_ids=ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = block(x, adapter_ids=ids)
    for b, w in zip(batches, want):
        ids.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_block_with_fp8_experts_and_adapters():
    from moe_dispatch import MoEConfig

    config = MoEConfig(256, 512, 8, 2)
    block, unfused = make_block(config, "cuda_fused", "fp8_e4m3"), make_block(config, "cuda", "fp8_e4m3")
    adapters = make_adapters(config, 4, (16, 16), 5)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(90, 256, generator=g).bfloat16().cuda()
    ids = torch.randint(-1, 4, (90,), generator=g, dtype=torch.int32).cuda()
    plain = block(x).clone()
    for b in (block, unfused):
        b.set_adapters(adapters)
    out = block(x, adapter_ids=ids).clone()
    assert torch.equal(unfused(x, adapter_ids=ids), out)
    assert torch.equal(out[ids < 0], plain[ids < 0]) and not torch.equal(out, plain)


def test_block_refuses_ids_that_do_not_fit():
    from moe_dispatch import MoEConfig

    config = MoEConfig(64, 64, 4, 2)
    block = make_block(config)
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="set_adapters"):
        block(x, adapter_ids=ids)
    block.set_adapters(make_adapters(config, 2, (8, 8), 1))
    for bad in (ids[:5], ids.cpu(), ids[None]):
        with pytest.raises(ValueError):
            block(x, adapter_ids=bad)
    with pytest.raises(TypeError):
        block(x, adapter_ids=ids.float())
    with pytest.raises(ValueError, match="device"):
        cpu = make_adapters(config, 2, (8, 0), 1)
        cpu.gate_up_a = cpu.gate_up_a.cpu()
        block.set_adapters(cpu)
    block.set_adapters(None)
    with pytest.raises(ValueError, match="set_adapters"):
        block(x, adapter_ids=ids)
    assert block(x[:0]).shape == (0, 64)


def test_calls_in_a_row_see_what_the_one_before_wrote():
    """In place, ids from the device, small forms back to back: each call reads the base and the
    ids that the kernels just before it have written, eagerly and in a graph."""
    from moe_dispatch import adapter_add

    p, _ = make_problem([40, 0, 30], 264, 1032, 5, 16, False, 12)
    p = {k: None if v is None else v.cuda() for k, v in p.items()}
    rounds = 8
    ids = torch.randint(-1, 5, (rounds, 70), device="cuda", dtype=torch.int32)

    def chain(row_ids, base, sync):
        for i in range(rounds):
            row_ids.copy_(ids[i])
            base.mul_(0.5)
            if sync:
                torch.cuda.synchronize()
            adapter_add(base, p["x"], p["a"], p["b"], row_ids, offsets=p["offsets"], scale=p["scale"], out=base)
            if sync:
                torch.cuda.synchronize()

    want = p["base"].clone()
    chain(torch.empty_like(ids[0]), want, True)
    for _ in range(20):
        got = p["base"].clone()
        chain(torch.empty_like(ids[0]), got, False)
        assert torch.equal(got, want)
    row_ids, got = torch.empty_like(ids[0]), p["base"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(row_ids, got, False)
    for _ in range(20):
        got.copy_(p["base"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
