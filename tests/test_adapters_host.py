"""What the adapters refuse, before anything reaches a GPU."""

import pytest
import torch

from moe_dispatch import MoEAdapters, MoEConfig, adapter_add, adapter_swiglu
from moe_dispatch.adapters import adapter_ids32, check_adapters
from moe_dispatch._extension import load_library

BF16 = torch.bfloat16


def add_args(**changes):
    args = dict(base=torch.zeros(6, 32, dtype=BF16), x=torch.zeros(6, 16, dtype=BF16),
                a=torch.zeros(3, 2, 8, 16, dtype=BF16), b=torch.zeros(3, 2, 32, 8, dtype=BF16),
                row_adapters=torch.zeros(6, dtype=torch.int32),
                offsets=torch.tensor([0, 2, 6], dtype=torch.int32), scale=torch.ones(3))
    args.update(changes)
    return args


@pytest.mark.parametrize("changes, error, message", [
    (dict(base=torch.zeros(5, 32, dtype=BF16)), ValueError, "expected base"),
    (dict(base=torch.zeros(6, 32)), TypeError, "BF16"),
    (dict(x=torch.zeros(6, 16)), TypeError, "BF16"),
    (dict(x=torch.zeros(16, 6, dtype=BF16).t()), ValueError, "contiguous"),
    (dict(base=torch.zeros(32, 6, dtype=BF16).t()), ValueError, "contiguous"),
    (dict(base=torch.zeros(6, 36, dtype=BF16), b=torch.zeros(3, 2, 36, 8, dtype=BF16)), ValueError, "multiples of 8"),
    (dict(a=torch.zeros(3, 1, 8, 16, dtype=BF16)), ValueError, "do not match"),
    (dict(b=torch.zeros(3, 2, 32, 16, dtype=BF16)), ValueError, "do not match"),
    (dict(a=torch.zeros(3, 2, 8, 16), b=torch.zeros(3, 2, 32, 8)), ValueError, "bf16"),
    (dict(a=torch.zeros(3, 2, 12, 16, dtype=BF16), b=torch.zeros(3, 2, 32, 12, dtype=BF16)), ValueError, "rank"),
    (dict(a=torch.zeros(3, 2, 136, 16, dtype=BF16), b=torch.zeros(3, 2, 32, 136, dtype=BF16)), ValueError, "rank"),
    (dict(a=torch.zeros(600, 2, 8, 16, dtype=BF16), b=torch.zeros(600, 2, 32, 8, dtype=BF16)), ValueError, "adapters"),
    (dict(a=torch.zeros(3, 2, 16, 8, dtype=BF16).transpose(2, 3)), ValueError, "contiguous"),
    (dict(offsets=torch.tensor([0, 2, 6])), ValueError, "offsets"),
    (dict(offsets=None), ValueError, "do not match"),
    (dict(scale=torch.ones(2)), ValueError, "scale"),
    (dict(scale=torch.ones(3, dtype=BF16)), ValueError, "scale"),
    (dict(row_adapters=torch.zeros(5, dtype=torch.int32)), ValueError, "per row"),
    (dict(row_adapters=torch.zeros(6)), TypeError, "int32 or int64"),
    (dict(out=torch.zeros(6, 16, dtype=BF16)), ValueError, "out"),
    (dict(a=torch.zeros(3, 2, 8, 16, dtype=BF16, requires_grad=True)), ValueError, "forward-only"),
    (dict(), RuntimeError, "require CUDA"),
])
def test_adapter_add_refuses(changes, error, message):
    with pytest.raises(error, match=message):
        adapter_add(**add_args(**changes))


def swiglu(**changes):
    args = add_args(**changes)
    return adapter_swiglu(args.pop("base"), **args)


def test_out_must_not_overlap_an_input():
    buffer = torch.zeros(13, 32, dtype=BF16)
    base = buffer[:6]
    with pytest.raises(ValueError, match="overlap"):
        adapter_add(**add_args(base=base, out=buffer[1:7]))
    with pytest.raises(RuntimeError, match="CUDA"):  # base itself is fine
        adapter_add(**add_args(base=base, out=buffer[:6]))
    with pytest.raises(RuntimeError, match="CUDA"):
        adapter_add(**add_args(base=base, out=buffer[6:12]))
    x = torch.zeros(6, 16, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        swiglu(x=x, out=x)
    with pytest.raises(ValueError, match="overlap"):
        swiglu(base=base, out=base.view(-1)[:96].view(6, 16))


def test_int64_ids_past_int32_stay_outside():
    ids = adapter_ids32(torch.tensor([0, 2**32, -2**40, 5]), 4, "row")
    assert ids.dtype == torch.int32 and ids.tolist() == [0, 2**31 - 1, -1, 5]


def block_adapters(**changes):
    args = dict(gate_up_a=torch.zeros(3, 4, 8, 64, dtype=BF16), gate_up_b=torch.zeros(3, 4, 256, 8, dtype=BF16),
                down_a=torch.zeros(3, 4, 16, 128, dtype=BF16), down_b=torch.zeros(3, 4, 64, 16, dtype=BF16),
                scale=torch.ones(3))
    args.update(changes)
    return MoEAdapters(**args)


@pytest.mark.parametrize("changes, message", [
    (dict(gate_up_a=None, gate_up_b=None, down_a=None, down_b=None), "need"),
    (dict(gate_up_a=None), "together"),
    (dict(down_b=None), "together"),
    (dict(gate_up_b=torch.zeros(3, 4, 128, 8, dtype=BF16)), "do not match"),
    (dict(down_a=torch.zeros(2, 4, 16, 128, dtype=BF16), down_b=torch.zeros(2, 4, 64, 16, dtype=BF16)), "same adapters"),
    (dict(scale=torch.ones(4)), "scale"),
])
def test_block_adapters_that_do_not_fit_are_refused(changes, message):
    config = MoEConfig(64, 128, 4, 2)
    check_adapters(block_adapters(), config, torch.device("cpu"))
    check_adapters(block_adapters(down_a=None, down_b=None, scale=None), config, torch.device("cpu"))
    with pytest.raises(ValueError, match=message):
        check_adapters(block_adapters(**changes), config, torch.device("cpu"))
    with pytest.raises(ValueError, match="device"):
        check_adapters(block_adapters(), config, torch.device("cuda", 0))


def adapter_call(lib, **changes):
    v = dict(base=16, x=16, a=16, b=16, scale=None, ids=16, offsets=16, out=32, rows=4, k=16, n=16, rank=8,
             adapters=2, experts=2, scratch=None, bytes=0)
    v.update(changes)
    call = lib.moe_adapter_swiglu if v.pop("swiglu", False) else lib.moe_adapter_add
    return call(*v.values(), None)


@pytest.mark.parametrize("changes, message", [
    (dict(rows=-1), "rows"), (dict(rows=2**30), "rows"), (dict(k=12), "multiples of 8"), (dict(n=0), "multiples of 8"),
    (dict(rank=4), "rank"), (dict(rank=136), "rank"), (dict(adapters=0), "adapters"), (dict(adapters=513), "adapters"),
    (dict(experts=0), "experts"), (dict(experts=513), "experts"), (dict(offsets=None), "offsets"),
    (dict(out=None), "null"), (dict(x=24), "aligned"), (dict(swiglu=True, out=16), "projection"),
    (dict(rows=2**29 - 1, n=2**20), "grid"),
])
def test_library_refuses(changes, message):
    lib = load_library()
    assert adapter_call(lib, **changes) == 1
    assert message in lib.moe_last_error().decode()


def test_library_refuses_bad_row_maps_and_queries():
    lib = load_library()
    assert adapter_call(lib, rows=0) == 0
    assert lib.moe_adapter_rows(None, None, None, None, None, 4, 0, 8, 16, None) == 1
    assert lib.moe_adapter_rows(None, None, None, None, None, 4, 2, 0, 16, None) == 1
    assert lib.moe_adapter_rows(None, None, None, None, None, 4, 2, 8, 16, None) == 1
    assert "null" in lib.moe_last_error().decode()
    assert lib.moe_adapter_scratch_bytes(4, 12, 8, 2, 1) == -1
    assert lib.moe_adapter_scratch_bytes(4, 16, 8, 600, 1) == -1


def test_library_refuses_rows_too_long_for_the_grid():
    lib = load_library()
    assert adapter_call(lib, k=2**26 + 8) == 1
    assert "2^26" in lib.moe_last_error().decode()
    assert lib.moe_adapter_scratch_bytes(4, 2**26 + 8, 8, 2, 1) == -1
