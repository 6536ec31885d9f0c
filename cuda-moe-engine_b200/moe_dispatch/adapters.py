"""Low-rank adapters of many requests beside the experts' grouped projections.

The experts' weights are shared by every request of a batch; a request may bring
its own low-rank change of them.  For packed row r of expert e whose request uses
adapter p,

    out[r] = base[r] + scale[p] * (x[r] A[p,e]^T) B[p,e]^T

where base is the shared projection's output.  ``MoEBlock.set_adapters`` and
``block(x, adapter_ids=...)`` run them inside the block; ``adapter_add`` and
``adapter_swiglu`` are the checked one-call forms, over the packed rows of
``dispatch`` or, without offsets, over the rows of any one shared projection.
Like the experts they are forward-only.  The reference has no counterpart.
"""

from dataclasses import dataclass

import torch

from ._extension import get_extension

MAX_ADAPTERS = 512
MAX_RANK = 128


@dataclass
class MoEAdapters:
    """P adapters of a block's experts, bf16 on the block's device.

    gate_up_a [P,E,r,H] and gate_up_b [P,E,2I,r] change the gate/up projection
    (gate rows 0..I-1, up rows I..2I-1 of b, as in ``MoEWeights``), down_a
    [P,E,r,I] and down_b [P,E,H,r] the down projection; either pair may be None,
    and the two may have different ranks.  scale [P] fp32 multiplies both (None:
    1).  Gate and up adapters with matrices a of their own go into one pair of
    twice the rank, with zeros in b where a half has no part.
    """

    gate_up_a: torch.Tensor = None
    gate_up_b: torch.Tensor = None
    down_a: torch.Tensor = None
    down_b: torch.Tensor = None
    scale: torch.Tensor = None

    @property
    def count(self):
        return (self.gate_up_a if self.gate_up_a is not None else self.down_a).shape[0]


def _check_pair(name, a, b, experts, k_dim, n_cols):
    if a.ndim != 4 or b.ndim != 4 or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
        raise ValueError(f"{name}: expected bf16 a[P,E,r,K] and b[P,E,N,r]")
    adapters, a_experts, rank, a_dim = a.shape
    if a_experts != experts or a_dim != k_dim or b.shape != (adapters, experts, n_cols, rank):
        raise ValueError(f"{name}: a and b do not match the projection")
    if not 1 <= adapters <= MAX_ADAPTERS:
        raise ValueError(f"{name}: adapters must be 1..{MAX_ADAPTERS}")
    if not 8 <= rank <= MAX_RANK or rank % 8:
        raise ValueError(f"{name}: rank must be a multiple of 8 up to {MAX_RANK}")
    if not a.is_contiguous() or not b.is_contiguous():
        raise ValueError(f"{name}: a and b must be contiguous")


def _check_scale(scale, adapters):
    if scale is not None and (scale.shape != (adapters,) or scale.dtype != torch.float32
                              or not scale.is_contiguous()):
        raise ValueError("expected contiguous fp32 scale[P]")


def check_adapters(adapters, config, device):
    """Reject adapters that do not fit a block of this configuration."""
    if adapters.gate_up_a is None and adapters.down_a is None:
        raise ValueError("adapters need a gate_up or a down pair")
    for name, a, b, k_dim, n_cols in (
            ("gate_up", adapters.gate_up_a, adapters.gate_up_b, config.hidden, 2 * config.intermediate),
            ("down", adapters.down_a, adapters.down_b, config.intermediate, config.hidden)):
        if (a is None) != (b is None):
            raise ValueError(f"{name}: a and b come together")
        if a is not None:
            _check_pair(name, a, b, config.experts, k_dim, n_cols)
            if a.shape[0] != adapters.count:
                raise ValueError("gate_up and down must hold the same adapters")
    _check_scale(adapters.scale, adapters.count)
    for tensor in (adapters.gate_up_a, adapters.gate_up_b, adapters.down_a, adapters.down_b,
                   adapters.scale):
        if tensor is not None and tensor.device != device:
            raise ValueError("adapters must be on the block's device")


def adapter_ids32(ids, count, what):
    """ids [count] as contiguous int32; values past int32 stay out of range."""
    if ids.ndim != 1 or ids.shape[0] != count:
        raise ValueError(f"expected one adapter id per {what}")
    if ids.dtype == torch.int32:
        return ids.contiguous()
    if ids.dtype != torch.int64:
        raise TypeError("adapter ids must be int32 or int64")
    return ids.clamp(-1, 2**31 - 1).to(torch.int32)


def _apply(base, x, a, b, row_adapters, offsets, scale, out, swiglu):
    if base.ndim != 2 or x.ndim != 2 or base.shape[0] != x.shape[0]:
        raise ValueError("expected base[R,N] and x[R,K]")
    if base.dtype != torch.bfloat16 or x.dtype != torch.bfloat16:
        raise TypeError("base and x must be BF16")
    rows, n_cols = base.shape
    k_dim = x.shape[1]
    halves = 2 if swiglu else 1
    if k_dim < 8 or k_dim % 8 or n_cols < 8 * halves or n_cols % (8 * halves):
        raise ValueError("projection dimensions must be multiples of 8")
    if offsets is None:
        experts = 1
    else:
        if offsets.ndim != 1 or offsets.numel() < 2 or offsets.dtype != torch.int32:
            raise ValueError("expected int32 offsets[E+1]")
        experts = offsets.numel() - 1
    _check_pair("adapter", a, b, experts, k_dim, n_cols)
    _check_scale(scale, a.shape[0])
    shape = (rows, n_cols // halves)
    device, grad = x.device, torch.is_grad_enabled()
    if out is not None:
        if out.shape != shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous bf16 tensor [{shape[0]},{shape[1]}]")
        if out.device != device:
            raise ValueError("all tensors must be on the same device")
        if grad and out.requires_grad:
            raise ValueError("CUDA operators are forward-only; detach inputs or use inference_mode")
        low = out.data_ptr()
        high = low + out.nbytes
    for t in (base, x, a, b, row_adapters, offsets, scale):
        if t is None:
            continue
        if t.device != device:
            raise ValueError("all tensors must be on the same device")
        if grad and t.requires_grad:
            raise ValueError("CUDA operators are forward-only; detach inputs or use inference_mode")
        if out is not None:
            start = t.data_ptr()
            if start < high and low < start + t.nbytes and (swiglu or t is not base or start != low):
                raise ValueError("out must not overlap an input (adapter_add may write base itself)")
    if not base.is_contiguous() or not x.is_contiguous():
        raise ValueError("base and x must be contiguous")
    if offsets is not None and not offsets.is_contiguous():
        raise ValueError("offsets must be contiguous")
    row_adapters = adapter_ids32(row_adapters, rows, "row")
    if not x.is_cuda:
        raise RuntimeError("adapters require CUDA")
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=device)
    extension = get_extension()
    function = extension.lib.moe_adapter_swiglu if swiglu else extension.lib.moe_adapter_add
    extension.launch_adapter(function, base, x, a, b, scale, row_adapters, offsets, out)
    return out


def adapter_add(base, x, a, b, row_adapters, *, offsets=None, scale=None, out=None):
    """base[r] + scale[p] * (x[r] a[p,e]^T) b[p,e]^T for every row r.

    base [R,N] and x [R,K] bf16; a [P,E,r,K] and b [P,E,N,r] bf16; row_adapters
    [R] int32 or int64: the row's adapter p, outside 0..P-1 (say -1) for none;
    offsets [E+1] int32, from 0 up: expert e has rows offsets[e]..offsets[e+1]-1
    (None: one expert with every row); scale [P] fp32 (None: 1).  Sums in fp32, rounded once.
    Writes ``out`` (base itself, or a bf16 [R,N] tensor that overlaps no input; a
    new one if None) and returns it.  Rows behind the last expert's are neither
    read nor written.  No host synchronisation; each call uses scratch of its own
    from torch's allocator, so calls on several streams or in several graphs are
    independent.
    """
    return _apply(base, x, a, b, row_adapters, offsets, scale, out, False)


def adapter_swiglu(projection, x, a, b, row_adapters, *, offsets=None, scale=None, out=None):
    """silu(y[:, :I]) * y[:, I:] of y = adapter_add(projection, ...), y not rounded.

    projection [R,2I] bf16 (gate columns 0..I-1, then up), b [P,E,2I,r]; ``out``
    [R,I] bf16 overlaps no input.  Otherwise as ``adapter_add``.
    """
    return _apply(projection, x, a, b, row_adapters, offsets, scale, out, True)
