"""Grouped MoE experts on microscaled 4-bit weights (``kernels.mx``): products of ragged groups of rows with their experts' weights
over the plans of ``experts``.  A (row, slot) pair's bits never depend on the other rows of the call, nor on the form of the plan.

Rows are quantised by the first projection; its activations are computed from fp32 sums and quantised once, from fp32, for the
second."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from . import experts as grouped
from .kernels import mx


@dataclass
class Experts:
    """One layer's experts: gate and up (SwiGLU) or up (relu^2), and down, as super-blocks with the expert outermost."""

    up: torch.Tensor          # [E, ceil(rows / 128), bytes] uint8; rows = 2 NI (gate and up interleaved) or NI
    down: torch.Tensor        # [E, ceil(D / 128), bytes]
    width: int                # NI
    dims: int                 # D
    limit: float = 0.0        # SwiGLU clip (0: none)
    gated: bool = True

    @property
    def count(self) -> int:
        return self.up.shape[0]

    @property
    def swiglu(self) -> bool:
        return self.gated

    def bytes_per_expert(self) -> int:
        return self.up[0].numel() + self.down[0].numel()


def make(up: list[tuple], down: tuple, *, limit: float = 0.0) -> Experts:
    """One layer's stored arrays: ``up`` [gate, up] (SwiGLU) or [up] (relu^2), ``down``, each (words [E, n, k / 8], scales)."""

    if len(up) not in (1, 2):
        raise ValueError("experts take a gate and an up projection, or an up projection alone")
    if up[0][0].dim() != 3 or down[0].dim() != 3:
        raise ValueError("experts: words [E, n, k / 8] are wanted")
    e, width, d8 = up[0][0].shape
    if width % mx.BLOCK or tuple(down[0].shape) != (e, d8 * 8, width // 8):
        raise ValueError(f"experts: down {tuple(down[0].shape)} does not follow up {tuple(up[0][0].shape)} (widths in whole blocks of 32)")
    u = mx.pack_experts(*up[0], up[1] if len(up) == 2 else None)
    return Experts(u, mx.pack_experts(*down), width, d8 * 8, float(limit), len(up) == 2)


def _items(plan: grouped.Plan, rows: int) -> int:
    return min(grouped.max_items(rows * plan.slots, plan.experts, plan.tile), plan.items.shape[0])


def _call(who, x, slots, table, n, k, plan, rows, out, operands, epi, limit, work, pdl=False):
    if plan.experts > table.shape[0]:
        raise ValueError(f"the plan routes to {plan.experts} experts but the table holds {table.shape[0]}")
    pairs = rows * plan.slots
    if rows < 1 or pairs > plan.members.shape[0]:
        raise ValueError(f"{who}: 1 to {plan.rows} rows fit the plan")
    if table.dtype != torch.uint8 or table.shape[1:] != (-(-n // 128), mx.super_block_bytes(k)) or not table[0].is_contiguous():
        raise ValueError(f"{who}: the table does not have the super-blocks of its shape")
    if table.device != plan.items.device:
        raise ValueError(f"{who}: the plan and the weights must share a CUDA device")
    stream = _lib.stream_of(table)
    items = _items(plan, rows)
    if x is not None:
        need = _lib.lib().tf_mx_experts_bytes(k, plan.tile, items)
        work = torch.empty((need,), dtype=torch.uint8, device=x.device) if need > 0 else None
    _lib.native().tf_mx_experts(
        who, x, 0 if x is None else x.stride(0), slots, table, table.stride(0), table.shape[0], n, k, plan.items, plan.counts, plan.members,
        pairs, items, plan.tile, out, 0 if out is None else out.stride(0), out is not None and out.dtype == torch.float32, operands, epi, limit,
        work, 0 if work is None else work.numel(), pdl, stream)


def _inputs(x, k, need, device, who):
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != k or x.shape[0] < need:
        raise ValueError(f"{who}: x must be ({need}, {k}) bf16")
    if x.device != device:
        raise ValueError(f"{who}: x and the weights must share a CUDA device")
    if x.stride(1) != 1 or x.stride(0) % 8 or x.stride(0) < k or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _outputs(out, need, cols, types, device, who):
    if out.dtype not in types or out.dim() != 2 or out.shape[1] != cols or out.shape[0] < need or out.stride(1) != 1 or out.stride(0) < cols \
            or out.device != device:
        raise ValueError(f"{who}: out must be ({need}, {cols}) with unit-stride rows on the weights' device")


def gate_up(x: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """x [R, D] bf16 -> out [R * slots, NI] bf16, each pair's activation (rounded once from its fp32 sums)."""

    x = _inputs(x, ex.dims, rows, ex.up.device, "gate_up")
    _outputs(out, rows * plan.slots, ex.width, (torch.bfloat16,), ex.up.device, "gate_up")
    _call("gate_up", x, plan.slots, ex.up, (2 if ex.gated else 1) * ex.width, ex.dims, plan, rows, out, None, 2 if ex.gated else 1, ex.limit,
          None)


def down(act: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """act [R * slots, NI] bf16 -> out [R * slots, D] per pair, fp32 or bf16."""

    act = _inputs(act, ex.width, rows * plan.slots, ex.down.device, "down")
    _outputs(out, rows * plan.slots, ex.dims, (torch.float32, torch.bfloat16), ex.down.device, "down")
    _call("down", act, 0, ex.down, ex.dims, ex.width, plan, rows, out, None, 0, 0.0, None)


def layer(x: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """x [R, D] bf16 -> out [R * slots, D] per pair, fp32 or bf16: both projections, the activations between them quantised where
    the first one computes them."""

    x = _inputs(x, ex.dims, rows, ex.up.device, "experts")
    _outputs(out, rows * plan.slots, ex.dims, (torch.float32, torch.bfloat16), ex.down.device, "experts")
    act = torch.empty((_items(plan, rows) * _lib.lib().tf_mx_operand_bytes(plan.tile, ex.width),), dtype=torch.uint8, device=x.device)
    _call("experts (gate, up)", x, plan.slots, ex.up, (2 if ex.gated else 1) * ex.width, ex.dims, plan, rows, None, act, 2 if ex.gated else 1,
          ex.limit, None)
    # the first projection waited for the plan, so the second may read it, and its weights, while the first runs
    _call("experts (down)", None, 0, ex.down, ex.dims, ex.width, plan, rows, out, None, 0, 0.0, act, pdl=True)
