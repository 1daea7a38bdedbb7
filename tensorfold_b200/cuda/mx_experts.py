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


def _call(what: int, x: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    _lib.native().mx_experts(what, x, ex.up, ex.down, ex.dims, ex.width, ex.gated, ex.limit, plan.items, plan.counts, plan.members, plan.slots,
                             plan.experts, plan.tile, out, rows)


def gate_up(x: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """x [R, D] bf16 -> out [R * slots, NI] bf16, each pair's activation (rounded once from its fp32 sums).  ``out`` may not share
    memory with x (nor act's in ``down``; ``layer`` has read x before it writes)."""

    _call(1, x, ex, plan, out, rows)


def down(act: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """act [R * slots, NI] bf16 -> out [R * slots, D] per pair, fp32 or bf16."""

    _call(2, act, ex, plan, out, rows)


def layer(x: torch.Tensor, ex: Experts, plan: grouped.Plan, out: torch.Tensor, rows: int) -> None:
    """x [R, D] bf16 -> out [R * slots, D] per pair, fp32 or bf16: both projections, the activations between them quantised where
    the first one computes them."""

    _call(0, x, ex, plan, out, rows)
