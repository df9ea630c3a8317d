"""Low-rank adapters of many requests beside a shared projection (adapters.hip).

One step of a model groups its rows once (:func:`adapter_plan`) and then adds the
adapters' part to each projection (:func:`adapter_add`).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

import polyrl_amd.ops as _ops
from . import ref

MOST_ADAPTERS = 4095
MOST_PARTS = 8
MOST_RANK = 256


class AdapterPlan:
    """Rows of a step by their adapters.  On the GPU the grouping is a tensor that
    :func:`adapter_plan` computed there: calls wait for nothing and can be captured."""

    def __init__(self, index: torch.Tensor, slots: int,
                 table: Optional[torch.Tensor]):
        self.index = index
        self.rows = index.shape[0]
        self.slots = slots
        self.table = table


def adapter_plan(index: torch.Tensor, slots: int) -> AdapterPlan:
    """index (T,) int32: every row's adapter; one outside of 0 .. slots - 1 names none."""
    if index.dim() != 1 or index.dtype != torch.int32:
        raise ValueError("adapter_plan: index (T,) int32")
    if not 1 <= slots <= MOST_ADAPTERS:
        raise ValueError(f"adapter_plan: 1 to {MOST_ADAPTERS} adapters")
    table = None
    if index.is_cuda:
        index = index.contiguous()
        table = _ops._require_ext().adapter_plan(index, slots)
    return AdapterPlan(index, slots, table)


def adapter_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor,
                b: torch.Tensor, scale: torch.Tensor, plan: AdapterPlan,
                widths: Optional[Sequence[int]] = None,
                ranks: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] + scale[i] * B_i (A_i x[t]) for the adapter i of every row, y[t] where a row
    has none (no autograd).

    y (T, N), x (T, K) rows of a projection's output and input; a (S, P, r, K) and b
    (S, N, r): the S adapters of a projection of P parts whose ``widths`` add up to N
    (q, k and v of one fused product; default: one part).  scale (S,) fp32.  ranks (S,)
    int32: how much of r an adapter uses (0: none, its rows are y's); what a and b hold
    beyond is not read.  ``out``: where the result goes, ``out=y`` in place, else apart from
    all operands.  bf16 or fp32, all of one type; at most 8 parts, r at most 256, K below
    2^20.  The adapters a and b are contiguous, rows of y, x and out may lie apart."""
    if y.is_cuda:                     # (checks and all in one call: 8 us for 9)
        if plan.table is None:
            raise ValueError("adapter_add: a plan of the CPU")
        return _ops._require_ext().adapter_add(
            y, x, a, b, scale, ranks, plan.table, plan.rows, plan.slots,
            () if widths is None else widths, out)
    widths = [y.shape[1]] if widths is None else [int(w) for w in widths]
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (y, x, a, b, scale, out)):
        raise RuntimeError("adapter_add has no gradients: call it under "
                           "torch.no_grad()")
    if plan.rows != y.shape[0] or a.shape[0] != plan.slots:
        raise ValueError(f"adapter_add: a plan of {plan.rows} rows and "
                         f"{plan.slots} adapters for {y.shape[0]} and {a.shape[0]}")
    if not 1 <= len(widths) <= MOST_PARTS or a.dim() != 4 \
            or not 1 <= a.shape[2] <= MOST_RANK or a.shape[3] >= 1 << 20:
        raise ValueError(f"adapter_add: 1 to {MOST_PARTS} parts, ranks 1 to "
                         f"{MOST_RANK}, inner widths below 2^20")
    if out is not None:
        in_place = out.data_ptr() == y.data_ptr() and out.stride() == y.stride()
        if any(ref.rows_overlap(out, t)
               for t in ((x, a, b) if in_place else (y, x, a, b))):
            raise ValueError("adapter_add: out on top of an operand")
    res = ref.adapter_add(y, x, a, b, scale, plan.index, widths, ranks)
    return res if out is None else out.copy_(res)
