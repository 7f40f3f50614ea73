"""(record, model) pairs sorted by model and back, on MI355X.

An ensemble of shadow models (attacks/ensemble/rmia/shadow_model_training.py:308 trains 16 of one base) is evaluated by the reference
model after model.  Here the pairs of all models run as one batch: ``route_rows`` plans it, ``dispatch_rows`` copies every record's row
to its pairs' places, the layers work on rows sorted by model (``adapters.adapter_linear`` takes ``plan.offsets``), and
``combine_rows`` brings the results back to the records, weighted.  Both copies carry gradients.  There is no CPU path.
"""
from __future__ import annotations

import operator

import torch
from torch import Tensor

from ._lib import native, no_tangents, ordinary

MAX_GROUPS = 1024  # MTK_ROUTE_MAX_GROUPS of include/mtk.h
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # enum mtk_dtype


def dtype_code(t: Tensor, what: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: {t.dtype} (float32, bfloat16 or float16)")
    return code


def rows_of(t: Tensor) -> Tensor:
    """``t`` [n, D] itself where its rows are contiguous (any row stride, also 0 of an expanded row), else a contiguous copy."""
    return t if t.shape[0] == 0 or ((t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= 0) else t.contiguous()


class RowPlan:
    """Where the pairs go: what ``route_rows`` returns.  ``order`` [P] int32: the pair in each place, ``slot`` (the shape of ``index``) int32: the
    place of each pair (for a pair whose index was out of range both hold the complement, ``~pair`` and ``~place``), ``offsets`` [n_groups + 1] int32: model e's pairs are in
    places ``offsets[e]`` to ``offsets[e + 1] - 1``, pairs without a model behind them all."""

    __slots__ = ("order", "slot", "offsets", "n_groups", "n_rows", "copies")

    def __init__(self, order: Tensor, slot: Tensor, offsets: Tensor, n_groups: int, n_rows: int, copies: int):
        self.order, self.slot, self.offsets = order, slot, offsets
        self.n_groups, self.n_rows, self.copies = n_groups, n_rows, copies


def route_rows(index: Tensor, n_groups: int) -> RowPlan:
    """Plan for ``index`` [N] or [N, k] (whole numbers): the model of record n's copy j, in [0, n_groups), or -1 for a copy without a
    model.  The same model twice in a record is two pairs.  Pairs keep their order within a model.  A pair whose index is out of
    range goes where -1 goes, and its rows are NaN: dispatched, combined and in gradients."""
    if not index.is_cuda:
        raise RuntimeError("route_rows: midst_toolkit_amd has no CPU path; move the indices to the MI355X")
    got = native().route(index, n_groups)
    if got is not None:
        return RowPlan(*got, n_groups, index.shape[0], 1 if index.dim() == 1 else index.shape[1])
    if index.dim() not in (1, 2) or index.dtype.is_floating_point or index.dtype.is_complex or index.dtype == torch.bool:
        raise ValueError(f"route_rows: index is [N] or [N, k] whole numbers, got {tuple(index.shape)} {index.dtype}")
    try:
        n_groups = operator.index(n_groups)
    except TypeError:
        raise ValueError(f"route_rows: n_groups is a whole number, got {n_groups!r}") from None
    if not 1 <= n_groups <= MAX_GROUPS:
        raise ValueError(f"route_rows: {n_groups} groups (1 to {MAX_GROUPS})")
    copies = 1 if index.dim() == 1 else index.shape[1]
    if copies < 1:
        raise ValueError("route_rows: index has no copies")
    if index.numel() > 0x7FFFFFFF:
        raise ValueError(f"route_rows: {index.numel()} pairs exceed 2^31 - 1")
    got = ordinary("route_rows", index.device, native().route, index.to(torch.int64).contiguous(), n_groups)
    return RowPlan(*got, n_groups, index.shape[0], copies)


def _check_rows(what: str, t: Tensor, rows: int, plan: RowPlan) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what}: midst_toolkit_amd has no CPU path; move the rows to the MI355X")
    if t.device != plan.order.device:
        raise ValueError(f"{what}: rows on {t.device}, plan on {plan.order.device}")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{what}: expected [{rows}, width] rows, got {tuple(t.shape)}")
    dtype_code(t, what)


def dispatch_rows(x: Tensor, plan: RowPlan) -> Tensor:
    """``x`` [N, D] -> [N * k, D]: every record's row in the places of its k pairs, sorted by model.  Differentiable in ``x`` (a record's
    gradient is the sum over its pairs, in fp32, in the order of its copies)."""
    if x.is_cuda:
        got = native().dispatch(x, plan.slot, plan.n_rows, plan.copies)
        if got is not None:
            return got
    _check_rows("dispatch_rows", x, plan.n_rows, plan)
    no_tangents("dispatch_rows", x)
    return ordinary("dispatch_rows", x.device, native().dispatch, rows_of(x), plan.slot, plan.n_rows, plan.copies)


def combine_rows(y: Tensor, plan: RowPlan, weights: Tensor | None = None) -> Tensor:
    """``y`` [N * k, D] in the plan's order -> [N, D]: ``sum_j weights[n, j] * y[slot[n, j]]`` (``weights`` None: ones), summed in fp32 and
    rounded once.  ``weights``: float32 of ``index``'s shape.  Differentiable in both."""
    if y.is_cuda:
        got = native().combine(y, plan.slot, plan.n_rows, plan.copies, weights)
        if got is not None:
            return got
    _check_rows("combine_rows", y, plan.n_rows * plan.copies, plan)
    no_tangents("combine_rows", y, weights)
    if weights is not None:
        if weights.device != y.device:
            raise ValueError(f"combine_rows: weights on {weights.device}, rows on {y.device}")
        if weights.dtype != torch.float32 or weights.numel() != plan.n_rows * plan.copies or weights.shape[:1] != (plan.n_rows,):
            raise ValueError(f"combine_rows: weights are float32 [{plan.n_rows}, {plan.copies}], got {weights.dtype} {tuple(weights.shape)}")
        weights = weights.reshape(plan.n_rows, plan.copies).contiguous()
    return ordinary("combine_rows", y.device, native().combine, rows_of(y), plan.slot, plan.n_rows, plan.copies, weights)
