"""Softmax cross entropy of queries over the rows of an item table, and its
gradients (mn_softmax_stats, mn_softmax_backward): the loss with which the
vectors that this package searches are learnt.  The table is taken in pieces;
no [t, v] matrix of logits is kept.  Has no counterpart in the reference.

softmax_loss is the whole of it with autograd.  softmax_stats, softmax_merge
and softmax_backward are its parts, for tables whose rows are spread over
processes (c_offset, as in knn_l2sq_qc) and for steps captured into a graph.
Capture those: a backward pass of autograd that is captured while an eager
graph of the same leaves lives ends the process (torch's own rule).

The calls only enqueue on the stream (default: the current one).  With `stream`
given the caller orders it after the work that made the inputs, as with
torch.cuda.stream(stream).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._torch import enqueue, on_device, ptr, require_aligned, stream_handle
from .scores import VALUE_TYPES


@dataclass
class SoftmaxStats:
    """Per query: rest = log sum exp of the logits but the target's, target =
    the target's logit (-inf where it is not among the rows), loss.  mean [2] =
    the mean of loss over the queries that take part, 1 / their number."""
    rest: torch.Tensor
    target: torch.Tensor
    loss: torch.Tensor
    mean: torch.Tensor


def _inputs(Q, items, targets):
    if not isinstance(Q, torch.Tensor) or Q.dtype not in VALUE_TYPES:
        raise TypeError("queries must be a float32 or bfloat16 tensor")
    q = require_aligned(Q, Q.dtype, "queries", 2)
    c = require_aligned(items, Q.dtype, "items", 2)
    if isinstance(targets, torch.Tensor) and targets.dtype == torch.int32:
        targets = targets.long()
    t = require_aligned(targets, torch.int64, "targets", 1)
    if q.shape[1] != c.shape[1]:
        raise ValueError(f"queries have {q.shape[1]} columns, items {c.shape[1]}")
    if t.shape[0] != q.shape[0]:
        raise ValueError(f"{q.shape[0]} queries and {t.shape[0]} targets")
    if c.shape[0] < 1 or c.shape[1] < 1:
        raise ValueError("items has no rows or no columns")
    if not q.device == c.device == t.device:
        raise ValueError("queries, items and targets must be on one device")
    return q, c, t


def _workspace(q, c, backward):
    need = C.c_size_t()
    _lib.check(_lib.lib().mn_softmax_workspace(q.shape[0], c.shape[0], q.shape[1], VALUE_TYPES[q.dtype],
                                               backward, C.byref(need)))
    return torch.empty(need.value, dtype=torch.int8, device=q.device)


@on_device
def softmax_stats(queries: torch.Tensor, items: torch.Tensor, targets: torch.Tensor, scale: float = 1.0,
                  c_offset: int = 0, stream=None) -> SoftmaxStats:
    """queries [t, d], items [v, d] (f32 or bf16), targets [t] (int64 or int32,
    global row ids; negative: the query has no part); logits scale q.c, scale >
    0.  items holds the rows c_offset .. c_offset + v - 1 of the table; a target
    among none of a table's rows makes its loss +inf."""
    with enqueue(stream, queries, items, targets):
        q, c, t = _inputs(queries, items, targets)
        out = torch.empty((3, q.shape[0]), dtype=torch.float32, device=q.device)
        mean = torch.empty(2, dtype=torch.float32, device=q.device)
        ws = _workspace(q, c, 0)
        _lib.check(_lib.lib().mn_softmax_stats(
            ptr(q), ptr(c), VALUE_TYPES[q.dtype], q.shape[0], c.shape[0], q.shape[1], ptr(t), c_offset,
            float(scale), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(mean), ptr(ws), ws.numel(),
            stream_handle()))
    return SoftmaxStats(out[0], out[1], out[2], mean)


@on_device
def softmax_merge(rests: torch.Tensor, zts: torch.Tensor, targets: torch.Tensor, stream=None) -> SoftmaxStats:
    """The stats of a whole table from those of its row ranges: rests and zts
    [parts, t] (softmax_stats' rest and target, gathered over the ranges)."""
    with enqueue(stream, rests, zts, targets):
        r = require_aligned(rests, torch.float32, "rests", 2)
        z = require_aligned(zts, torch.float32, "zts", 2)
        t = require_aligned(targets.long(), torch.int64, "targets", 1)
        if r.shape != z.shape or r.shape[1] != t.shape[0] or r.shape[0] < 1:
            raise ValueError(f"rests {tuple(r.shape)}, zts {tuple(z.shape)} and targets {tuple(t.shape)} do not fit")
        out = torch.empty((3, t.shape[0]), dtype=torch.float32, device=r.device)
        mean = torch.empty(2, dtype=torch.float32, device=r.device)
        _lib.check(_lib.lib().mn_softmax_merge(ptr(r), ptr(z), r.shape[0], t.shape[0], ptr(t), ptr(out[0]),
                                               ptr(out[1]), ptr(out[2]), ptr(mean), stream_handle()))
    return SoftmaxStats(out[0], out[1], out[2], mean)


@on_device
def softmax_backward(queries: torch.Tensor, items: torch.Tensor, targets: torch.Tensor, rest: torch.Tensor,
                     target: torch.Tensor, grad: torch.Tensor, scale: float = 1.0, c_offset: int = 0,
                     grad_scale: torch.Tensor | None = None, need=(True, True), stream=None):
    """(d queries, d items) of sum(grad * loss), from the WHOLE table's rest and
    target (softmax_stats, or softmax_merge where items is a row range: then d
    queries is the range's part, to be added up).  grad: f32, one value per
    query or one for all; grad_scale: one f32 that multiplies it (mean[1] for
    the mean).  need: which of the two to compute (None for the other)."""
    with enqueue(stream, queries, items, targets, rest, target, grad, grad_scale):
        q, c, t = _inputs(queries, items, targets)
        n = q.shape[0]
        re = require_aligned(rest, torch.float32, "rest", 1)
        zt = require_aligned(target, torch.float32, "target", 1)
        g = require_aligned(grad.reshape(-1), torch.float32, "grad", 1)
        if re.shape[0] != n or zt.shape[0] != n:
            raise ValueError(f"rest and target need {n} values")
        if g.shape[0] not in (1, n):
            raise ValueError(f"grad needs 1 or {n} values, got {g.shape[0]}")
        gs = None
        if grad_scale is not None:
            gs = require_aligned(grad_scale.reshape(-1), torch.float32, "grad_scale", 1)
            if gs.shape[0] != 1:
                raise ValueError("grad_scale needs one value")
        dq = torch.empty_like(q) if need[0] else None
        dc = torch.empty_like(c) if need[1] else None
        if n == 0:
            return dq, dc.zero_() if need[1] else None
        if need[0] or need[1]:
            ws = _workspace(q, c, 1)
            _lib.check(_lib.lib().mn_softmax_backward(
                ptr(q), ptr(c), VALUE_TYPES[q.dtype], n, c.shape[0], q.shape[1], ptr(t), c_offset, float(scale),
                ptr(re), ptr(zt), ptr(g), g.shape[0], ptr(gs) if gs is not None else None,
                ptr(dq) if need[0] else None, ptr(dc) if need[1] else None, ptr(ws), ws.numel(),
                stream_handle()))
    return dq, dc


class _SoftmaxLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, items, targets, scale, reduction):
        st = softmax_stats(queries, items, targets, scale)
        ctx.save_for_backward(queries, items, targets, st.rest, st.target, st.mean)
        ctx.scale, ctx.reduction = scale, reduction
        if reduction == "mean":
            return st.mean[0].clone()
        return st.loss if reduction == "none" else st.loss.sum()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        queries, items, targets, rest, target, mean = ctx.saved_tensors
        dq, dc = softmax_backward(queries, items, targets, rest, target, grad, ctx.scale,
                                  grad_scale=mean[1] if ctx.reduction == "mean" else None,
                                  need=ctx.needs_input_grad[:2])
        return dq, dc, None, None, None


@on_device
def softmax_loss(queries: torch.Tensor, items: torch.Tensor, targets: torch.Tensor, scale: float = 1.0,
                 reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of queries [t, d] over all rows of items [v, d]
    (f32 or bf16) with logits scale q.c, f32; differentiable once in queries
    and items.  targets [t]: row ids, negative: the query has no part (loss 0,
    gradient 0).  reduction: "mean" over the queries that take part (0 when
    there is none), "sum" or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none'")
    return _SoftmaxLoss.apply(queries, items, targets, float(scale), reduction)
