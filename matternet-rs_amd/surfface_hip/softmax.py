"""Softmax cross entropy of queries over the rows of an item table, and its
gradients (mn_softmax_stats, mn_softmax_backward): the loss with which the
vectors that this package searches are learnt.  The table is taken in pieces;
no [t, v] matrix of logits is kept.  Has no counterpart in the reference.

softmax_loss is the whole of it with autograd.  softmax_stats, softmax_merge
and softmax_backward are its parts, for tables whose rows are spread over
processes (c_offset, as in knn_l2sq_qc) and for steps captured into a graph.
softmax_loss with gradients is refused in a capture, and so is its backward pass
on a stream that is being captured: a backward pass of autograd that is captured
while an eager graph of the same leaves lives ends the process.

The calls only enqueue on the stream (default: the current one).  With `stream`
given the caller orders it after the work that made the inputs, as with
torch.cuda.stream(stream).

Values of items and of queries that take part have to be finite (else what they
meet is NaN); an item that holds the type's lowest value where the queries are
positive is masked out: its logit is far below all others.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._torch import enqueues, raw_stream, require_aligned, require_cuda
from .scores import VALUE_TYPES


@dataclass
class SoftmaxStats:
    """Per query: rest = log sum exp of the logits but the target's, target =
    the target's logit (-inf where it is not among the rows), loss.  mean = the
    mean of loss over the queries that take part, share [1] = 1 / their number."""
    rest: torch.Tensor
    target: torch.Tensor
    loss: torch.Tensor
    mean: torch.Tensor
    share: torch.Tensor


def _inputs(Q, items, targets):
    if not isinstance(Q, torch.Tensor) or Q.dtype not in VALUE_TYPES:
        raise TypeError("queries must be a float32 or bfloat16 tensor")
    q = require_aligned(Q, Q.dtype, "queries", 2)
    c = require_aligned(items, Q.dtype, "items", 2, q.device)
    if isinstance(targets, torch.Tensor) and targets.dtype == torch.int32:
        targets = targets.long()
    t = require_aligned(targets, torch.int64, "targets", 1, q.device)
    n, d = q.shape
    v = c.shape[0]
    if c.shape[1] != d:
        raise ValueError(f"queries have {d} columns, items {c.shape[1]}")
    if t.shape[0] != n:
        raise ValueError(f"{n} queries and {t.shape[0]} targets")
    if v < 1 or d < 1:
        raise ValueError("items has no rows or no columns")
    return q, c, t, n, v, d, VALUE_TYPES[Q.dtype]


def _values(x, name, device, *sizes):
    """A dense f32 vector of one of these sizes."""
    x = require_cuda(x.reshape(-1), torch.float32, name)
    if x.shape[0] not in sizes:
        raise ValueError(f"{name} needs {' or '.join(map(str, sizes))} values, got {x.shape[0]}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, other tensors of the call on {device}")
    return x


def _workspace(L, n, v, d, kind, backward, device):
    need = C.c_size_t()
    _lib.check(L.mn_softmax_workspace(n, v, d, kind, backward, C.byref(need)))
    return torch.empty(need.value, dtype=torch.int8, device=device)


def _stats_out(n, device):
    f = lambda *shape: torch.empty(shape, dtype=torch.float32, device=device)
    # tensors of their own: the caller may change loss and mean in place
    st = SoftmaxStats(f(n), f(n), f(n), f(), f(1))
    return st, [x.data_ptr() for x in (st.rest, st.target, st.loss, st.mean, st.share)]


@enqueues
def softmax_stats(queries: torch.Tensor, items: torch.Tensor, targets: torch.Tensor, scale: float = 1.0,
                  c_offset: int = 0) -> SoftmaxStats:
    """queries [t, d], items [v, d] (f32 or bf16), targets [t] (int64 or int32,
    global row ids; negative: the query has no part); logits scale q.c, scale >
    0.  items holds the rows c_offset .. c_offset + v - 1 of the table; a target
    among none of a table's rows makes its loss +inf."""
    return _stats(_inputs(queries, items, targets), scale, c_offset)


def _stats(inputs, scale, c_offset):
    q, c, t, n, v, d, kind = inputs
    st, out = _stats_out(n, q.device)
    L = _lib.lib()
    ws = _workspace(L, n, v, d, kind, 0, q.device)
    _lib.check(L.mn_softmax_stats(q.data_ptr(), c.data_ptr(), kind, n, v, d, t.data_ptr(), c_offset, float(scale),
                                  *out, ws.data_ptr(), ws.numel(), raw_stream(q)))
    return st


@enqueues
def softmax_merge(rests: torch.Tensor, zts: torch.Tensor, targets: torch.Tensor) -> SoftmaxStats:
    """The stats of a whole table from those of its row ranges: rests and zts
    [parts, t] (softmax_stats' rest and target, gathered over the ranges)."""
    r = require_aligned(rests, torch.float32, "rests", 2)
    z = require_aligned(zts, torch.float32, "zts", 2, r.device)
    if isinstance(targets, torch.Tensor) and targets.dtype == torch.int32:
        targets = targets.long()
    t = require_aligned(targets, torch.int64, "targets", 1, r.device)
    parts, n = r.shape
    if r.shape != z.shape or n != t.shape[0] or parts < 1:
        raise ValueError(f"rests {tuple(r.shape)}, zts {tuple(z.shape)} and targets {tuple(t.shape)} do not fit")
    st, out = _stats_out(n, r.device)
    _lib.check(_lib.lib().mn_softmax_merge(r.data_ptr(), z.data_ptr(), parts, n, t.data_ptr(), *out,
                                           raw_stream(r)))
    return st


@enqueues
def softmax_backward(queries: torch.Tensor, items: torch.Tensor, targets: torch.Tensor, rest: torch.Tensor,
                     target: torch.Tensor, grad: torch.Tensor, scale: float = 1.0, c_offset: int = 0,
                     grad_scale: torch.Tensor | None = None, need=(True, True)):
    """(d queries, d items) of sum(grad * loss), from the WHOLE table's rest and
    target (softmax_stats, or softmax_merge where items is a row range: then d
    queries is the range's part, to be added up).  grad: f32, one value per
    query or one for all; grad_scale: one f32 that multiplies it (share for
    the mean).  need: which of the two to compute (None for the other)."""
    q, c, t, n, v, d, kind = _inputs(queries, items, targets)
    re = _values(rest, "rest", q.device, n)
    zt = _values(target, "target", q.device, n)
    g = _values(grad, "grad", q.device, 1, n)
    gs = None if grad_scale is None else _values(grad_scale, "grad_scale", q.device, 1)
    return _backward(q, c, t, n, v, d, kind, re, zt, g, scale, c_offset, gs, need)


def _backward(q, c, t, n, v, d, kind, re, zt, g, scale, c_offset, gs, need):
    dq = torch.empty_like(q) if need[0] else None
    dc = torch.empty_like(c) if need[1] else None
    if n == 0:
        return dq, dc.zero_() if need[1] else None
    if need[0] or need[1]:
        L = _lib.lib()
        ws = _workspace(L, n, v, d, kind, 1, q.device)
        _lib.check(L.mn_softmax_backward(
            q.data_ptr(), c.data_ptr(), kind, n, v, d, t.data_ptr(), c_offset, float(scale), re.data_ptr(),
            zt.data_ptr(), g.data_ptr(), g.shape[0], None if gs is None else gs.data_ptr(),
            dq.data_ptr() if need[0] else None, dc.data_ptr() if need[1] else None, ws.data_ptr(), ws.numel(),
            raw_stream(q)))
    return dq, dc


class _SoftmaxLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, queries, items, targets, scale, reduction):
        inputs = _inputs(queries, items, targets)
        st = _stats(inputs, scale, 0)
        ctx.save_for_backward(queries, items, targets)
        # what the caller may change in place (loss, mean) is not kept, nor is
        # a dense copy of an input
        same = inputs[0] is queries and inputs[1] is items and inputs[2] is targets
        ctx.of = (inputs[3:] if same else None, st.rest, st.target, st.share if reduction == "mean" else None, scale)
        if reduction == "sum":  # (torch's sum over many blocks cannot be captured)
            return st.mean / st.share[0]
        return st.mean if reduction == "mean" else st.loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if torch.cuda.is_current_stream_capturing():  # the loss was computed on this stream before
            raise RuntimeError("softmax_loss's backward pass in a graph capture: capture softmax_stats and softmax_backward")
        tensors = ctx.saved_tensors
        sizes, rest, target, share, scale = ctx.of
        inputs = (*tensors, *sizes) if sizes else _inputs(*tensors)
        dq, dc = _backward(*inputs, rest, target, grad.reshape(-1).contiguous(), scale, 0, share,
                           ctx.needs_input_grad[:2])
        return dq, dc, None, None, None


@enqueues
def softmax_loss(queries: torch.Tensor, items: torch.Tensor, targets: torch.Tensor, scale: float = 1.0,
                 reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of queries [t, d] over all rows of items [v, d]
    (f32 or bf16) with logits scale q.c, f32; differentiable once in queries
    and items.  targets [t]: row ids, negative: the query has no part (loss 0,
    gradient 0).  reduction: "mean" over the queries that take part (0 when
    there is none), "sum" or "none".  In a graph capture only without gradients
    (else RuntimeError): capture softmax_stats and softmax_backward.  A step of
    few rows is bound by the host: 130 us, 68 inside
    torch.autograd.set_multithreading_enabled(False), 49 with those two."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none'")
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad and x.is_cuda
                                       for x in (queries, items)) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("softmax_loss with gradients in a graph capture: capture softmax_stats and softmax_backward")
    return _SoftmaxLoss.apply(queries, items, targets, float(scale), reduction)
