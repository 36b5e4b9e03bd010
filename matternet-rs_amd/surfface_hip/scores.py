"""Item scores in 8 bits: a table kept as int8 rows with a scale each, and the
scores of quantised queries against it (mn_quantize_rows_i8, mn_scores_i8).

Stands beside knn_cos_bf16_qc and search_lambda_aware for tables that are kept
at a quarter of their f32 size.  Has no counterpart in the reference.

The calls only enqueue on the stream (default: the current one) and can be
captured into a graph.  With `stream` given the caller orders it after the work
that made the inputs, as with torch.cuda.stream(stream).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._torch import enqueues, raw_stream, require_aligned, require_cuda

VALUE_TYPES = {torch.float32: _lib.MN_F32, torch.bfloat16: _lib.MN_BF16}


def row_stride(d: int) -> int:
    """Bytes from one row of codes to the next: whole pieces of 16."""
    return (d + 15) // 16 * 16


@dataclass
class Int8Rows:
    """n rows of d values in 8 bits: value = codes[:, :d] * scale[:, None].

    codes [n, ld] int8 with ld a multiple of 16 (row_stride(d), say); what
    lies behind column d has no effect.  scale [n] f32."""
    codes: torch.Tensor
    scale: torch.Tensor
    d: int

    def __len__(self) -> int:
        return self.codes.shape[0]


def _rows(r: Int8Rows, name: str, device=None):
    if not isinstance(r, Int8Rows):
        raise TypeError(f"{name} must be Int8Rows (quantize_rows)")
    codes = require_aligned(r.codes, torch.int8, f"{name}.codes", 2, device)
    scale = require_aligned(r.scale, torch.float32, f"{name}.scale", 1, codes.device)
    n, ld = codes.shape
    if scale.shape[0] != n:
        raise ValueError(f"{name} has {n} rows and {scale.shape[0]} scales")
    if r.d < 1 or ld < r.d or ld % 16:
        raise ValueError(f"{name}.codes needs rows of at least d = {r.d} bytes and a multiple of 16, got {ld}")
    return codes, scale, n, ld


@enqueues
def quantize_rows(X: torch.Tensor) -> Int8Rows:
    """Rows of X [n, d] (f32 or bf16) in 8 bits: scale = max|x| / 127, code =
    rint(x (127 (1 / max|x|))).  A row of zeros gets scale 0; a row that holds an
    infinity or a NaN gets scale NaN, which every score with it shows."""
    if not isinstance(X, torch.Tensor) or X.dtype not in VALUE_TYPES:
        raise TypeError("X must be a float32 or bfloat16 tensor")
    x = require_cuda(X, X.dtype, "X", 2)
    n, d = x.shape
    if d < 1:
        raise ValueError("X has no columns")
    ld = row_stride(d)
    codes = torch.empty((n, ld), dtype=torch.int8, device=x.device)
    scale = torch.empty(n, dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().mn_quantize_rows_i8(x.data_ptr(), VALUE_TYPES[x.dtype], n, d, codes.data_ptr(), ld,
                                              scale.data_ptr(), raw_stream(x)))
    return Int8Rows(codes, scale, d)


@enqueues
def dequantize_rows(rows: Int8Rows, dtype=torch.float32) -> torch.Tensor:
    """The values [n, d] that the codes stand for, as f32 or rounded to bf16."""
    if dtype not in VALUE_TYPES:
        raise TypeError("dtype must be float32 or bfloat16")
    codes, scale, n, ld = _rows(rows, "rows")
    X = torch.empty((n, rows.d), dtype=dtype, device=codes.device)
    _lib.check(_lib.lib().mn_dequantize_rows_i8(codes.data_ptr(), ld, scale.data_ptr(), n, rows.d, X.data_ptr(),
                                                VALUE_TYPES[dtype], raw_stream(X)))
    return X


@enqueues
def scores_i8(queries: Int8Rows, items: Int8Rows, dtype=torch.float32) -> torch.Tensor:
    """[m, n] scores of every query with every item: the int8 product (exact
    sums, d <= 131071) times the query's and the item's scale, f32 or rounded
    to bf16."""
    if dtype not in VALUE_TYPES:
        raise TypeError("dtype must be float32 or bfloat16")
    c, cs, n, ldc = _rows(items, "items")
    q, qs, m, ldq = _rows(queries, "queries", c.device)
    d = queries.d
    if d != items.d:
        raise ValueError(f"queries have {d} columns, items {items.d}")
    L = _lib.lib()
    need = 0
    if d % 64 and m:  # whole k-steps need no workspace
        b = C.c_size_t()
        _lib.check(L.mn_scores_i8_workspace(m, d, C.byref(b)))
        need = b.value
    ws = torch.empty(need, dtype=torch.int8, device=c.device) if need else None
    Y = torch.empty((m, n), dtype=dtype, device=c.device)
    _lib.check(L.mn_scores_i8(q.data_ptr(), ldq, qs.data_ptr(), m, c.data_ptr(), ldc, cs.data_ptr(), n, d,
                              Y.data_ptr(), VALUE_TYPES[dtype], ws.data_ptr() if need else None, need,
                              raw_stream(Y)))
    return Y
