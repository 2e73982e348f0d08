"""Matrix products in 8-bit integers with a scale for every row of both sides (tokens and channels), for projections whose weights are not ternary -- the
vocabulary's above all, which a decode step reads whole.  Kernels and the layout of packed rows: csrc/int8_linear_kernel.h.

Tensors of one GPU, which need not be the current one; calls enqueue on that GPU's current stream and raise ValueError (TypeError where an argument is no
tensor) for what the kernels do not take, before anything is enqueued.  No backward pass.
"""
from __future__ import annotations

from typing import NamedTuple, Union

import torch

from . import _lib


class Int8Rows(NamedTuple):
    """Rows in 8 bits, in the order in which the product reads them (see include/ternaspmm.h): row r stands for scale[r] * integers."""
    packed: torch.Tensor
    scale: torch.Tensor
    rows: int
    columns: int


def quantise_rows(x: torch.Tensor) -> Int8Rows:
    """x [R, K] (bfloat16 or float32, rows any distance apart; K up to 131056): scale = max|x| / 127 of every row, integers rint(x * (127 / max|x|)), ties to
    even.  A row whose magnitudes all lie below 2^-120 is zeros; one with NaN or an infinity has the scale NaN."""
    packed, scale = _lib.native().int8_quantise(x)
    return Int8Rows(packed, scale, *x.shape)


def int8_rows(q: torch.Tensor, scale: torch.Tensor) -> Int8Rows:
    """Rows that are integers already: q int8 [R, K], scale float32 [R]."""
    if not isinstance(q, torch.Tensor) or not isinstance(scale, torch.Tensor):
        raise TypeError("int8_rows: rows and scales are tensors")
    if scale.dtype != torch.float32 or scale.shape != q.shape[:1] or scale.device != q.device:
        raise ValueError("int8_rows: scale is float32 [R] beside the rows")
    return Int8Rows(_lib.native().int8_pack(q), scale.contiguous(), *q.shape)


def int8_linear(x: Union[torch.Tensor, Int8Rows], weight: Int8Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """x [M, K] times the weights [N, K] transposed: [M, N] in bfloat16 or float32, float(sum x w) * x.scale[m] * weight.scale[n], the sums exact.  x in
    bfloat16 or float32 is quantised as by `quantise_rows`, in the call."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"int8_linear: results in bfloat16 or float32, not {dtype}")
    if not isinstance(weight, Int8Rows):
        raise TypeError("int8_linear: the weights are Int8Rows")
    if isinstance(x, Int8Rows):
        if x.columns != weight.columns:
            raise ValueError(f"int8_linear: x has {x.columns} columns, the weights {weight.columns}")
        return _lib.native().int8_linear(x.packed, x.scale, x.rows, weight.packed, weight.scale, weight.rows, weight.columns, dtype == torch.float32)
    return _lib.native().int8_linear(x, None, 0, weight.packed, weight.scale, weight.rows, weight.columns, dtype == torch.float32)
