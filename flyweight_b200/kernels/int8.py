"""Matrix products in 8-bit integers with a scale for every token's row and every channel's weights.

A model's matrix is laid out once (``matrix_int8``); in a step a token's row becomes integers (``rows_int8``, or with the RMS
norm in front of it ``rmsnorm_int8``) and goes through ``linear_int8`` (with the residual sum) or ``gated_int8`` (gate and up
projection, ``act(gate) * up``).  A weight is one byte instead of bfloat16's two, and the integer tensor cores do twice the
bfloat16 rate.  The integer sums are exact: a result does not depend on the kernel, the batch or a cut of the work.

    w_gate_up = int8.matrix_int8(torch.cat([gate, up]))           # [2 F][H] -> integers and F channels' scales, once
    a = int8.gated_int8(int8.rmsnorm_int8(x, norm, eps), w_gate_up)
    x = int8.linear_int8(a, w_down, torch.float32, addend=x, out=x)
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import lib
from .lib import KernelError, c_float, check_tensor, is_bf16, ptr, stream

MAX_COLUMNS = 131071          # 128 * 128 * K stays below 2^31


class Int8Rows:
    """Rows of integers: ``values`` int8 [R][stride], zero from column ``columns`` on (``stride``: the next multiple of 16),
    ``scales`` fp32 [R]; element (r, k) stands for ``values[r, k] * scales[r]``."""
    __slots__ = ("values", "scales", "columns")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, columns: int):
        self.values, self.scales, self.columns = values, scales, columns

    @property
    def shape(self):
        return (self.values.shape[0], self.columns)

    def float(self) -> torch.Tensor:
        """What the integers stand for, fp32 [R][columns]."""
        return self.values[:, :self.columns].float() * self.scales[:, None]


class Int8Matrix(Int8Rows):
    """A weight matrix [features][columns] as integers, a scale a feature."""
    __slots__ = ()


def _quantize(x: torch.Tensor, delta, norm, rows, eps: float, kind):
    K = x.shape[-1]
    R = rows.numel() if rows is not None else x.shape[0]
    stride = (K + 15) & ~15
    values = torch.empty((R, stride), dtype=torch.int8, device=x.device)
    scales = torch.empty(R, dtype=torch.float32, device=x.device)
    lib.call("fwb_rows_int8", ptr(x), is_bf16(x), ptr(delta), ptr(norm), ptr(rows), ptr(values), ptr(scales), R, K, stride,
             eps, stream())
    return kind(values, scales, K)


def _check_rows(name: str, x: torch.Tensor) -> None:
    check_tensor(name, x)
    is_bf16(x)
    if x.dim() != 2 or not 0 < x.shape[1] <= MAX_COLUMNS:
        raise KernelError(f"{name} must be [rows][1 to {MAX_COLUMNS} columns], got {tuple(x.shape)}")


def rows_int8(x: torch.Tensor) -> Int8Rows:
    """Every row of ``x`` ([R][K], bf16 or fp32) as integers of [-127, 127]: ``scale = max|x| / 127`` in fp32,
    ``value = round(x / scale)``, ties to even.  A row of zeros (nothing above 1e-30) has the scale 0; a row with an infinity
    or a NaN has the scale NaN."""
    _check_rows("rows", x)
    return _quantize(x, None, None, None, 0.0, Int8Rows)


def matrix_int8(w: torch.Tensor) -> Int8Matrix:
    """A weight matrix ([features][K], bf16 or fp32) laid out for the products, once: ``rows_int8`` of its features."""
    _check_rows("weight", w)
    made = _quantize(w, None, None, None, 0.0, Int8Matrix)
    # The products ask for weights before the kernel in front of them has ended.  A launch that is not overlapped with its
    # neighbours lies between the two from here on: the copy.
    made.scales = made.scales.clone()
    return made


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float, delta: Optional[torch.Tensor] = None,
                 rows: Optional[torch.Tensor] = None) -> Int8Rows:
    """``ops.rmsnorm`` whose rows leave as integers: ``(x / sqrt(mean(x^2) + eps)) * weight`` per row of the fp32 residual
    ``x``.  With ``delta`` the residual sum ``x += delta`` happens first, in place; with ``rows`` (int32) only those rows are
    normalised, into compact rows (not together with ``delta``)."""
    check_tensor("residual", x, torch.float32)
    _check_rows("residual", x)
    check_tensor("norm weight", weight, torch.float32, (x.shape[1],))
    if delta is not None:
        check_tensor("delta", delta, torch.float32, x.shape)
        if rows is not None:
            raise KernelError("a residual sum goes over every row: delta and rows exclude each other")
    if rows is not None:
        check_tensor("row indices", rows, torch.int32)
    return _quantize(x, delta, weight, rows, float(eps), Int8Rows)


def _operands(x, w):
    if not isinstance(w, Int8Matrix):
        raise KernelError("the weight must be an Int8Matrix (matrix_int8)")
    if not isinstance(x, Int8Rows):
        x = rows_int8(x)
    if x.columns != w.columns:
        raise KernelError(f"8-bit product: input has {x.columns} columns, weight has {w.columns}")
    return x


def _product(x: Int8Rows, w: Int8Matrix, out: torch.Tensor, addend, features: int, epilogue: int, limit: float = 0.0) -> None:
    xv, wv = x.values, w.values
    M = xv.shape[0]
    lib.call("fwb_gemm_int8", xv.data_ptr(), x.scales.data_ptr(), wv.data_ptr(), w.scales.data_ptr(), out.data_ptr(),
             ptr(addend), M, features, x.columns, xv.shape[1], wv.shape[1], wv.shape[0], epilogue, features, limit, stream())


def linear_int8(x: Union[Int8Rows, torch.Tensor], w: Int8Matrix, out_dtype: torch.dtype,
                addend: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T`` [M][N] in fp32 or bf16.  ``x``: integer rows, or a bf16/fp32 matrix, which is brought to integers first.
    ``addend`` (fp32 [M][N], with an fp32 result): added behind the scales; ``out`` may be the addend itself (a residual sum in
    place)."""
    x = _operands(x, w)
    shape = (x.values.shape[0], w.values.shape[0])
    if out_dtype is not torch.float32 and out_dtype is not torch.bfloat16:
        raise KernelError(f"an 8-bit product leaves as float32 or bfloat16, not {out_dtype}")
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=x.values.device)
    else:
        check_tensor("product output", out, out_dtype, shape)
    epilogue = 1 if out_dtype is torch.bfloat16 else 0
    if addend is not None:
        check_tensor("product addend", addend, torch.float32, shape)
        if epilogue:
            raise KernelError("an addend needs a float32 result")
        epilogue = 2
    _product(x, w, out, addend, shape[1], epilogue)
    return out


def gated_int8(x: Union[Int8Rows, torch.Tensor], w: Int8Matrix, activation: str = "silu", limit: float = 0.0) -> torch.Tensor:
    """``act(x @ gate.T) * (x @ up.T)`` as bf16 [M][F], ``w`` holding the F gate rows and then the F up rows; activations as
    ``ops.gate_act_mul``."""
    from .ops import GATE_ACTIVATIONS
    x = _operands(x, w)
    try:
        act = GATE_ACTIVATIONS[activation]
    except KeyError:
        raise KernelError(f"unknown gate activation {activation!r}; known: " + ", ".join(GATE_ACTIVATIONS)) from None
    rows = w.values.shape[0]
    if rows % 2:
        raise KernelError("gate|up needs an even number of rows")
    out = torch.empty((x.values.shape[0], rows // 2), dtype=torch.bfloat16, device=x.values.device)
    _product(x, w, out, None, rows // 2, 3 | act << 8, float(limit))
    return out
