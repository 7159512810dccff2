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
from .lib import KernelError, check_tensor
from .ops import GATE_ACTIVATIONS

MAX_COLUMNS = 131071          # 128 * 128 * K stays below 2^31
# up to here the product brings rows to integers by itself, in one launch (one token, 2048 x 2048, with its host time 14.1 -> 11.2 us;
# every block does it, so with more tokens or columns a launch of its own is faster); the kernel refuses more (int8_product.cuh)
MAX_RAW, MAX_RAW_COLUMNS = 8, 4096
_FP32, _BF16 = torch.float32, torch.bfloat16


class Int8Rows:
    """Rows of integers with a scale each: element (r, k) stands for ``values[r, k] * scales[r]``.  ``values``: int8 [R][stride],
    zero from column ``columns`` on (``stride``: the next multiple of 16); ``scales``: fp32 [R].  One buffer holds both."""
    __slots__ = ("_buffer", "_rows", "columns", "_stride", "_address", "_scales")

    def __init__(self, buffer: torch.Tensor, rows: int, columns: int):
        self._buffer, self._rows, self.columns = buffer, rows, columns
        self._stride = (columns + 15) & ~15
        self._address = buffer.data_ptr()
        self._scales = self._address + rows * self._stride

    @property
    def shape(self):
        return (self._rows, self.columns)

    @property
    def device(self):
        return self._buffer.device

    @property
    def values(self) -> torch.Tensor:
        return self._buffer[:self._rows * self._stride].view(torch.int8).view(self._rows, self._stride)

    @property
    def scales(self) -> torch.Tensor:
        return self._buffer[self._rows * self._stride:].view(_FP32)

    def float(self) -> torch.Tensor:
        """What the integers stand for, fp32 [R][columns]."""
        return self.values[:, :self.columns].float() * self.scales[:, None]


class Int8Matrix(Int8Rows):
    """A weight matrix [features][columns] as integers, a scale a feature."""
    __slots__ = ()


def _input(name: str, x: torch.Tensor) -> int:
    """Checks of a matrix that becomes integers; 1 for bfloat16, 0 for float32."""
    dtype = x.dtype
    if x.dim() != 2 or not x.is_contiguous() or not x.is_cuda or (dtype is not _BF16 and dtype is not _FP32):
        check_tensor(name, x)
        raise KernelError(f"{name} must be a float32 or bfloat16 matrix, got {dtype} {tuple(x.shape)}")
    if not 0 < x.shape[1] <= MAX_COLUMNS:
        raise KernelError(f"{name} must have 1 to {MAX_COLUMNS} columns, got {x.shape[1]}")
    _here(name, x)
    return 1 if dtype is _BF16 else 0


def _here(name: str, x: torch.Tensor) -> None:
    if x.get_device() != lib._device_index():
        raise KernelError(f"{name} is on {x.device}, the kernels are launched on cuda:{lib._device_index()}")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    start, other = a.data_ptr(), b.data_ptr()
    return start < other + b.numel() * b.element_size() and other < start + a.numel() * a.element_size()


def _scratch(rows: int, columns: int, device) -> torch.Tensor:
    return torch.empty(rows * (((columns + 15) & ~15) + 4), dtype=torch.uint8, device=device)


def _quantize(x: torch.Tensor, is_bf16: int, delta, norm, rows, eps: float, kind):
    K = x.shape[1]
    R = rows.numel() if rows is not None else x.shape[0]
    made = kind(_scratch(R, K, x.device), R, K)
    lib.call("fwb_rows_int8", x.data_ptr(), is_bf16, lib.ptr(delta), lib.ptr(norm), lib.ptr(rows), made._address, made._scales, R, K,
             made._stride, x.shape[0], eps, lib.stream())
    return made


def rows_int8(x: torch.Tensor) -> Int8Rows:
    """Every row of ``x`` ([R][K], bf16 or fp32) as integers of [-127, 127]: ``scale = max|x| / 127`` in fp32,
    ``value = round(x / scale)``, ties to even.  A row of zeros (nothing from 127 * 2^-125 = 3e-36 on) has the scale 0; a row
    with an infinity or a NaN has the scale NaN, and what is made of it is NaN."""
    return _quantize(x, _input("rows", x), None, None, None, 0.0, Int8Rows)


def matrix_int8(w: torch.Tensor) -> Int8Matrix:
    """A weight matrix ([features][K], bf16 or fp32) laid out for the products, once: ``rows_int8`` of its features."""
    made = _quantize(w, _input("weight", w), None, None, None, 0.0, Int8Matrix)
    # The products ask for weights before the kernel in front of them has ended.  A launch that does not overlap its
    # neighbours lies between the two from here on.
    made._buffer.new_ones(1)
    return made


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float, delta: Optional[torch.Tensor] = None,
                 rows: Optional[torch.Tensor] = None) -> Int8Rows:
    """``ops.rmsnorm`` whose rows leave as integers: ``(x / sqrt(mean(x^2) + eps)) * weight`` per row of the fp32 residual
    ``x``.  With ``delta`` the residual sum ``x += delta`` happens first, in place; with ``rows`` (int32) only those rows are
    normalised, into compact rows (not together with ``delta``); an index that is no row of ``x`` gives a row of zeros."""
    if _input("residual", x):
        raise KernelError("the residual must be float32")
    check_tensor("norm weight", weight, _FP32, (x.shape[1],))
    _here("norm weight", weight)
    if delta is not None:
        check_tensor("delta", delta, _FP32, x.shape)
        _here("delta", delta)
        if rows is not None:
            raise KernelError("a residual sum goes over every row: delta and rows exclude each other")
    if rows is not None:
        check_tensor("row indices", rows, torch.int32)
        _here("row indices", rows)
    return _quantize(x, 0, delta, weight, rows, float(eps), Int8Rows)


def _product(x: Int8Rows, w: Int8Matrix, out: torch.Tensor, addend, features: int, epilogue: int, limit: float = 0.0,
             tile: int = 0, splits: int = 1) -> None:
    lib.call("fwb_gemm_int8", x._address, x._scales, w._address, w._scales, out.data_ptr(), lib.ptr(addend), x._rows, features,
             x.columns, x._stride, w._stride, w._rows, epilogue, features, limit, tile, splits, lib.stream())


def _run(x, w: Int8Matrix, out, out_dtype, addend, features: int, epilogue: int, limit: float) -> torch.Tensor:
    if type(w) is not Int8Matrix:
        raise KernelError("the weight must be an Int8Matrix (matrix_int8)")
    ready = isinstance(x, Int8Rows)
    is_bf16 = 0 if ready else _input("rows", x)
    M, K = x.shape
    if K != w.columns:
        raise KernelError(f"8-bit product: input has {K} columns, weight has {w.columns}")
    _here("weight", w._buffer)
    if addend is not None:
        check_tensor("product addend", addend, _FP32, (M, features))
        _here("product addend", addend)
        if out is None:
            out = torch.empty_like(addend)
    if out is None:
        out = torch.empty((M, features), dtype=out_dtype, device=w._buffer.device)
    elif out is not addend:
        check_tensor("product output", out, out_dtype, (M, features))
        _here("product output", out)
    if ready:
        _here("rows", x._buffer)
        _product(x, w, out, addend, features, epilogue, limit)
    else:
        address, scratch = x.data_ptr(), None
        # (a result over its own input: every block reads all of a row, so the integers are made first)
        if M > MAX_RAW or K > MAX_RAW_COLUMNS or K & 7 or address & 15 or _overlap(x, out):
            held = _scratch(M, K, w._buffer.device)
            scratch = held.data_ptr()
        lib.call("fwb_linear_int8", address, is_bf16, scratch, w._address, w._scales, out.data_ptr(),
                 lib.ptr(addend), M, features, K, w._stride, w._rows, epilogue, features, limit, lib.stream(), launches=2 if scratch else 1)
    return out


def linear_int8(x: Union[Int8Rows, torch.Tensor], w: Int8Matrix, out_dtype: torch.dtype,
                addend: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T`` [M][N] in fp32 or bf16.  ``x``: integer rows, or a bf16/fp32 matrix, which is brought to integers first.
    ``addend`` (fp32 [M][N], with an fp32 result): added behind the scales; ``out`` may be the addend itself (a residual sum in
    place) or the matrix ``x``."""
    if out_dtype is _FP32:
        epilogue = 0 if addend is None else 2
    elif out_dtype is not _BF16:
        raise KernelError(f"an 8-bit product leaves as float32 or bfloat16, not {out_dtype}")
    elif addend is not None:
        raise KernelError("an addend needs a float32 result")
    else:
        epilogue = 1
    return _run(x, w, out, out_dtype, addend, getattr(w, "_rows", 0), epilogue, 0.0)


def gated_int8(x: Union[Int8Rows, torch.Tensor], w: Int8Matrix, activation: str = "silu", limit: float = 0.0) -> torch.Tensor:
    """``act(x @ gate.T) * (x @ up.T)`` as bf16 [M][F], ``w`` holding the F gate rows and then the F up rows; activations as
    ``ops.gate_act_mul``."""
    act = GATE_ACTIVATIONS.get(activation)
    if act is None:
        raise KernelError(f"unknown gate activation {activation!r}; known: " + ", ".join(GATE_ACTIVATIONS))
    rows = getattr(w, "_rows", 0)
    if rows % 2:
        raise KernelError("gate|up needs an even number of rows")
    return _run(x, w, None, _BF16, None, rows // 2, 3 | act << 8, limit)
