"""Products of a few tokens with INT4 weights: 4-bit codes with a scale and a zero point per group of columns, as AWQ checkpoints have them.

``from_parts`` lays a weight out once, when it is loaded; ``linear`` multiplies the tokens of a step by it.  A value is ``(code - zero) * scale``: codes minus
zero points are whole numbers, which the tensor cores multiply exactly, and scales are applied in FP32, so that nothing is rounded before the result.

Calls are asynchronous on the current CUDA stream of their inputs' device, keep nothing, and may be made from any thread or captured in a graph
(``from_parts`` waits for its checks, and may not).  Inference only: nothing here has a gradient.  There is no CPU path.  The reference decodes INT4
weights to BF16 and multiplies those.
"""
from __future__ import annotations

import torch

from . import _lib
from .mx4 import _DTYPES, _current_device, _launch, _matrix, _stream_of, _workspace

__all__ = ["Int4Tensor", "from_parts", "dequantize", "linear"]

GROUPS = (32, 64, 128)
_HALVES = {torch.bfloat16: 0, torch.float16: 1}
_MOST_ROWS, _MOST_COLS, _MOST_TOKENS = 1 << 27, 1 << 24, 1 << 21


def _bytes(rows: int, cols: int, group: int) -> int:
    return (rows + 127) // 128 * ((cols + 127) // 128) * (8192 + 512 * (128 // group))


class Int4Tensor:
    """A ``rows`` x ``cols`` weight in 4 bits as ``linear`` reads it (``data``, a flat uint8 tensor); made by ``from_parts``."""

    __slots__ = ("_data", "_rows", "_cols", "_group", "_scale_dtype", "_bytes")

    data = property(lambda self: self._data)
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    group = property(lambda self: self._group)
    shape = property(lambda self: (self._rows, self._cols))

    @property
    def device(self) -> torch.device:
        return self._data.device

    def __repr__(self) -> str:
        return f"Int4Tensor(shape={self.shape}, group={self.group}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize(self, dtype)


def _check(w, name: str) -> int:
    """The index of the weight's device.  A tensor can be cut off after it was made; what the kernels read has to be there now."""
    if not isinstance(w, Int4Tensor):
        raise ValueError(f"{name} must be an Int4Tensor (see from_parts)")
    data = w._data
    index = data.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if data.numel() < w._bytes:
        raise ValueError(f"{name} has lost a part of its data")
    return index


def from_parts(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *, group: int = 128) -> Int4Tensor:
    """A weight from its parts: ``codes`` ``uint8 [rows, cols]``, one of 0 to 15 a byte, ``scales`` ``[rows, ceil(cols / group)]`` (float16, bfloat16, or
    uint16, which is read as float16's bits) and ``zeros`` ``uint8`` of the same shape, 0 to 15, or None: 8 everywhere.
    ``group`` is 32, 64 or 128.

    The AWQ entries of this library take scales as uint16, too, and compare their bits only: bfloat16's would do there, and come here as ``scales.view(torch.bfloat16)``."""
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}")
    if not isinstance(codes, torch.Tensor) or codes.dtype != torch.uint8 or codes.dim() != 2 or codes.shape[1] == 0:
        raise ValueError("codes must be a uint8 matrix of at least one column")
    rows, cols = codes.shape
    if rows > _MOST_ROWS or cols > _MOST_COLS:
        raise ValueError("an INT4 weight has at most 2^27 rows and 2^24 columns")
    shape = (rows, -(-cols // group))
    if not isinstance(scales, torch.Tensor) or scales.dtype not in (torch.float16, torch.bfloat16, torch.uint16) or tuple(scales.shape) != shape:
        raise ValueError(f"scales must be float16, bfloat16 or uint16, of shape {shape}")
    if zeros is not None and (not isinstance(zeros, torch.Tensor) or zeros.dtype != torch.uint8 or tuple(zeros.shape) != shape):
        raise ValueError(f"zeros must be uint8, of shape {shape}")
    parts = [t for t in (codes, scales, zeros) if t is not None]
    if not all(t.is_cuda for t in parts):
        raise ValueError("codes, scales and zeros must be CUDA tensors")
    if any(t.device != codes.device for t in parts):
        raise ValueError("codes, scales and zeros must be on the same device")
    if not all(t.is_contiguous() for t in parts):
        raise ValueError("codes, scales and zeros must be contiguous")
    for t, name in ((codes, "codes"), (zeros, "zeros")):
        if t is not None and t.numel() and int(t.amax()) > 15:
            raise ValueError(f"{name} must be below 16")
    w = Int4Tensor.__new__(Int4Tensor)
    w._rows, w._cols, w._group, w._bytes = rows, cols, group, _bytes(rows, cols, group)
    w._scale_dtype = 0 if scales.dtype == torch.bfloat16 else 1
    w._data = codes.new_empty(w._bytes)
    _workspace(codes.get_device())      # there before the first product, which may be captured
    _launch(codes.get_device(), "mps_int4_pack", codes.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(), rows, cols, group,
            w._data.data_ptr())
    return w


def dequantize(w: Int4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The weight's values.  Exact in float32; the 16-bit types round once."""
    index = _check(w, "w")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16, float16 or float32")
    out = w._data.new_empty(w._rows, w._cols, dtype=dtype)
    _launch(index, "mps_int4_dequantize", w._data.data_ptr(), w._rows, w._cols, w._group, w._scale_dtype, _DTYPES[dtype], out.data_ptr())
    return out


def linear(x: torch.Tensor, w: Int4Tensor, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ w.T``: ``x`` ``[..., cols]`` in bfloat16 or float16, ``w`` ``[rows, cols]``; sums are FP32, rounded once to ``dtype``, bfloat16 or
    float16, by default ``x``'s.

    A group's products are summed before its scale multiplies them: a bfloat16 token beyond 2^116 may pass FP32's range there, though its result would not.

    Made for the tokens of a decoding step.  Any number of them is served, 64 at a time."""
    index = _check(w, "w")
    rows, cols, stride = _matrix(x, "x")
    x_dtype = x.dtype
    if dtype is None:
        dtype = x_dtype
    if x_dtype not in _HALVES or dtype not in _HALVES:
        raise ValueError("x and the result must be bfloat16 or float16")
    if cols != w._cols:
        raise ValueError(f"x has {cols} columns, the weight {w._cols}")
    if x.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    out_cols = w._rows
    if out_cols == 0:
        raise ValueError("a weight must have at least one row")
    if rows > _MOST_TOKENS:
        raise ValueError("x has more than 2^21 rows")
    out = x.new_empty(*x.shape[:-1], out_cols) if dtype is x_dtype else x.new_empty(*x.shape[:-1], out_cols, dtype=dtype)
    ws = _workspace(index)
    at, aligned = x.data_ptr(), None
    if at % 16 or rows > 1 and (stride % 8 or stride < cols):      # copied first, into memory of this call: freed on return, and not handed to another stream before it is done
        aligned = x.new_empty(rows * ((cols + 7) // 8 * 8))
    args = _lib.INT4_LINEAR.pack(at, 0 if aligned is None else aligned.data_ptr(), w._data.data_ptr(), out.data_ptr(), rows, cols, out_cols, stride, out_cols, w._group, _HALVES[x_dtype],
                                 w._scale_dtype, _HALVES[dtype])
    if _current_device() == index:
        rc = _lib.load().mps_int4_product(args, ws.data_ptr(), ws.numel(), _stream_of(index))
        if rc:
            _lib.check(rc)
    else:
        _launch(index, "mps_int4_product", args, ws.data_ptr(), ws.numel())
    return out
