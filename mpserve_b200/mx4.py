"""Serving in 4 bits: MXFP4 matrices, their products, and the norms, gate and residual around a block.

A compressed checkpoint is decoded once (``sidecar.FusedDecoder``, ``api.huffman_decode_fp8``), its weights are quantised to
MXFP4 (``quantize``), or MXFP4 weights are taken from a checkpoint as they are (``from_parts``); every step then normalises
the residual stream (``rms_norm``), multiplies (``linear``, ``gated_linear``) and joins the block's result to the stream
(``block_join``).  ``GatedMlp`` is a whole block of these.  What passes between the operators may stay in MXFP4.

Every call is asynchronous on the current CUDA stream of its inputs' device and may be made from any thread, or captured in a graph; scratch is of the
call.  Inference only: nothing here has a gradient.  There is no CPU path: without the built library
or a CUDA device the calls raise.  The reference has no counterpart; it multiplies decoded weights in BF16.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

__all__ = ["Mx4Tensor", "quantize", "dequantize", "from_parts", "linear", "gated_linear", "rms_norm", "block_join", "GatedMlp",
           "product_timed_out"]

BLOCK = 32
_MX4 = 3
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTIVATIONS = {"silu": 0, "gelu": 1}
_MOST_NORM_COLS = 32768

# Tokens up to which a product quantises them itself; more of them need x_tiles (include/mpserve_b200.h).
_TOKENS_INSIDE = 8

_workspaces: dict[int, torch.Tensor] = {}
_stream_of = torch._C._cuda_getCurrentRawStream      # the current stream's handle by device index, without an object around it
_current_device = torch._C._cuda_getDevice


def _workspace(index: int) -> torch.Tensor:
    """Where products record a wait that ran out, one per device.  Nothing else outlives a call: what passes between a call's kernels is in memory of
    that call, so that host threads on one stream, and graphs captured on it, do not share any."""
    ws = _workspaces.get(index)
    if ws is None:
        ws = torch.zeros(int(_lib.load().mps_mx4_workspace_bytes()), dtype=torch.uint8, device=torch.device("cuda", index))
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(index).synchronize()      # other streams use it next
        ws = _workspaces.setdefault(index, ws)
    return ws


def _launch(index: int, name: str, *args) -> None:
    """The library's ``name(*args, stream)`` on the current stream of device ``index``."""
    fn = getattr(_lib.load(), name)
    if _current_device() == index:
        rc = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream_of(index))
    if rc:
        _lib.check(rc)


def _matrix(t, name: str) -> tuple[int, int, int]:
    """``t`` as rows x columns of unit column stride: (rows, cols, row stride)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32")
    shape = t.shape
    if len(shape) == 2:
        rows, cols = shape
        stride, unit = t.stride()
        if cols > 1 and unit != 1:
            raise ValueError(f"{name} must have unit stride along its last dimension")
        if cols == 0:
            raise ValueError(f"{name} must have at least one column")
        return rows, cols, stride if rows > 1 else cols
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"{name} must have at least one dimension and one column")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous where it is not a matrix")
    cols = shape[-1]
    return t.numel() // cols, cols, cols


def _tile_bytes(rows: int, cols: int) -> int:
    if rows > 1 << 31 or cols > 1 << 24:
        raise ValueError("an MXFP4 matrix has at most 2^31 rows and 2^24 columns")
    return (rows + 127) // 128 * ((cols + 255) // 256) * 17408


class Mx4Tensor:
    """A ``rows`` x ``cols`` matrix in MXFP4: E2M1 codes and one power-of-two scale per 32 columns, in the tiles that the tensor
    cores read (``data``, a flat uint8 tensor).  ``shape`` is the shape of the tensor it was made of.  None of them can be replaced."""

    __slots__ = ("_data", "_rows", "_cols", "_shape", "_bytes")

    def __init__(self, data: torch.Tensor, rows: int, cols: int, shape=None):
        rows, cols = int(rows), int(cols)
        shape = (rows, cols) if shape is None else tuple(int(n) for n in shape)
        if rows < 0 or cols < 1:
            raise ValueError("an MXFP4 matrix has at least one column and no negative number of rows")
        if len(shape) == 0 or shape[-1] != cols or min(shape) < 0 or math.prod(shape[:-1]) != rows:
            raise ValueError(f"shape {shape} is not that of {rows} rows of {cols} columns")
        need = _tile_bytes(rows, cols)
        if not isinstance(data, torch.Tensor) or data.dtype != torch.uint8 or data.dim() != 1 or not data.is_contiguous():
            raise ValueError("data must be a flat, contiguous uint8 tensor")
        if data.numel() < need:
            raise ValueError(f"data has {data.numel()} bytes, the tiles of {rows} x {cols} {need}")
        self._data, self._rows, self._cols, self._shape, self._bytes = data, rows, cols, shape, need

    data = property(lambda self: self._data)
    rows = property(lambda self: self._rows)
    cols = property(lambda self: self._cols)
    shape = property(lambda self: self._shape)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def __repr__(self) -> str:
        return f"Mx4Tensor(shape={self.shape}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize(self, dtype)

    def parts(self) -> tuple[torch.Tensor, torch.Tensor]:
        """As checkpoints store it: codes ``uint8 [rows, ceil(cols / 2)]``, the even column in a byte's low half, and E8M0 scales
        ``uint8 [rows, ceil(cols / 32)]``."""
        _check_mx4(self, "this matrix")
        dev = self.device
        codes = torch.empty((self.rows, (self.cols + 1) // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((self.rows, -(-self.cols // BLOCK)), dtype=torch.uint8, device=dev)
        _launch(dev.index, "mps_mx4_unpack", self.data.data_ptr(), self.rows, self.cols, codes.data_ptr(), scales.data_ptr())
        return codes, scales


def _mx4(data: torch.Tensor, rows: int, cols: int, shape) -> Mx4Tensor:
    """One whose fields are known to fit: the checks of the public way would be two microseconds of a call's ten."""
    q = Mx4Tensor.__new__(Mx4Tensor)
    q._data, q._rows, q._cols, q._shape, q._bytes = data, rows, cols, shape, data.numel()
    return q


def _check_mx4(q, name: str) -> int:
    """The index of ``q``'s device.  A tensor can be moved or cut off after it was checked; what the kernels read has to be there now."""
    if not isinstance(q, Mx4Tensor):
        raise ValueError(f"{name} must be an Mx4Tensor (see quantize and from_parts)")
    data = q._data
    index = data.get_device()
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if data.numel() < q._bytes:
        raise ValueError(f"{name} has lost a part of its data")
    return index


def quantize(x: torch.Tensor) -> Mx4Tensor:
    """``x`` (BF16, F16 or F32; a matrix of unit column stride, or contiguous) in MXFP4, blocks along the last dimension.

    A block's scale is 2^(floor(log2 max) - 2); codes are rounded to nearest, halfway to the even code, and saturate at 6.  A
    block with an infinity or a NaN becomes NaN."""
    rows, cols, stride = _matrix(x, "x")
    data = x.new_empty(_tile_bytes(rows, cols), dtype=torch.uint8)
    _workspace(x.get_device())      # there before the first product, which may be captured
    _launch(x.get_device(), "mps_mx4_quantize", x.data_ptr(), _DTYPES[x.dtype], rows, cols, stride, data.data_ptr())
    return _mx4(data, rows, cols, x.shape)


def dequantize(q: Mx4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``q`` stands for.  Exact in BF16 and F32, up to their range, which a checkpoint's scale above 2^125 may pass; F16 rounds, and overflows
    beyond 65504."""
    index = _check_mx4(q, "q")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16, float16 or float32")
    data = q._data
    out = data.new_empty(*q._shape, dtype=dtype)
    _launch(index, "mps_mx4_dequantize", data.data_ptr(), q._rows, q._cols, _DTYPES[dtype], out.data_ptr())
    return out


def from_parts(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> Mx4Tensor:
    """An MXFP4 matrix as checkpoints store it: ``codes`` ``uint8 [rows, ceil(cols / 2)]``, the even column in a byte's low half,
    and ``scales`` ``uint8 [rows, ceil(cols / 32)]`` (E8M0).  Laid out once, when a weight is loaded."""
    cols = int(cols)
    if cols <= 0:
        raise ValueError("cols must be > 0")
    for t, name, width in ((codes, "codes", (cols + 1) // 2), (scales, "scales", -(-cols // BLOCK))):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2:
            raise ValueError(f"{name} must be a uint8 matrix")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.shape[1] != width:
            raise ValueError(f"{name} must have {width} columns for {cols} columns of values")
    if codes.shape[0] != scales.shape[0] or codes.device != scales.device:
        raise ValueError("codes and scales must have the same rows and device")
    rows = codes.shape[0]
    data = codes.new_empty(_tile_bytes(rows, cols))
    _workspace(codes.get_device())
    _launch(codes.get_device(), "mps_mx4_pack", codes.data_ptr(), scales.data_ptr(), rows, cols, data.data_ptr())
    return _mx4(data, rows, cols, (rows, cols))


# ---- products --------------------------------------------------------------------------------------------

def _run_product(args, index: int) -> None:
    ws = _workspace(index)
    rc = _lib.load().mps_mx4_product(args, ws.data_ptr(), ws.numel(), _stream_of(index))
    if rc:
        _lib.check(rc)


def _product(x, w, w_up, activation: int, dtype, quantized: bool):
    index = _check_mx4(w, "w" if w_up is None else "w_gate")
    w_data, out_cols, w_cols, up = w._data, w._rows, w._cols, 0
    if w_up is not None:
        if _check_mx4(w_up, "w_up") != index:
            raise ValueError("all tensors must be on the same CUDA device")
        if w_up._rows != out_cols or w_up._cols != w_cols:
            raise ValueError("w_gate and w_up must have the same shape")
        up = w_up._data.data_ptr()
    if out_cols == 0:
        raise ValueError("a weight must have at least one row")
    tiles, stride = None, 0
    if isinstance(x, Mx4Tensor):
        _check_mx4(x, "x")
        rows, cols, x_dtype, data = x._rows, x._cols, _MX4, x._data
        if dtype is None:
            dtype = torch.bfloat16
    else:
        rows, cols, stride = _matrix(x, "x")
        data, x_dtype = x, _DTYPES[x.dtype]
        if dtype is None:
            dtype = torch.bfloat16 if x_dtype == 2 else x.dtype
        if rows > _TOKENS_INSIDE:
            tiles = w_data.new_empty(_tile_bytes(rows, cols))      # of this call: freed on return, and not handed to another stream before it is done
    if cols != w_cols:
        raise ValueError(f"x has {cols} columns, the weight {w_cols}")
    if data.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    shape = (*x.shape[:-1], out_cols)
    if quantized:
        out = w_data.new_empty(_tile_bytes(rows, out_cols))
        out_dtype, result = _MX4, _mx4(out, rows, out_cols, shape)
    else:
        if dtype is not torch.bfloat16 and dtype is not torch.float16:
            raise ValueError("a product's dtype must be bfloat16 or float16")
        out = result = data.new_empty(*shape) if data.dtype is dtype else data.new_empty(*shape, dtype=dtype)
        out_dtype = _DTYPES[dtype]
    args = _lib.MX4_LINEAR.pack(data.data_ptr(), 0 if tiles is None else tiles.data_ptr(), w_data.data_ptr(), up, out.data_ptr(), rows, cols, out_cols,
                                stride, out_cols, x_dtype, out_dtype, activation, 0)
    if _current_device() == index:
        _run_product(args, index)
    else:
        with torch.cuda.device(index):
            _run_product(args, index)
    return result


def linear(x, w: Mx4Tensor, *, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ w.T``: ``x`` ``[..., cols]`` an ``Mx4Tensor``, or a tensor that is quantised on the way; ``w`` ``[rows, cols]``.

    Both operands are MXFP4, sums are FP32, rounded once to ``dtype``: bfloat16 or float16, by default that of ``x`` where
    it is one of the two, else bfloat16."""
    return _product(x, w, None, 0, dtype, False)


def gated_linear(x, w_gate: Mx4Tensor, w_up: Mx4Tensor, *, activation: str = "silu", dtype: torch.dtype | None = None,
                 quantized: bool = False):
    """``act(x @ w_gate.T) * (x @ w_up.T)`` with ``act`` "silu" or "gelu" (its tanh form), without the two products in memory.

    ``quantized``: the result as an ``Mx4Tensor`` for the next product, rounded once, from FP32."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}")
    _check_mx4(w_up, "w_up")
    return _product(x, w_gate, w_up, _ACTIVATIONS[activation], dtype, bool(quantized))


def product_timed_out(device: torch.device | None = None) -> bool:
    """Waits for the device's current stream and tells whether a product on the device, a replayed graph's included, gave up on one of its bounded waits
    since the last call (its outputs are then incomplete).  Of other streams' products, those that have ended count.  Always False in
    normal operation."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    with torch.cuda.device(index):
        ws = _workspace(index)
        flag = C.c_int32(0)
        _lib.check(_lib.load().mps_mx4_status(ws.data_ptr(), ws.numel(), _stream_of(index), C.byref(flag)))
    return bool(flag.value)


# ---- norms, gate and residual ------------------------------------------------------------------------------

def _gain(t, name: str, cols: int, index: int) -> tuple[int, int]:
    """(pointer, dtype) of a norm's weight."""
    dtype = _DTYPES.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if dtype is None or t.dim() != 1 or t.numel() != cols:
        raise ValueError(f"{name} must be a bfloat16, float16 or float32 vector of {cols} values")
    if t.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr(), dtype


def _gains(post_weight, next_weight, cols: int, index: int):
    """(pointers or 0, the dtype that the two share)."""
    post = nxt = dtype = 0
    if post_weight is not None:
        post, dtype = _gain(post_weight, "post_weight", cols, index)
    if next_weight is not None:
        post_dtype = dtype
        nxt, dtype = _gain(next_weight, "next_weight", cols, index)
        if post_weight is not None and post_dtype != dtype:
            raise ValueError("post_weight and next_weight must have the same dtype")
    return post, nxt, dtype


def _check_norm_cols(cols: int) -> None:
    if cols > _MOST_NORM_COLS:
        raise ValueError(f"a norm has at most {_MOST_NORM_COLS} columns")


def _normed(like, rows, cols, dtype, quantized: bool):
    """Where a norm's result goes, in ``like``'s shape: (what the caller gets, pointer, dtype)."""
    if quantized:
        data = like.new_empty(_tile_bytes(rows, cols), dtype=torch.uint8)
        return _mx4(data, rows, cols, like.shape), data.data_ptr(), _MX4
    n = like.new_empty(*like.shape) if like.dtype is dtype else like.new_empty(*like.shape, dtype=dtype)
    return n, n.data_ptr(), _DTYPES[dtype]


def rms_norm(h: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-5, dtype: torch.dtype | None = None, quantized: bool = False):
    """``h * rsqrt(mean(h^2) + eps) * weight`` along the last dimension, in ``dtype`` (by default ``h``'s) or, ``quantized``, as an
    ``Mx4Tensor`` that never was anything but FP32 before."""
    rows, cols, stride = _matrix(h, "h")
    _check_norm_cols(cols)
    dtype = h.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16, float16 or float32")
    index = h.get_device()
    w, w_dtype = _gain(weight, "weight", cols, index)
    n, n_ptr, n_dtype = _normed(h, rows, cols, dtype, quantized)
    args = _lib.MX4_NORM.pack(0, h.data_ptr(), 0, 0, w, 0, n_ptr, rows, cols, 0, stride, 0, cols, 0, 0, 0, _DTYPES[h.dtype], n_dtype, 0,
                              w_dtype, eps, 1.0)
    _launch(index, "mps_mx4_norm_rows", args)
    return n


def _check_inplace(h, rows: int, cols: int, stride: int, others) -> None:
    """Refuses an ``h`` that cannot be written row by row while ``others`` (name, tensor, rows, columns, row stride) are read: a CTA reads a row of each
    and writes that row, in no order.  One that is ``h`` itself, element by element, is read where it is written and does no harm."""
    if rows > 1 and stride < cols:
        raise ValueError("h has rows that share memory and cannot be updated in place")
    if rows == 0:
        return
    start, size = h.data_ptr(), h.element_size()
    pitch, width = stride * size, cols * size
    end = start + (rows - 1) * pitch + width
    for name, t, t_rows, t_cols, t_stride in others:
        if t is None:
            continue
        t_start, t_size = t.data_ptr(), t.element_size()
        t_pitch, t_width = t_stride * t_size, t_cols * t_size
        if t_start >= end or t_start + (t_rows - 1) * t_pitch + t_width <= start:
            continue
        if t_start == start and t_width == width and t_size == size and t_rows == rows and (rows == 1 or t_pitch == pitch):
            continue
        # columns of one wider matrix: rows of the same pitch that lie beside one another
        beside = (t_start - start) % pitch
        if t_rows > 1 and t_pitch == pitch and beside >= width and beside + t_width <= pitch:
            continue
        raise ValueError(f"{name} shares memory with h, which cannot be updated in place")


def block_join(y: torch.Tensor, h: torch.Tensor, *, post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               residual_scale: float = 1.0, next_weight: torch.Tensor | None = None, eps: float = 1e-5,
               quantized: bool = False, inplace: bool = False):
    """The end of a block and the norm before the next, one pass over ``y`` (the block's result) and ``h`` (the residual stream):

        ``h' = residual_scale * h + gate * rms_norm(y, post_weight)``      (``y`` itself without ``post_weight``)
        ``n  = rms_norm(h', next_weight)``

    Returns ``(h', n)``; ``n`` is None without ``next_weight``, in ``y``'s dtype otherwise or, ``quantized``, an ``Mx4Tensor``.
    ``gate``: None, or any shape that broadcasts to ``y``'s with one value per column, per row or per element.  ``h`` may be
    FP32 beside a 16-bit ``y``; ``h'`` has its type, and is ``h`` itself where ``inplace``.  The two weights share a dtype."""
    rows, cols, y_stride = _matrix(y, "y")
    _, _, h_stride = _matrix(h, "h")
    shape, index = y.shape, y.get_device()
    if shape != h.shape:
        raise ValueError("y and h must have the same shape")
    _check_norm_cols(cols)
    if h.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    n = None
    n_ptr = n_dtype = g = g_dtype = g_row = g_col = 0
    post, nxt, weight_dtype = _gains(post_weight, next_weight, cols, index)
    if gate is not None:
        g, g_dtype, g_row, g_col = _gate(gate, y, rows, cols)
    if inplace:
        _check_inplace(h, rows, cols, h_stride, (("y", y, rows, cols, y_stride), ("gate", gate, *_gate_extent(gate, g_row, rows, cols)),
                                                 ("post_weight", post_weight, 1, cols, cols), ("next_weight", next_weight, 1, cols, cols)))
        joined, out_stride = h, h_stride
    else:
        joined, out_stride = h.new_empty(*shape), cols
    if nxt:
        n, n_ptr, n_dtype = _normed(y, rows, cols, y.dtype, quantized)
    args = _lib.MX4_NORM.pack(y.data_ptr(), h.data_ptr(), post, g, nxt, joined.data_ptr(), n_ptr, rows, cols, y_stride, h_stride, out_stride, cols,
                              g_row, g_col, _DTYPES[y.dtype], _DTYPES[h.dtype], n_dtype, g_dtype, weight_dtype, eps, residual_scale)
    _launch(index, "mps_mx4_norm_rows", args)
    return joined, n


def _gate(gate, y, rows: int, cols: int):
    """(pointer, dtype, row stride, column stride) of a gate that broadcasts to ``y``."""
    if not isinstance(gate, torch.Tensor) or gate.dtype not in _DTYPES:
        raise ValueError("gate must be a bfloat16, float16 or float32 tensor")
    if gate.get_device() != y.get_device():
        raise ValueError("all tensors must be on the same CUDA device")
    if gate.dim() <= y.dim() and gate.is_contiguous():
        if gate.dim() == 1 and gate.numel() == cols:
            return gate.data_ptr(), _DTYPES[gate.dtype], 0, int(cols > 1)
        shape = (1,) * (y.dim() - gate.dim()) + tuple(gate.shape)
        last = shape[-1]
        if last == 1 or last == cols:
            per_column = int(last == cols and cols > 1)
            if gate.numel() == last:
                return gate.data_ptr(), _DTYPES[gate.dtype], 0, per_column
            if shape[:-1] == tuple(y.shape[:-1]):
                return gate.data_ptr(), _DTYPES[gate.dtype], last, per_column
    raise ValueError("gate must be contiguous and have one value per column, per row or per element of y")


def _gate_extent(gate, row_stride: int, rows: int, cols: int) -> tuple[int, int, int]:
    """(rows, columns, row stride) of what ``_gate`` has found."""
    if gate is None:
        return 0, 0, 0
    return (rows, row_stride, row_stride) if row_stride else (1, gate.numel(), gate.numel())


class GatedMlp:
    """A gated MLP block in 4 bits: ``rms_norm`` -> ``gated_linear`` -> ``linear`` -> ``block_join``.

    ``gate_proj`` and ``up_proj`` ``[inter, hidden]``, ``down_proj`` ``[hidden, inter]`` are ``Mx4Tensor``; ``post_weight``, ``gate``,
    ``residual_scale`` and ``next_weight`` are as for ``block_join``.  ``forward(h)`` returns ``(h', n)``.

    Between ``linear`` and ``block_join`` the block's result is rounded to ``h``'s type (BF16 beside an FP32 stream; beyond F16's range it stays what it
    is), and ``n`` has that type too.  With ``result_dtype=torch.float32`` it is not rounded, and ``n`` has ``h``'s type.  All of these are attributes that may be
    replaced, and a tensor's storage with them: a call takes them as they are then, and refuses what does not fit."""

    def __init__(self, gate_proj: Mx4Tensor, up_proj: Mx4Tensor, down_proj: Mx4Tensor, *, pre_weight: torch.Tensor,
                 post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                 next_weight: torch.Tensor | None = None, eps: float = 1e-5, activation: str = "silu",
                 result_dtype: torch.dtype | None = None):
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj
        self.pre_weight, self.post_weight, self.gate, self.next_weight = pre_weight, post_weight, gate, next_weight
        self.residual_scale, self.eps, self.activation, self.result_dtype = residual_scale, eps, activation, result_dtype
        _, hidden, _, _, _ = self._operands()
        if gate is not None and isinstance(gate, torch.Tensor) and gate.dim() == 1 and gate.numel() == hidden:
            _gate(gate, pre_weight, 1, hidden)      # a value per row or per element has to fit the tokens, which come with a call

    @property
    def hidden(self) -> int:
        return self.gate_proj.cols

    @property
    def inter(self) -> int:
        return self.gate_proj.rows

    def _operands(self):
        """What the attributes hold now: (device index, hidden, inter, pointers, (dtype of pre_weight, of the other two, activation))."""
        g, u, d = self.gate_proj, self.up_proj, self.down_proj
        index = _check_mx4(g, "gate_proj")
        if _check_mx4(u, "up_proj") != index or _check_mx4(d, "down_proj") != index:
            raise ValueError("all tensors must be on the same CUDA device")
        inter, hidden = g._rows, g._cols
        if inter == 0 or u._rows != inter or u._cols != hidden or d._rows != hidden or d._cols != inter:
            raise ValueError("gate_proj and up_proj must be [inter, hidden], down_proj [hidden, inter]")
        if self.activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}")
        if self.result_dtype is not None and self.result_dtype is not torch.float32:
            raise ValueError("result_dtype must be None or float32")
        _check_norm_cols(hidden)
        pre, pre_dtype = _gain(self.pre_weight, "pre_weight", hidden, index)
        post, nxt, dtype = _gains(self.post_weight, self.next_weight, hidden, index)
        return index, hidden, inter, (g._data.data_ptr(), u._data.data_ptr(), d._data.data_ptr(), pre, post, nxt), (
            pre_dtype, dtype, _ACTIVATIONS[self.activation])

    def forward(self, h: torch.Tensor, *, inplace: bool = False):
        index, hidden, inter, (g, u, d, pre, post, nxt), (pre_dtype, dtype, activation) = self._operands()
        rows, cols, stride = _matrix(h, "h")
        if cols != hidden:
            raise ValueError(f"h has {cols} columns, the block {hidden}")
        if h.get_device() != index:
            raise ValueError("all tensors must be on the same CUDA device")
        gate = gate_dtype = gate_row = gate_col = 0
        if self.gate is not None:
            gate, gate_dtype, gate_row, gate_col = _gate(self.gate, h, rows, cols)
        block = _lib.MX4_MLP.pack(g, u, d, pre, post, gate, nxt, hidden, inter, gate_row, gate_col, gate_dtype, pre_dtype, dtype, activation, self.eps,
                                  self.residual_scale, self.result_dtype is not None)
        h_dtype = _DTYPES[h.dtype]
        n_dtype = 0 if h_dtype == 2 and self.result_dtype is None else h_dtype
        if inplace:
            _check_inplace(h, rows, cols, stride, (("gate", self.gate, *_gate_extent(self.gate, gate_row, rows, cols)),
                                                   ("post_weight", self.post_weight, 1, cols, cols), ("next_weight", self.next_weight, 1, cols, cols)))
            joined, out_stride = h, stride
        else:
            joined, out_stride = h.new_empty(*h.shape), cols
        n = None
        if nxt:
            n = h.new_empty(*h.shape) if n_dtype == h_dtype else h.new_empty(*h.shape, dtype=torch.bfloat16)
        scratch_bytes = _tile_bytes(rows, inter) + max(_tile_bytes(rows, cols) + rows * cols * 2, rows * cols * 4)
        scratch = h.new_empty(scratch_bytes, dtype=torch.uint8)      # of this call: freed on return, and not handed to another stream before it is done
        args = (_lib.Mx4Mlp.from_buffer_copy(block), h.data_ptr(), h_dtype, stride, rows, joined.data_ptr(), out_stride, None if n is None else n.data_ptr(),
                n_dtype, scratch.data_ptr(), scratch_bytes)
        if _current_device() == index:
            self._run(args, index)
        else:
            with torch.cuda.device(index):
                self._run(args, index)
        return joined, n

    __call__ = forward

    @staticmethod
    def _run(args, index: int) -> None:
        ws = _workspace(index)
        rc = _lib.load().mps_mx4_gated_mlp(*args, ws.data_ptr(), ws.numel(), _stream_of(index))
        if rc:
            _lib.check(rc)
