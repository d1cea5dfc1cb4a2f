"""Serving in 4 bits: MXFP4 matrices, their products, and the norms, gate and residual around a block.

A compressed checkpoint is decoded once (``sidecar.FusedDecoder``, ``api.huffman_decode_fp8``), its weights are quantised to
MXFP4 (``quantize``), or MXFP4 weights are taken from a checkpoint as they are (``from_parts``); every step then normalises
the residual stream (``rms_norm``), multiplies (``linear``, ``gated_linear``) and joins the block's result to the stream
(``block_join``).  ``GatedMlp`` is a whole block of these.  What passes between the operators may stay in MXFP4.

Every call is asynchronous on the current CUDA stream of its inputs' device; scratch is kept per device and stream, as the decoder
keeps its own.  Inference only: nothing here has a gradient.  There is no CPU path: without the built library
or a CUDA device the calls raise.  The reference has no counterpart; it multiplies decoded weights in BF16.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

__all__ = ["Mx4Tensor", "quantize", "dequantize", "from_parts", "linear", "gated_linear", "rms_norm", "block_join", "GatedMlp",
           "product_timed_out"]

BLOCK = 32
_MX4 = 3
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTIVATIONS = {"silu": 0, "gelu": 1}
_MOST_NORM_COLS = 32768

_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def _workspace(device: torch.device, stream: int) -> torch.Tensor:
    """Zeroed counters and partial sums, one per (device, stream); the products hand the counters back zeroed."""
    key = (device.index, stream)
    ws = _workspaces.get(key)
    if ws is None:
        ws = torch.zeros(int(_lib.load().mps_mx4_workspace_bytes()), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


class _on:
    """The device of the inputs, and its current stream's handle."""

    def __init__(self, device: torch.device):
        self.device = device
        self.other = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self) -> int:
        if self.other is not None:
            self.other.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.other is not None:
            self.other.__exit__(*exc)


def _matrix(t, name: str) -> tuple[torch.Tensor, int, int, int]:
    """``t`` as rows x columns of unit column stride: (tensor, rows, cols, row stride)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32")
    if t.dim() == 2:
        rows, cols = t.shape
        if cols > 1 and t.stride(1) != 1:
            raise ValueError(f"{name} must have unit stride along its last dimension")
        stride = t.stride(0) if rows > 1 else cols
        if stride < 0 or cols == 0:
            raise ValueError(f"{name} must have at least one column")
        return t, rows, cols, stride
    if t.dim() == 0 or t.shape[-1] == 0:
        raise ValueError(f"{name} must have at least one dimension and one column")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous where it is not a matrix")
    cols = t.shape[-1]
    return t, t.numel() // cols, cols, cols


def _tiles(rows: int, cols: int, device: torch.device) -> torch.Tensor:
    nbytes = int(_lib.load().mps_mx4_bytes(rows, cols))
    if nbytes < 0:
        raise ValueError("an MXFP4 matrix has at most 2^31 rows and 2^24 columns")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


class Mx4Tensor:
    """A ``rows`` x ``cols`` matrix in MXFP4: E2M1 codes and one power-of-two scale per 32 columns, in the tiles that the tensor
    cores read (``data``).  ``shape`` is the shape of the tensor it was made of."""

    __slots__ = ("data", "rows", "cols", "shape")

    def __init__(self, data: torch.Tensor, rows: int, cols: int, shape=None):
        self.data, self.rows, self.cols = data, rows, cols
        self.shape = (rows, cols) if shape is None else tuple(shape)

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
        dev = self.device
        codes = torch.empty((self.rows, (self.cols + 1) // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((self.rows, -(-self.cols // BLOCK)), dtype=torch.uint8, device=dev)
        with _on(dev) as stream:
            _lib.check(_lib.load().mps_mx4_unpack(self.data.data_ptr(), self.rows, self.cols, codes.data_ptr(), scales.data_ptr(), stream))
        return codes, scales


def _check_mx4(q, name: str) -> None:
    if not isinstance(q, Mx4Tensor):
        raise ValueError(f"{name} must be an Mx4Tensor (see quantize and from_parts)")


def quantize(x: torch.Tensor) -> Mx4Tensor:
    """``x`` (BF16, F16 or F32; a matrix of unit column stride, or contiguous) in MXFP4, blocks along the last dimension.

    A block's scale is 2^(floor(log2 max) - 2); codes are rounded to nearest, halfway to the even code, and saturate at 6.  A
    block with an infinity or a NaN becomes NaN."""
    x, rows, cols, stride = _matrix(x, "x")
    dev = x.device
    data = _tiles(rows, cols, dev)
    with _on(dev) as s:
        _lib.check(_lib.load().mps_mx4_quantize(x.data_ptr(), _DTYPES[x.dtype], rows, cols, stride, data.data_ptr(), s))
    return Mx4Tensor(data, rows, cols, x.shape)


def dequantize(q: Mx4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``q`` stands for.  Exact in BF16 and F32; F16 rounds, and overflows beyond 65504."""
    _check_mx4(q, "q")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16, float16 or float32")
    dev = q.device
    out = torch.empty(q.shape, dtype=dtype, device=dev)
    with _on(dev) as s:
        _lib.check(_lib.load().mps_mx4_dequantize(q.data.data_ptr(), q.rows, q.cols, _DTYPES[dtype], out.data_ptr(), s))
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
    rows, dev = codes.shape[0], codes.device
    data = _tiles(rows, cols, dev)
    with _on(dev) as s:
        _lib.check(_lib.load().mps_mx4_pack(codes.data_ptr(), scales.data_ptr(), rows, cols, data.data_ptr(), s))
    return Mx4Tensor(data, rows, cols)


# ---- products --------------------------------------------------------------------------------------------

def _product(x, w, w_up, activation: int, dtype, quantized: bool):
    _check_mx4(w, "w" if w_up is None else "w_gate")
    if w_up is not None:
        _check_mx4(w_up, "w_up")
        if (w_up.rows, w_up.cols) != (w.rows, w.cols):
            raise ValueError("w_gate and w_up must have the same shape")
    if w.rows == 0:
        raise ValueError("a weight must have at least one row")
    dev = w.device
    a = _lib.Mx4Linear()
    if isinstance(x, Mx4Tensor):
        rows, cols, tiles = x.rows, x.cols, None
        a.x, a.x_dtype = x.data.data_ptr(), _MX4
        if dtype is None:
            dtype = torch.bfloat16
    else:
        x, rows, cols, a.x_stride = _matrix(x, "x")
        if dtype is None:
            dtype = torch.bfloat16 if x.dtype == torch.float32 else x.dtype
        tiles = _tiles(rows, cols, dev)
        a.x, a.x_dtype, a.x_tiles = x.data_ptr(), _DTYPES[x.dtype], tiles.data_ptr()
    if cols != w.cols:
        raise ValueError(f"x has {cols} columns, the weight {w.cols}")
    if x.device != dev or (w_up is not None and w_up.device != dev):
        raise ValueError("all tensors must be on the same CUDA device")
    shape = (*x.shape[:-1], w.rows)
    if quantized:
        out = _tiles(rows, w.rows, dev)
        a.out, a.out_dtype = out.data_ptr(), _MX4
        result = Mx4Tensor(out, rows, w.rows, shape)
    else:
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("a product's dtype must be bfloat16 or float16")
        result = torch.empty(shape, dtype=dtype, device=dev)
        a.out, a.out_dtype, a.out_stride = result.data_ptr(), _DTYPES[dtype], w.rows
    a.w = w.data.data_ptr()
    if w_up is not None:
        a.w_up = w_up.data.data_ptr()
    a.tokens, a.cols, a.rows, a.activation = rows, cols, w.rows, activation
    with _on(dev) as s:
        ws = _workspace(dev, s)
        _lib.check(_lib.load().mps_mx4_product(C.byref(a), ws.data_ptr(), ws.numel(), s))
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
    """Waits for the current stream and tells whether a product launched on it since the last call gave up on one of its bounded
    waits (its outputs are then incomplete).  Always False in normal operation."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    with _on(dev) as s:
        ws = _workspace(dev, s)
        flag = C.c_int32(0)
        _lib.check(_lib.load().mps_mx4_status(ws.data_ptr(), ws.numel(), s, C.byref(flag)))
    return bool(flag.value)


# ---- norms, gate and residual ------------------------------------------------------------------------------

def _gain(t, name: str, cols: int, dev, a) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES or t.dim() != 1 or t.shape[0] != cols:
        raise ValueError(f"{name} must be a bfloat16, float16 or float32 vector of {cols} values")
    if t.device != dev:
        raise ValueError("all tensors must be on the same CUDA device")
    if cols > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _check_norm_cols(cols: int) -> None:
    if cols > _MOST_NORM_COLS:
        raise ValueError(f"a norm has at most {_MOST_NORM_COLS} columns")


def _normed(a, shape, rows, cols, dtype, dev, quantized: bool):
    if quantized:
        data = _tiles(rows, cols, dev)
        a.n_out, a.n_dtype = data.data_ptr(), _MX4
        return Mx4Tensor(data, rows, cols, shape)
    n = torch.empty(shape, dtype=dtype, device=dev)
    a.n_out, a.n_dtype, a.n_stride = n.data_ptr(), _DTYPES[dtype], cols
    return n


def _launch_norm(a, dev) -> None:
    with _on(dev) as s:
        _lib.check(_lib.load().mps_mx4_norm_rows(C.byref(a), s))


def rms_norm(h: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-5, dtype: torch.dtype | None = None, quantized: bool = False):
    """``h * rsqrt(mean(h^2) + eps) * weight`` along the last dimension, in ``dtype`` (by default ``h``'s) or, ``quantized``, as an
    ``Mx4Tensor`` that never was anything but FP32 before."""
    h, rows, cols, stride = _matrix(h, "h")
    _check_norm_cols(cols)
    dtype = h.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16, float16 or float32")
    dev = h.device
    a = _lib.Mx4Norm()
    a.next_weight, a.weight_dtype = _gain(weight, "weight", cols, dev, a), _DTYPES[weight.dtype]
    a.h, a.h_stride, a.h_dtype = h.data_ptr(), stride, _DTYPES[h.dtype]
    a.rows, a.cols, a.eps, a.residual_scale = rows, cols, eps, 1.0
    n = _normed(a, h.shape, rows, cols, dtype, dev, quantized)
    _launch_norm(a, dev)
    return n


def block_join(y: torch.Tensor, h: torch.Tensor, *, post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               residual_scale: float = 1.0, next_weight: torch.Tensor | None = None, eps: float = 1e-5,
               quantized: bool = False, inplace: bool = False):
    """The end of a block and the norm before the next, one pass over ``y`` (the block's result) and ``h`` (the residual stream):

        ``h' = residual_scale * h + gate * rms_norm(y, post_weight)``      (``y`` itself without ``post_weight``)
        ``n  = rms_norm(h', next_weight)``

    Returns ``(h', n)``; ``n`` is None without ``next_weight``, in ``y``'s dtype otherwise or, ``quantized``, an ``Mx4Tensor``.
    ``gate``: None, or any shape that broadcasts to ``y``'s with one value per column, per row or per element.  ``h`` may be
    FP32 beside a 16-bit ``y``; ``h'`` has its type, and is ``h`` itself where ``inplace``.  The two weights share a dtype."""
    y, rows, cols, y_stride = _matrix(y, "y")
    h, h_rows, h_cols, h_stride = _matrix(h, "h")
    if y.shape != h.shape:
        raise ValueError("y and h must have the same shape")
    _check_norm_cols(cols)
    dev = y.device
    if h.device != dev:
        raise ValueError("all tensors must be on the same CUDA device")
    a = _lib.Mx4Norm()
    if post_weight is not None:
        a.post_weight, a.weight_dtype = _gain(post_weight, "post_weight", cols, dev, a), _DTYPES[post_weight.dtype]
    if next_weight is not None:
        a.next_weight = _gain(next_weight, "next_weight", cols, dev, a)
        if post_weight is not None and post_weight.dtype != next_weight.dtype:
            raise ValueError("post_weight and next_weight must have the same dtype")
        a.weight_dtype = _DTYPES[next_weight.dtype]
    if gate is not None:
        a.gate, a.gate_dtype, a.gate_row_stride, a.gate_col_stride = _gate(gate, y, rows, cols)
    a.y, a.y_stride, a.y_dtype = y.data_ptr(), y_stride, _DTYPES[y.dtype]
    a.h, a.h_stride, a.h_dtype = h.data_ptr(), h_stride, _DTYPES[h.dtype]
    if inplace:
        joined = h
        if rows > 1 and h_stride < cols:
            raise ValueError("h has rows that share memory and cannot be updated in place")
        a.h_out, a.h_out_stride = h.data_ptr(), h_stride
    else:
        joined = torch.empty(h.shape, dtype=h.dtype, device=dev)
        a.h_out, a.h_out_stride = joined.data_ptr(), cols
    a.rows, a.cols, a.eps, a.residual_scale = rows, cols, eps, residual_scale
    n = None if next_weight is None else _normed(a, y.shape, rows, cols, y.dtype, dev, quantized)
    _launch_norm(a, dev)
    return joined, n


def _gate(gate, y, rows: int, cols: int):
    """(pointer, dtype, row stride, column stride) of a gate that broadcasts to ``y``."""
    if not isinstance(gate, torch.Tensor) or gate.dtype not in _DTYPES:
        raise ValueError("gate must be a bfloat16, float16 or float32 tensor")
    if gate.device != y.device:
        raise ValueError("all tensors must be on the same CUDA device")
    shape = (1,) * (y.dim() - gate.dim()) + tuple(gate.shape)
    if len(shape) == y.dim() and gate.is_contiguous() and shape[-1] in (1, cols):
        lead = gate.numel() // shape[-1]
        per_column = shape[-1] == cols and cols > 1
        if lead == 1:
            return gate.data_ptr(), _DTYPES[gate.dtype], 0, int(per_column)
        if shape[:-1] == tuple(y.shape[:-1]):
            return gate.data_ptr(), _DTYPES[gate.dtype], shape[-1], int(per_column)
    raise ValueError("gate must be contiguous and have one value per column, per row or per element of y")


class GatedMlp:
    """A gated MLP block in 4 bits: ``rms_norm`` -> ``gated_linear`` -> ``linear`` -> ``block_join``.

    ``gate_proj`` and ``up_proj`` ``[inter, hidden]``, ``down_proj`` ``[hidden, inter]`` are ``Mx4Tensor``; ``post_weight``, ``gate``,
    ``residual_scale`` and ``next_weight`` are as for ``block_join``.  ``forward(h)`` returns ``(h', n)``."""

    def __init__(self, gate_proj: Mx4Tensor, up_proj: Mx4Tensor, down_proj: Mx4Tensor, *, pre_weight: torch.Tensor,
                 post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, residual_scale: float = 1.0,
                 next_weight: torch.Tensor | None = None, eps: float = 1e-5, activation: str = "silu"):
        for q, name in ((gate_proj, "gate_proj"), (up_proj, "up_proj"), (down_proj, "down_proj")):
            _check_mx4(q, name)
        if (up_proj.rows, up_proj.cols) != (gate_proj.rows, gate_proj.cols) or (down_proj.rows, down_proj.cols) != (gate_proj.cols, gate_proj.rows):
            raise ValueError("gate_proj and up_proj must be [inter, hidden], down_proj [hidden, inter]")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}")
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj
        self.pre_weight, self.post_weight, self.gate, self.next_weight = pre_weight, post_weight, gate, next_weight
        self.residual_scale, self.eps, self.activation = float(residual_scale), float(eps), activation

    def forward(self, h: torch.Tensor, *, inplace: bool = False):
        x = rms_norm(h, self.pre_weight, eps=self.eps, quantized=True)
        a = gated_linear(x, self.gate_proj, self.up_proj, activation=self.activation, quantized=True)
        y = linear(a, self.down_proj, dtype=torch.bfloat16 if h.dtype == torch.float32 else h.dtype)
        return block_join(y, h, post_weight=self.post_weight, gate=self.gate, residual_scale=self.residual_scale,
                          next_weight=self.next_weight, eps=self.eps, inplace=inplace)

    __call__ = forward
