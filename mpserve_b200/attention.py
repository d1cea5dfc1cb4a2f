"""The attention of a decoding step: norms and position rotation of queries and keys, the paged cache, and attention behind a prefix that a batch shares.

Between the projection of a step's tokens (``int4.linear``, ``mx4.linear``) and the projection of the result, per layer:
``norm_rotate_append`` normalises and rotates the heads and writes keys and values into the cache, ``shared_prefix_attention`` answers the queries.  A prompt's tokens
take ``norm_rotate``.

Calls are asynchronous on the current CUDA stream of their inputs' device and may be made from any thread, or captured in a graph; scratch is of the
call.  Inference only: nothing here has a gradient.  There is no CPU path.  The reference leaves attention to the engine that it is plugged into.
"""
from __future__ import annotations

import ctypes as C
import functools
import math

import torch

from . import _lib
from .mx4 import _DTYPES, _current_device, _launch, _stream_of, _workspace

__all__ = ["Rotary", "KvCache", "norm_rotate", "norm_rotate_append", "shared_prefix_attention"]

_MOST_DIM, _MOST_HEADS, _MOST_SEQUENCES, _MOST_KEYS = 256, 1024, 1 << 16, 1 << 30


class Rotary:
    """How positions turn a head: pair ``j`` of its first ``dims`` values turns by ``position * frequencies[j]`` (radians), with ``frequencies`` a vector of
    ``dims / 2`` values, by default ``base ** (-2 j / dims)``.

    A pair is ``(j, j + dims / 2)`` or, ``interleaved``, ``(2 j, 2 j + 1)``.  Positions with several axes (time, height, width): ``axes`` has, for each
    pair, the index of the axis that turns it, or ``sections`` how many pairs in a row each axis turns.  Turned values are multiplied by ``scale``.
    Frequencies are kept in float64; the handle may be used from every device's calls after ``to``."""

    def __init__(self, dims: int, *, base: float = 10000.0, frequencies: torch.Tensor | None = None, axes=None, sections=None, interleaved: bool = False,
                 scale: float = 1.0, device: torch.device | str | None = None):
        dims = int(dims)
        if dims < 0 or dims % 2 or dims > _MOST_DIM:
            raise ValueError(f"dims must be even, from 0 to {_MOST_DIM}")
        pairs = dims // 2
        if frequencies is None:
            frequencies = torch.tensor([float(base) ** (-2.0 * j / dims) for j in range(pairs)], dtype=torch.float64)
        elif not isinstance(frequencies, torch.Tensor) or not frequencies.is_floating_point() or tuple(frequencies.shape) != (pairs,):
            raise ValueError(f"frequencies must be a floating-point vector of {pairs} values")
        elif device is None:
            device = frequencies.device
        if axes is not None and sections is not None:
            raise ValueError("axes and sections exclude one another")
        if sections is not None:
            axes = [i for i, n in enumerate(sections) for _ in range(int(n))]
        if axes is not None:
            axes = [int(i) for i in axes]
            if len(axes) != pairs or any(i < 0 or i > 255 for i in axes):
                raise ValueError(f"every one of the {pairs} pairs must have an axis, from 0 to 255")
        device = torch.device("cuda" if device is None else device)
        self.dims, self.interleaved, self.scale = dims, bool(interleaved), float(scale)
        self.axes = 1 + max(axes, default=0) if axes is not None else 1
        self._turns = (frequencies.to(torch.float64) / (2.0 * math.pi)).to(device).contiguous()
        self._axis = None if axes is None or self.axes == 1 else torch.tensor(axes, dtype=torch.uint8).to(device)

    @property
    def device(self) -> torch.device:
        return self._turns.device

    def to(self, device) -> "Rotary":
        """The same on another device."""
        r = Rotary.__new__(Rotary)
        r.dims, r.interleaved, r.scale, r.axes = self.dims, self.interleaved, self.scale, self.axes
        r._turns, r._axis = self._turns.to(device), None if self._axis is None else self._axis.to(device)
        return r


class KvCache:
    """The pages of a paged cache: ``k_pages`` and ``v_pages`` ``[pages, page_size, kv_heads, head_dim]``, one dtype (bfloat16, float16; float32 for
    ``norm_rotate_append`` alone), the last dimension of unit stride, the others of any that keeps 16-byte alignment; no two places share memory.  The tensors are the
    caller's, and cannot be replaced; slot ``i`` is place ``i % page_size`` of page ``i // page_size``.  ``page_size`` is a power of two."""

    __slots__ = ("_k_pages", "_v_pages")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if not isinstance(t, torch.Tensor) or t.dim() != 4:
                raise ValueError(f"{name} must have the dimensions [pages, page_size, kv_heads, head_dim]")
            if t.dtype not in _DTYPES:
                raise ValueError(f"{name} must be bfloat16, float16 or float32")
            if not t.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor")
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
            raise ValueError("k_pages and v_pages must have the same shape, dtype and device")
        pages, page_size, heads, dim = k_pages.shape
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if heads < 1 or heads > _MOST_HEADS or dim < 1 or dim > _MOST_DIM or pages > 0x7FFFFFFF:
            raise ValueError(f"a cache has 1 to {_MOST_HEADS} heads of 1 to {_MOST_DIM} values, and less than 2^31 pages")
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if dim > 1 and t.stride(3) != 1:
                raise ValueError(f"{name} must have unit stride along its last dimension")
            unit = 16 // t.element_size()
            if t.data_ptr() % 16 or any(s % unit for n, s in zip(t.shape[:3], t.stride()[:3]) if n > 1):
                raise ValueError(f"{name} must be 16-byte aligned, with strides that keep it so")
            reach = dim
            for n, s in sorted(zip(t.shape[:3], t.stride()[:3]), key=lambda ns: ns[1]):
                if n > 1 and s < reach:
                    raise ValueError(f"{name} has places that share memory")
                if n > 1:
                    reach = s * (n - 1) + reach
        if torch.cuda.is_available():
            _workspace(k_pages.get_device())      # there before the first call, which may be captured: a graph's own memory goes with it
        self._k_pages, self._v_pages = k_pages, v_pages

    k_pages = property(lambda self: self._k_pages)
    v_pages = property(lambda self: self._v_pages)
    pages = property(lambda self: self.k_pages.shape[0])
    page_size = property(lambda self: self.k_pages.shape[1])
    kv_heads = property(lambda self: self.k_pages.shape[2])
    head_dim = property(lambda self: self.k_pages.shape[3])


# The checks below are written out, tensor by tensor: as functions they were a third of the ten microseconds that a call took on the host.

def _refuse_heads(t, name: str):
    """Says what is wrong with what should have been ``[tokens, heads, head_dim]`` on a GPU."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must have the dimensions [tokens, heads, head_dim]")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    raise ValueError(f"{name} must have unit stride along its last dimension")


def _head_weight(t, name: str, dim: int, index: int) -> tuple[int, int]:
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES or t.dim() != 1 or t.numel() != dim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bfloat16, float16 or float32 vector of {dim} values")
    if t.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    return t.data_ptr(), _DTYPES[t.dtype]


def _rotate(q, k, v, positions, rotary, cache, slots, q_weight, k_weight, eps):
    for t, name in ((q, "q"), (k, "k")):
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            _refuse_heads(t, name)
    (tokens, q_heads, dim), (k_tokens, kv_heads, k_dim) = q.shape, k.shape
    (q_token, q_head, q_unit), (k_token, k_head, k_unit) = q.stride(), k.stride()
    dtype, index = q.dtype, q.get_device()
    kind = _DTYPES.get(dtype)
    if kind is None or index < 0 or (q_unit != 1 and dim > 1):
        _refuse_heads(q, "q")
    if k_tokens != tokens or k_dim != dim or k.dtype is not dtype:
        raise ValueError("q and k must have the same tokens, head_dim and dtype")
    if k_unit != 1 and dim > 1:
        _refuse_heads(k, "k")
    if not 0 < q_heads <= _MOST_HEADS or not 0 < kv_heads <= _MOST_HEADS or not 0 < dim <= _MOST_DIM:
        raise ValueError(f"there must be 1 to {_MOST_HEADS} heads of 1 to {_MOST_DIM} values")
    if not isinstance(rotary, Rotary):
        raise ValueError("rotary must be a Rotary")
    turned, turns, axis = rotary.dims, rotary._turns, rotary._axis
    if turned > dim:
        raise ValueError(f"rotary turns {turned} values, a head has {dim}")
    if not isinstance(positions, torch.Tensor) or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 or int64 tensor")
    wide, shape = positions.dtype is torch.int64, positions.shape
    if not wide and positions.dtype is not torch.int32:
        raise ValueError("positions must be a contiguous int32 or int64 tensor")
    if len(shape) not in (1, 2) or shape[-1] != tokens or (shape[0] if len(shape) == 2 else 1) < rotary.axes:
        raise ValueError(f"positions must be [{tokens}] or, with a row for each of {rotary.axes} axes, [axes, {tokens}]")
    if k.get_device() != index or positions.get_device() != index or turns.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    qw = kw = weight_kind = 0
    if q_weight is not None:
        qw, weight_kind = _head_weight(q_weight, "q_weight", dim, index)
    if k_weight is not None:
        q_kind = weight_kind
        kw, weight_kind = _head_weight(k_weight, "k_weight", dim, index)
        if qw and q_kind != weight_kind:
            raise ValueError("q_weight and k_weight must have the same dtype")
    if cache is None:
        k_out = k.new_empty(tokens, kv_heads, dim)
        k_ptr, v_ptr, v_out, slots_ptr = k_out.data_ptr(), 0, 0, 0
        v_token = v_head = k_page = k_slot = k_place = v_page = v_slot = v_place = pages = page_size = 0
    else:
        if not isinstance(cache, KvCache):
            raise ValueError("cache must be a KvCache")
        if not isinstance(v, torch.Tensor) or v.dim() != 3:
            _refuse_heads(v, "v")
        if v.shape != k.shape or v.dtype is not dtype:
            raise ValueError("k and v must have the same shape and dtype")
        v_token, v_head, v_unit = v.stride()
        if v_unit != 1 and dim > 1:
            _refuse_heads(v, "v")
        k_out, v_pages = cache._k_pages, cache._v_pages
        pages, page_size, cache_heads, cache_dim = k_out.shape
        if cache_heads != kv_heads or cache_dim != dim or k_out.dtype is not dtype:
            raise ValueError("the cache must have the heads, head_dim and dtype of k")
        k_page, k_slot, k_place, _ = k_out.stride()
        v_page, v_slot, v_place, _ = v_pages.stride()
        if not isinstance(slots, torch.Tensor) or slots.dtype is not torch.int64 or slots.dim() != 1 or slots.numel() != tokens or not slots.is_contiguous():
            raise ValueError(f"slots must be a contiguous int64 vector of {tokens} values")
        if v.get_device() != index or k_out.get_device() != index or slots.get_device() != index:
            raise ValueError("all tensors must be on the same CUDA device")
        k_ptr, v_ptr, v_out, slots_ptr = k_out.data_ptr(), v.data_ptr(), v_pages.data_ptr(), slots.data_ptr()
    q_out = q.new_empty(tokens, q_heads, dim)
    args = _lib.HEAD_ROTATE.pack(q.data_ptr(), k.data_ptr(), v_ptr, q_out.data_ptr(), k_ptr, v_out, qw, kw, positions.data_ptr(), turns.data_ptr(),
                                 0 if axis is None else axis.data_ptr(), slots_ptr, tokens, q_token, q_head, k_token, k_head, v_token, v_head, k_page, k_slot,
                                 k_place, v_page, v_slot, v_place, pages, page_size, q_heads, kv_heads, dim, turned, rotary.interleaved, wide, kind, weight_kind,
                                 eps, rotary.scale)
    if _current_device() == index:
        rc = _lib.load().mps_head_rotate_rows(args, _stream_of(index))
        if rc:
            _lib.check(rc)
    else:
        _launch(index, "mps_head_rotate_rows", args)
    return q_out, k_out


def norm_rotate(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, *, q_weight: torch.Tensor | None = None,
                k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries ``[tokens, q_heads, dim]`` and keys ``[tokens, kv_heads, dim]``, each head normalised (``x * rsqrt(mean(x^2) + eps) * weight``, where a weight ``[dim]`` is
    given) and rotated by its token's position; new, contiguous tensors of the same dtype.

    ``q`` and ``k`` may be views of one projection's result (unit stride along ``dim``).  ``positions``: int32 or int64, ``[tokens]`` or ``[axes, tokens]``.  Angles are
    products in 64 bits taken modulo a turn: off by 2^-51 of the whole angle, ``position * frequency``, which FP32 does not show up to 2^27, and beyond that by FP32's rounding of
    what is left of it.  All else is FP32, rounded once."""
    return _rotate(q, k, None, positions, rotary, None, None, q_weight, k_weight, eps)


def norm_rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, rotary: Rotary, cache: KvCache, slots: torch.Tensor, *,
                       q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """``norm_rotate`` whose keys go into the cache, with the values ``v``: those of token ``t`` at slot ``slots[t]`` (int64).  Returns the queries.

    A slot outside the cache (as -1 for a padded token) is not written.  Where two tokens of a call have the same slot, it holds either's
    values, or some of each.  The cache must not share memory with ``q``, ``k`` or ``v``."""
    if cache is None:
        raise ValueError("cache must be a KvCache")
    return _rotate(q, k, v, positions, rotary, cache, slots, q_weight, k_weight, eps)[0]


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(index: int, batch, table_columns, prefix, page_size, q_heads, kv_heads, dim, dtype) -> int:
    args = _lib.PREFIX_ATTEND.pack(0, 0, 0, 0, 0, 0, 0, 0, batch, table_columns, prefix, 0, page_size, 0, 0, 0, 0, 0, 0, 0, 0, q_heads, kv_heads, dim, dtype, 1.0)
    with torch.cuda.device(index):
        need = int(_lib.load().mps_prefix_attend_scratch_bytes(args))
    if need < 0:
        raise ValueError(_lib.load().mps_last_error().decode(errors="replace"))
    return need


def shared_prefix_attention(q: torch.Tensor, cache: KvCache, tables: torch.Tensor, lengths: torch.Tensor, *, prefix_table: torch.Tensor | None = None,
                            prefix_length: int = 0, scale: float | None = None, return_lse: bool = False):
    """``softmax(scale * q k^T) v`` for one query per sequence and head, over a prefix that all sequences share and tokens of each one's own: ``[batch, q_heads, dim]``.

    ``q`` ``[batch, q_heads, dim]`` in the cache's dtype, ``q_heads`` a multiple of the cache's heads (neighbouring ones share a key head), ``dim`` 64 or 128; a page has 16
    tokens at least.  Sequence ``b`` has ``lengths[b]`` (int32, on the device) tokens of its own, in the pages ``tables[b]`` (int32 ``[batch, n]``); the prefix has
    ``prefix_length`` tokens in the pages ``prefix_table`` (int32).  The prefix is read once for the whole batch.  ``scale`` is by default ``dim ** -0.5``.

    A length below 0 counts as 0, one beyond its table as the table; keys of a page outside the cache are absent.  A query with nothing to attend to gets zeros.
    Softmax and sums are FP32; the weights of the values are rounded to the cache's dtype before they multiply them.
    With ``return_lse`` also the FP32 logarithms of the softmax's denominators, ``[batch, q_heads]``."""
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        _refuse_heads(q, "q")
    batch, q_heads, dim = q.shape
    q_token, q_head, q_unit = q.stride()
    dtype, index = q.dtype, q.get_device()
    if index < 0 or q_unit != 1:
        _refuse_heads(q, "q")
    if not isinstance(cache, KvCache):
        raise ValueError("cache must be a KvCache")
    k_pages, v_pages = cache._k_pages, cache._v_pages
    pages, page_size, kv_heads, cache_dim = k_pages.shape
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("q must be bfloat16 or float16")
    if k_pages.dtype is not dtype or cache_dim != dim:
        raise ValueError("q must have the dtype and head_dim of the cache")
    if dim != 64 and dim != 128:
        raise ValueError("head_dim must be 64 or 128")
    if page_size < 16 or page_size > 1 << 20:
        raise ValueError("a page must have 16 to 2^20 tokens")
    if q_heads < 1 or q_heads > _MOST_HEADS or q_heads % kv_heads:
        raise ValueError(f"q_heads must be a multiple of the cache's {kv_heads} heads, at most {_MOST_HEADS}")
    if batch > _MOST_SEQUENCES:
        raise ValueError(f"a batch has at most {_MOST_SEQUENCES} sequences")
    if not isinstance(tables, torch.Tensor) or tables.dtype is not torch.int32 or tables.dim() != 2 or not tables.is_contiguous():
        raise ValueError(f"tables must be a contiguous int32 matrix of {batch} rows")
    table_rows, columns = tables.shape
    if table_rows != batch:
        raise ValueError(f"tables must be a contiguous int32 matrix of {batch} rows")
    if not isinstance(lengths, torch.Tensor) or lengths.dtype is not torch.int32 or lengths.dim() != 1 or lengths.numel() != batch or not lengths.is_contiguous():
        raise ValueError(f"lengths must be a contiguous int32 vector of {batch} values")
    prefix_length, prefix_ptr = int(prefix_length), 0
    if prefix_length < 0:
        raise ValueError("prefix_length must not be negative")
    if prefix_length:
        if (not isinstance(prefix_table, torch.Tensor) or prefix_table.dtype is not torch.int32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous()
                or prefix_table.numel() * page_size < prefix_length):
            raise ValueError(f"prefix_table must be a contiguous int32 vector with the pages of {prefix_length} tokens")
        if prefix_table.get_device() != index:
            raise ValueError("all tensors must be on the same CUDA device")
        prefix_ptr = prefix_table.data_ptr()
    if columns * page_size > _MOST_KEYS or prefix_length > _MOST_KEYS:
        raise ValueError("a table and the prefix may have at most 2^30 tokens")
    if k_pages.get_device() != index or tables.get_device() != index or lengths.get_device() != index:
        raise ValueError("all tensors must be on the same CUDA device")
    at = q.data_ptr()
    if at % 16 or (q_token % 8 and batch > 1) or (q_head % 8 and q_heads > 1):
        raise ValueError("q must be 16-byte aligned, with strides that keep it so")
    k_page, k_slot, k_place, _ = k_pages.stride()
    v_page, v_slot, v_place, _ = v_pages.stride()
    out = q.new_empty(batch, q_heads, dim)
    lse = q.new_empty(batch, q_heads, dtype=torch.float32) if return_lse else None
    if batch:
        kind = _DTYPES[dtype]
        need = _scratch_bytes(index, batch, columns, prefix_length, page_size, q_heads, kv_heads, dim, kind)
        scratch = q.new_empty(need, dtype=torch.uint8)      # of this call: freed on return, and not handed to another stream before it is done
        ws = _workspace(index)
        args = _lib.PREFIX_ATTEND.pack(at, k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                                       tables.data_ptr(), lengths.data_ptr(), prefix_ptr, batch, columns, prefix_length, pages, page_size, q_token, q_head,
                                       k_page, k_slot, k_place, v_page, v_slot, v_place, q_heads, kv_heads, dim, kind, dim ** -0.5 if scale is None else scale)
        if _current_device() == index:
            rc = _lib.load().mps_prefix_attend_tokens(args, scratch.data_ptr(), need, ws.data_ptr(), ws.numel(), _stream_of(index))
            if rc:
                _lib.check(rc)
        else:
            _launch(index, "mps_prefix_attend_tokens", args, scratch.data_ptr(), need, ws.data_ptr(), ws.numel())
    return (out, lse) if return_lse else out
