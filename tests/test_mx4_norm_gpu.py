"""Norms, gate and residual against the formula in 64 bits.

Off by at most: each factor of a value rounds once in FP32 (2^-24); a mean of n squares summed in any order is off by n 2^-24 of itself at most,
here by log2(n) + 8 roundings along the longest path (eight per lane and step, up to eight steps in a row, then a tree), half of
which reach the root; then the result rounds to its type.
"""
import numpy as np
import pytest
import torch

from mpserve_b200 import mx4
from tests import _mx4 as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _norm(x, w, eps):
    return x / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps) * (1 if w is None else w)


def _make(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(ref.TYPES[dtype])


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 31), (7, 33), (130, 255), (5, 256), (2, 257), (9, 1000), (3, 4097), (2, 8192), (2, 16384), (1, 32768)])
def test_rms_norm(rows, cols, dtype, quantized):
    h, w = _make((rows, cols), dtype, cols), _make((cols,), "bf16", cols + 1) + 1
    ref.poison()
    n = mx4.rms_norm(h, w, eps=1e-6, quantized=quantized)
    want = _norm(ref.to64(h), ref.to64(w), float(np.float32(1e-6)))
    off = np.abs(want) * 80 * U
    if quantized:
        ref.check_rounded(n, want, off)
    else:
        assert n.dtype == h.dtype
        small = 2.0 ** -25 if dtype == "f16" else 0.0        # half of F16's least number
        assert (np.abs(ref.to64(n) - want) <= off + np.abs(want) * ref.ROUND[h.dtype] * (1 + 2.0 ** -8) + small).all()


@pytest.mark.parametrize("rows,cols,dtype,stream,gate,post,nxt,alpha,quantized", [
    (1, 4096, "bf16", "bf16", "column", True, True, 1.0, False),
    (1, 4096, "bf16", "bf16", "column", True, True, 1.0, True),
    (5, 1000, "f16", "f32", "row", True, True, 0.75, False),
    (133, 257, "bf16", "f32", "full", False, True, 1.0, True),
    (133, 256, "f16", "f16", "none", True, True, 0.5, True),
    (64, 33, "f32", "f32", "full", True, True, 1.0, False),
    (3, 31, "bf16", "bf16", "row", False, False, 2.0, False),
    (2, 8192, "f16", "f16", "one", True, False, 0.0, False),
    (4, 1, "f32", "bf16", "full", True, True, 1.0, False),
    (2, 12345, "bf16", "f32", "column", True, True, 1.0, False),
    (2, 32768, "bf16", "f32", "full", True, True, 1.0, True),
])
def test_block_join(rows, cols, dtype, stream, gate, post, nxt, alpha, quantized):
    y, h = _make((rows, cols), dtype, 1, 3.0), _make((rows, cols), stream, 2)
    pw, nw = (_make((cols,), "bf16", 3) + 1 if post else None), (_make((cols,), "bf16", 4) + 1 if nxt else None)
    shape = {"none": None, "one": (1,), "column": (cols,), "row": (rows, 1), "full": (rows, cols)}[gate]
    g = None if shape is None else _make(shape, "bf16" if gate == "full" else "f32", 5)
    eps = float(np.float32(1e-5))
    y64, h64 = ref.to64(y), ref.to64(h)
    t = _norm(y64, ref.to64(pw), eps) if post else y64
    t = t if g is None else t * ref.to64(g)
    joined = alpha * h64 + t
    off = (np.abs(alpha * h64) + np.abs(t)) * 84 * U
    for inplace in (False, True):
        ref.poison()
        stream_in = h.clone()
        got, n = mx4.block_join(y, stream_in, post_weight=pw, gate=g, residual_scale=alpha, next_weight=nw, eps=1e-5, quantized=quantized,
                                inplace=inplace)
        assert (got is stream_in) == inplace and (n is None) == (not nxt)
        if not inplace:
            assert torch.equal(stream_in, h)
        least = 2.0 ** -25 if stream == "f16" else 0.0
        assert (np.abs(ref.to64(got) - joined) <= off + np.abs(joined) * ref.ROUND[h.dtype] * (1 + 2.0 ** -8) + least).all()
        if not nxt:
            continue
        want = _norm(joined, ref.to64(nw), eps)
        # the stream's own error passes through the norm: by its share of the row's root mean square, and of the mean
        rms = np.sqrt((joined ** 2).mean(axis=1, keepdims=True) + eps)
        n_off = off / rms * np.abs(ref.to64(nw)) + np.abs(want) * (80 * U + (off * np.abs(joined)).mean(axis=1, keepdims=True) / rms ** 2)
        if quantized:
            ref.check_rounded(n, want, n_off)
        else:
            least = 2.0 ** -25 if dtype == "f16" else 0.0
            assert n.dtype == y.dtype
            assert (np.abs(ref.to64(n) - want) <= n_off + np.abs(want) * ref.ROUND[y.dtype] * (1 + 2.0 ** -8) + least).all()


@pytest.mark.parametrize("rows,cols", [(1000, 40), (515, 256), (700, 300), (600, 500), (513, 2000), (600, 2056), (520, 9000), (530, 1337)])
def test_many_rows_are_each_themselves(rows, cols):
    """Rows that share a CTA, and the last CTA's missing ones: what a row gives does not depend on its neighbours."""
    y, h = _make((rows, cols), "bf16", 6), _make((rows, cols), "f32", 7)
    w = _make((cols,), "f32", 8) + 1
    g = _make((rows, 1), "f32", 9)
    guard = torch.full((rows + 8, cols), 7.0, device="cuda")
    guard[:rows] = h
    joined, n = mx4.block_join(y, guard[:rows], post_weight=w, gate=g, next_weight=w, inplace=True)
    assert (guard[rows:] == 7).all()
    q = mx4.rms_norm(h, w, quantized=True).dequantize()
    for first in (0, 17, rows - 3):
        some = slice(first, first + 3)
        few = mx4.block_join(y[some], h[some], post_weight=w, gate=g[some], next_weight=w)
        torch.testing.assert_close(joined[some], few[0], rtol=2.0 ** -20, atol=2.0 ** -18)
        torch.testing.assert_close(n[some], few[1], rtol=2.0 ** -7, atol=2.0 ** -18)
        assert torch.isfinite(q[some]).all()
    want = _norm(ref.to64(h), ref.to64(w), float(np.float32(1e-5)))
    ref.check_rounded(mx4.rms_norm(h, w, quantized=True), want, np.abs(want) * 80 * U)


def test_rows_of_zeros_and_of_nan_keep_to_themselves():
    h = torch.randn((4, 512), device="cuda").to(torch.bfloat16)
    h[1], h[2, 7] = 0, float("nan")
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    n = mx4.rms_norm(h, w, eps=1e-5)
    assert (n[1] == 0).all() and n[2].isnan().all() and n[0].isfinite().all() and n[3].isfinite().all()
    q = mx4.rms_norm(h, w, eps=1e-5, quantized=True).dequantize()
    assert (q[1] == 0).all() and q[2].isnan().all() and q[0].isfinite().all() and q[3].isfinite().all()


def test_strides_shapes_and_no_rows():
    whole = torch.randn((12, 1200), device="cuda").to(torch.bfloat16)
    w = torch.rand(500, device="cuda") + 0.5
    for view in (whole[:, 8:508], whole[:, 3:503], whole[::3, :500]):
        assert torch.equal(mx4.rms_norm(view, w), mx4.rms_norm(view.contiguous(), w))
        joined, n = mx4.block_join(view, view, gate=w, next_weight=w)
        same = mx4.block_join(view.contiguous(), view.contiguous(), gate=w, next_weight=w)
        assert torch.equal(joined, same[0]) and torch.equal(n, same[1])
    cube = whole[:, :500].contiguous().view(3, 4, 500)
    gate = torch.randn((3, 4, 1), device="cuda")
    joined, n = mx4.block_join(cube, cube, gate=gate, next_weight=w)
    flat = mx4.block_join(cube.view(12, 500), cube.view(12, 500), gate=gate.view(12, 1), next_weight=w)
    assert joined.shape == cube.shape and torch.equal(joined.view(12, 500), flat[0]) and torch.equal(n.view(12, 500), flat[1])
    none = whole[:0, :500]
    joined, n = mx4.block_join(none, none, next_weight=w)
    assert joined.shape == n.shape == (0, 500)


def test_refusals():
    h = torch.zeros((4, 64), device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda")
    for call, match in (
            (lambda: mx4.rms_norm(h.cpu(), w), "CUDA tensor"),
            (lambda: mx4.rms_norm(h, w[:63]), "vector of 64"),
            (lambda: mx4.rms_norm(h, w.cpu()), "same CUDA device"),
            (lambda: mx4.rms_norm(h, w.double()), "weight must be"),
            (lambda: mx4.rms_norm(h, w, dtype=torch.int8), "dtype"),
            (lambda: mx4.rms_norm(torch.zeros((1, 32769), device="cuda"), torch.zeros(32769, device="cuda")), "32768"),
            (lambda: mx4.block_join(h, h[:3]), "same shape"),
            (lambda: mx4.block_join(h, h, gate=torch.zeros((3, 1), device="cuda")), "gate must be contiguous"),
            (lambda: mx4.block_join(h, h, gate=torch.zeros((64, 4), device="cuda").t()), "gate must be contiguous"),
            (lambda: mx4.block_join(h, h, gate=torch.zeros(64)), "same CUDA device"),
            (lambda: mx4.block_join(h, h, post_weight=w, next_weight=w.half()), "same dtype"),
            (lambda: mx4.block_join(h, h[:1].expand(4, 64), inplace=True), "share memory")):
        with pytest.raises(ValueError, match=match):
            call()
