"""``GatedMlp`` against 64 bits.

What passes between its first operators is in 4 bits, a code apart where two evaluations fall on either side of a halfway point; those operators alone
give the same codes (they are the same kernels), so the formula starts from them.  From there on, off by at most:

  the block's result y: (inter / 32 + 4) 2^-23 of the sum of magnitudes (a step of the tensor cores as two additions, four parts), and
  ROUND of y where it is rounded to 16 bits;
  t = gate * norm(y): 84 roundings of 2^-24 of itself (tests/test_mx4_norm_gpu.py), and what y's error makes of it: by its share of the row's root mean
  square, and of the mean, to the first order and 2^-6 of that for the higher ones (y is off by 2^-8 of itself at most);
  n: the same again with h' in y's place.
"""
import numpy as np
import pytest
import torch

from mpserve_b200 import mx4
from tests import _mx4 as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


def _randn(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * scale


def _through_norm(v, dv, w, eps):
    """norm(v) * w and how far it is off where v is off by dv."""
    rms = np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)
    out = v / rms * w
    return out, (dv / rms * np.abs(w) + np.abs(out) * (dv * np.abs(v)).mean(axis=1, keepdims=True) / rms ** 2) * (1 + 2.0 ** -6) + np.abs(out) * 80 * U


def _check(block, h, down_scale=1.0):
    joined, n = block(h)
    wide = block.result_dtype is torch.float32
    kept = torch.float32 if wide else torch.bfloat16 if h.dtype == torch.float32 else h.dtype
    assert joined.dtype == h.dtype and n.dtype == (h.dtype if wide else kept)
    x = mx4.rms_norm(h, block.pre_weight, eps=EPS, quantized=True)
    a = ref.values(mx4.gated_linear(x, block.gate_proj, block.up_proj, quantized=True))
    d, h64, eps = ref.values(block.down_proj), ref.to64(h), float(np.float32(EPS))
    y = a @ d.T
    dy = np.abs(a) @ np.abs(d).T * ((a.shape[1] / 32 + 4) * 2.0 ** -23) + (0 if wide else np.abs(y) * ref.ROUND[kept])
    if kept == torch.float16:
        dy = dy + 2.0 ** -25
    t, dt = (y, dy) if block.post_weight is None else _through_norm(y, dy, ref.to64(block.post_weight), eps)
    if block.gate is not None:
        g = ref.to64(block.gate)
        t, dt = t * g, dt * np.abs(g)
    want = h64 + t
    off = dt + (np.abs(h64) + np.abs(t)) * 4 * U
    least = 2.0 ** -25 if h.dtype == torch.float16 else 0.0
    assert (np.abs(ref.to64(joined) - want) <= off + (np.abs(want) + off) * ref.ROUND[h.dtype] + least).all()
    nw, n_off = _through_norm(want, off, ref.to64(block.next_weight), eps)
    least = 2.0 ** -25 if n.dtype == torch.float16 else 0.0
    assert (np.abs(ref.to64(n) - nw) <= n_off + (np.abs(nw) + n_off) * ref.ROUND[n.dtype] + least).all()
    assert mx4.product_timed_out() is False
    return y, joined, n


def _block(hidden, inter, stream, seed, post=True, gate=True, scales=(0.05, 0.05, 0.05), **kw):
    w = [mx4.quantize(_randn(s, seed + i, scales[i])) for i, s in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    vec = [_randn((hidden,), seed + 10 + i, 0.1).to(torch.bfloat16) + 1 for i in range(3)]
    return mx4.GatedMlp(*w, pre_weight=vec[0], post_weight=vec[1] if post else None, next_weight=vec[2],
                        gate=_randn((hidden,), seed + 20).to(torch.bfloat16) if gate else None, eps=EPS, **kw)


@pytest.mark.parametrize("result", [None, torch.float32])
@pytest.mark.parametrize("stream", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,hidden,inter", [(1, 256, 640), (8, 300, 1000), (20, 1000, 385), (64, 256, 512), (70, 331, 700), (200, 512, 640), (700, 517, 300)])
def test_block(tokens, hidden, inter, stream, result):
    h = _randn((tokens, hidden), tokens).to(ref.TYPES[stream])
    ref.poison()
    _check(_block(hidden, inter, stream, 100, result_dtype=result), h)
    _check(_block(hidden, inter, stream, 200, post=False, gate=False, result_dtype=result), h)


@pytest.mark.parametrize("result", [None, torch.float32])
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_results_beyond_f16(tokens, result):
    """A block whose result leaves F16's range inside: its norm brings it back, and the stream is what the formula says."""
    h = _randn((tokens, 256), 5).to(torch.float16)
    block = _block(256, 640, "f16", 300, scales=(2.0, 2.0, 4.0), result_dtype=result)
    y, joined, n = _check(block, h)
    assert (np.abs(y) > 65504).any(axis=1).all()
    assert joined.isfinite().all() and n.isfinite().all()
    # an infinity that is the formula's own stays one
    h[0, 3] = float("inf")
    joined, n = block(h)
    assert n[0].isnan().any() and joined[1:].isfinite().all() and n[1:].isfinite().all()


def test_a_result_dtype_that_is_not_served():
    with pytest.raises(ValueError, match="None or float32"):
        _block(64, 64, "bf16", 1, result_dtype=torch.float64)
