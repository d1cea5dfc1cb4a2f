"""Products and quantisation where earlier bounds leave room: sums of four parts at most, and the edges of F16's range.

A step of the tensor cores adds 64 products to an FP32 accumulator; taking each of its two blocks of 32 as one rounded or cut addition, and an addition for
each of the four parts that several CTAs may add up, a sum over ``cols`` is off by at most (cols / 32 + 4) 2^-23 of the sum of magnitudes.  The result
rounds to its type.
"""
import numpy as np
import pytest
import torch

from mpserve_b200 import mx4
from tests import _mx4 as ref
from tests.test_mx4_convert_gpu import _same

pytestmark = pytest.mark.gpu


def _pair(tokens, cols, rows, seed):
    """Operands whose sums cancel: the second half of the columns takes the first half's sums back but for a small part."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    half = cols // 2
    x = torch.randn((tokens, cols), generator=g, device="cuda") * torch.exp2(torch.randint(-3, 4, (tokens, cols), generator=g, device="cuda").float())
    w = torch.randn((rows, cols), generator=g, device="cuda")
    x[:, half:2 * half] = x[:, :half]
    w[:, half:2 * half] = -w[:, :half] * torch.where(torch.rand((rows, half), generator=g, device="cuda") < 0.03, 0.5, 1.0)
    return mx4.quantize(x), mx4.quantize(w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,cols,rows", [(1, 256, 128), (1, 4096, 1000), (7, 2048, 300), (16, 8192, 128), (20, 1024, 517), (32, 4096, 256), (64, 2048, 384),
                                              (100, 6144, 130), (128, 512, 1000), (257, 1024, 511), (1025, 2048, 700), (3, 30000, 40)])
def test_sums_that_cancel(tokens, cols, rows, dtype):
    xq, wq = _pair(tokens, cols, rows, tokens + cols)
    x, w = (torch.from_numpy(ref.values(q)).cuda() for q in (xq, wq))
    want = x @ w.t()
    off = (x.abs() @ w.abs().t()) * ((cols / 32 + 4) * 2.0 ** -23) + want.abs() * ref.ROUND[dtype] * (1 + 2.0 ** -8) + (2.0 ** -25 if dtype == torch.float16 else 0)
    y = mx4.linear(xq, wq, dtype=dtype)
    worst = ((y.double() - want).abs() / off.clamp_min(1e-300)).max().item()
    assert worst <= 1, worst
    a = mx4.gated_linear(xq, wq, wq, dtype=dtype)
    g = want
    da = 1.13 * (off - want.abs() * ref.ROUND[dtype]) + (g * torch.sigmoid(g)).abs() * 2.0 ** -19      # tests/test_mx4_product_gpu.py
    exact = g * torch.sigmoid(g) * g
    bound = da * (g.abs() + off) + (g * torch.sigmoid(g)).abs() * off + exact.abs() * ref.ROUND[dtype] * (1 + 2.0 ** -8) + (2.0 ** -25 if dtype == torch.float16 else 0)
    held = exact.abs() < 60000 if dtype == torch.float16 else torch.ones_like(exact, dtype=torch.bool)
    assert ((a.double() - exact).abs() <= bound)[held].all()


def _rows(dtype):
    t = torch.finfo(dtype)
    r = [
        [float("nan") if i == 17 else 1.0 for i in range(32)], [float("inf") if i == 31 else 1.0 for i in range(32)],
        [-float("inf") if i == 0 else 1.0 for i in range(32)], [float("nan")] * 32, [float("inf")] * 32,
        [t.max if i == 3 else t.max / 64 * i for i in range(32)], [-t.max] * 32, [t.max if i % 2 else -t.max / 2 for i in range(32)],
        [t.tiny * (1 + i / 32) for i in range(32)], [t.smallest_normal / 1024 * i for i in range(32)], [t.smallest_normal / 1024] * 32,
        [t.smallest_normal / 1024 if i == 9 else 0.0 for i in range(32)], [0.0] * 32, [-0.0] * 32,
        # every halfway point, both signs, under the scale 1, and their neighbours
        [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.0, 7.0, 7.9375, -7.5] + [0.0] * 13,
        [4.0] + [v * s for v in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0) for s in (1 - 2.0 ** -7, 1 + 2.0 ** -7)] + [0.0] * 17,
        [(2 - 2.0 ** -7)] + [0.25] * 31, [2.0] + [0.25] * 31,
    ]
    return torch.tensor(r, dtype=torch.float64).to(dtype).cuda()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_edges_of_every_type_in_short_long_and_unaligned_rows(dtype):
    x = _rows(ref.TYPES[dtype])
    wide = x.repeat(1, 33)
    shifted = torch.zeros((x.shape[0], 33 * 32 + 3), dtype=x.dtype, device="cuda")
    shifted[:, 3:] = wide
    for v in (x, x[:, :31], wide, wide[:, :1000], wide[:, :1055], shifted[:, 3:], torch.cat([x, x.flip(0)], 1)):
        ref.poison()
        q = mx4.quantize(v)
        _same(q, ref.to64(v))
        np.testing.assert_array_equal(ref.to64(q.dequantize(torch.float32)), ref.values(q))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_products_quantise_the_edges_alike(dtype):
    """Up to eight tokens by the product's kernel, more by one before it: the same as quantised tokens give."""
    x = _rows(ref.TYPES[dtype]).repeat(1, 20)
    w = mx4.quantize(torch.randn((140, x.shape[1]), device="cuda"))
    for v in (x[:8], x[8:16], x[10:], x, x[5:6], x[:, :600][:7]):
        u = w if v.shape[1] == x.shape[1] else mx4.quantize(torch.randn((140, v.shape[1]), device="cuda"))
        got, want = mx4.linear(v, u, dtype=torch.bfloat16), mx4.linear(mx4.quantize(v), u)
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
        got, want = mx4.gated_linear(v, u, u, dtype=torch.bfloat16), mx4.gated_linear(mx4.quantize(v), u, u)
        torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)
