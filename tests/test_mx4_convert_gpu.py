"""MXFP4 quantisation, its ways back and the tiles: byte for byte against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from mpserve_b200 import mx4
from tests import _mx4 as ref

pytestmark = pytest.mark.gpu


def _same(q, x64):
    codes, scales = ref.encode(x64)
    got_codes, got_scales = (t.cpu().numpy() for t in q.parts())
    np.testing.assert_array_equal(got_scales, scales)
    # -0 and 0 are one value; the codes of a block that is NaN say nothing
    mine, want = ref.unpack(got_codes, q.cols), codes.copy()
    zero = ((mine & 7) == 0) & ((want & 7) == 0)
    nan = np.repeat(scales == 255, 32, axis=1)[:, :q.cols]
    np.testing.assert_array_equal(np.where(zero | nan, 0, mine), np.where(zero | nan, 0, want))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 31), (127, 32), (128, 33), (129, 255), (2, 256), (300, 257), (64, 1000), (5, 1025),
                                       (257, 1337), (2, 5121)])
def test_quantize_and_back(rows, cols, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows * 7919 + cols)
    x = (torch.randn((rows, cols), generator=g, device="cuda") * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g, device="cuda").float())).to(ref.TYPES[dtype])
    ref.poison()
    q = mx4.quantize(x)
    assert q.shape == (rows, cols)
    _same(q, ref.to64(x))
    want = ref.values(q)
    np.testing.assert_array_equal(ref.to64(q.dequantize()), want)
    np.testing.assert_array_equal(ref.to64(q.dequantize(torch.float32)), want)
    half = torch.from_numpy(want).to(torch.float16)
    assert torch.equal(q.dequantize(torch.float16).cpu(), half)
    assert mx4.product_timed_out() is False


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1024), (3, 784), (130, 1040), (5, 1296), (7, 1536), (2, 1808), (33, 2064), (1, 8192), (9, 4080)])
def test_long_rows(rows, cols, dtype):
    """Rows of four pieces and more, a multiple of 16 columns: every number of tiles that the last step of a warp can have."""
    x = torch.randn((rows, cols), device="cuda") * torch.exp2(torch.randint(-12, 12, (rows, cols), device="cuda").float())
    x[0, ::37] = 0
    x = x.to(ref.TYPES[dtype])
    ref.poison()
    q = mx4.quantize(x)
    _same(q, ref.to64(x))
    np.testing.assert_array_equal(ref.to64(q.dequantize()), ref.values(q))
    np.testing.assert_array_equal(ref.to64(q.dequantize(torch.float32)), ref.values(q))
    # the columns that fill up the last tile are zeros of the least scale: rows of garbage there would show in a product
    w = mx4.quantize(torch.ones((4, cols), device="cuda"))
    assert mx4.linear(q, w).isfinite().all()


def _edge_rows(t):
    return [
        [0.0] * 32, [-0.0] * 32,
        [2.0 ** e for e in range(-16, 16)],
        [2.0 ** -126 * (1 + i / 32) for i in range(32)],
        [2.0 ** -133 * i for i in range(32)],                        # subnormal in both types
        [2.0 ** -127 * i / 4 for i in range(32)],
        [(2 - 2.0 ** -7) * 2.0 ** 127 if i == 3 else 2.0 ** 125 * i for i in range(32)],     # up to the largest
        [float("nan") if i == 17 else 1.0 for i in range(32)],
        [float("inf") if i == 31 else 1.0 for i in range(32)],
        [-float("inf") if i == 0 else 1.0 for i in range(32)],
        # every halfway point, both signs, under the scale 1
        [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.0, 7.0, 7.9375, -7.5] + [0.0] * 13,
        # and their neighbours
        [4.0] + [v * s for v in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0) for s in (1 - 2.0 ** -7, 1 + 2.0 ** -7)] + [0.0] * 17,
        # a largest value just below and at a power of two
        [(2 - 2.0 ** -7)] + [0.25] * 31, [2.0] + [0.25] * 31,
    ]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_edges_of_the_number_range(dtype):
    t = ref.TYPES[dtype]
    rows = _edge_rows(t)
    for x in (torch.tensor(rows, dtype=torch.float64), torch.tensor(rows, dtype=torch.float64).repeat(1, 33)):      # short rows and long ones
        x = x.to(t).cuda()
        q = mx4.quantize(x)
        _same(q, ref.to64(x))
        np.testing.assert_array_equal(ref.to64(q.dequantize(torch.float32)), ref.values(q))
        np.testing.assert_array_equal(ref.to64(q.dequantize()), ref.values(q))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strided_and_shaped_inputs(dtype):
    t = ref.TYPES[dtype]
    whole = torch.randn((70, 1100), device="cuda").to(t)
    for view in (whole[:, 8:8 + 512], whole[:, 3:3 + 700], whole[::2], whole[5:6, 1:1 + 40], whole[3:4].expand(9, 1100)):
        _same(mx4.quantize(view), ref.to64(view))
    cube = torch.randn((3, 5, 96), device="cuda").to(t)
    q = mx4.quantize(cube)
    assert q.shape == (3, 5, 96) and q.dequantize().shape == (3, 5, 96)
    _same(q, ref.to64(cube.reshape(15, 96)))
    vector = torch.randn((77,), device="cuda").to(t)
    assert mx4.quantize(vector).dequantize().shape == (77,)
    empty = mx4.quantize(torch.empty((0, 64), dtype=t, device="cuda"))
    assert empty.dequantize().shape == (0, 64) and empty.parts()[0].shape == (0, 32)


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 33), (130, 96), (128, 256), (17, 255), (300, 1001)])
def test_parts_there_and_back(rows, cols):
    rng = np.random.default_rng(rows + cols)
    codes = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, -(-cols // 32)), dtype=np.uint8)
    packed = ref.pack(codes)
    if cols % 2:
        packed[:, -1] |= 0xF0      # a stray half byte after the last column is not taken over
    ref.poison()
    q = mx4.from_parts(torch.from_numpy(packed).cuda(), torch.from_numpy(scales).cuda(), cols)
    got = [t.cpu().numpy() for t in q.parts()]
    np.testing.assert_array_equal(got[0], ref.pack(codes))
    np.testing.assert_array_equal(got[1], scales)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(ref.to64(q.dequantize(torch.float32)), ref.decode(codes, scales).astype(np.float32))


def test_another_stream():
    x = torch.randn((400, 3000), device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = mx4.quantize(x)
        out = q.dequantize()
    side.synchronize()
    np.testing.assert_array_equal(ref.to64(out), ref.values(q))


def test_refusals():
    x = torch.zeros((4, 64), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mx4.quantize(x.cpu())
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        mx4.quantize(x.to(torch.int32))
    with pytest.raises(ValueError, match="unit stride"):
        mx4.quantize(x.t())
    with pytest.raises(ValueError, match="contiguous"):
        mx4.quantize(x.view(2, 2, 64)[:, :1])
    with pytest.raises(ValueError, match="column"):
        mx4.quantize(x[:, :0])
    with pytest.raises(ValueError, match="Mx4Tensor"):
        mx4.dequantize(x)
    with pytest.raises(ValueError, match="dtype"):
        mx4.quantize(x).dequantize(torch.float64)
    codes, scales = torch.zeros((4, 32), dtype=torch.uint8, device="cuda"), torch.zeros((4, 2), dtype=torch.uint8, device="cuda")
    for bad, match in (((codes, scales, 66), "33 columns"), ((codes, scales[:3], 64), "same rows"), ((codes.cpu(), scales, 64), "CUDA"),
                       ((codes.float(), scales, 64), "uint8"), ((codes.t(), scales, 64), "contiguous"), ((codes, scales, 0), "> 0")):
        with pytest.raises(ValueError, match=match):
            mx4.from_parts(*bad)
