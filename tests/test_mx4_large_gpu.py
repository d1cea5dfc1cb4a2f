"""Matrices beyond 2^31 elements and 2^32 bytes: rows at their end come out as the same rows at their start do."""
import pytest
import torch

from mpserve_b200 import mx4

pytestmark = pytest.mark.gpu

ROWS, COLS = 1_000_003, 8192          # 4.6 GB of tiles, 8.2 G elements


def _room(nbytes: int) -> None:
    if torch.cuda.mem_get_info()[0] < nbytes:
        pytest.skip("not enough free memory on this GPU")


def _some_rows(cols):
    g = torch.Generator(device="cuda").manual_seed(1)
    return torch.randn((1, cols), generator=g, device="cuda").to(torch.bfloat16)


def test_quantize_and_product():
    _room(16 << 30)
    one = _some_rows(COLS)
    q = mx4.quantize(one.expand(ROWS, COLS))
    assert q.data.numel() > 1 << 32
    first = mx4.quantize(one)
    tile_row = (COLS // 256) * 17408
    tail = mx4.Mx4Tensor(q.data[(ROWS - 1) // 128 * tile_row:], (ROWS - 1) % 128 + 1, COLS)
    assert torch.equal(tail.dequantize(), first.dequantize().expand(tail.rows, COLS))
    w = mx4.quantize(torch.randn((24, COLS), device="cuda"))
    y = mx4.linear(q, w)
    assert torch.equal(y[-300:], y[:300]) and torch.equal(y[0], y[ROWS // 2])
    a = mx4.gated_linear(q, w, w)
    assert torch.equal(a[-300:], a[:300])
    del y, a
    # as a weight: so many output columns that an output's row is 2 MB
    out = mx4.linear(one.expand(3, COLS), q)
    assert torch.equal(out[:, -300:], out[:, :300]) and torch.equal(out[2], out[0])


def test_an_output_of_many_elements():
    _room(16 << 30)
    tokens, rows, cols = 70_001, 33_000, 64      # 2.3 G elements, 4.6 GB
    x, w = mx4.quantize(_some_rows(cols).expand(tokens, cols)), mx4.quantize(torch.randn((rows, cols), device="cuda"))
    y = mx4.linear(x, w)
    assert y.numel() > 1 << 31
    assert torch.equal(y[-5], y[0]) and torch.equal(y[tokens // 2], y[0])
    a = mx4.gated_linear(x, w, w, quantized=True)
    small = mx4.gated_linear(mx4.quantize(_some_rows(cols).expand(300, cols)), w, w, quantized=True)
    tile_row = -(-rows // 256) * 17408
    tail = mx4.Mx4Tensor(a.data[(tokens - 1) // 128 * tile_row:], (tokens - 1) % 128 + 1, rows)
    assert torch.equal(tail.dequantize()[0], small.dequantize()[0])


def test_norms():
    _room(40 << 30)
    rows, cols = 1_100_000, 4096                 # 4.5 G elements
    one = _some_rows(cols)
    many = one.expand(rows, cols)
    w = torch.rand(cols, device="cuda")
    n = mx4.rms_norm(many, w)
    assert n.numel() > 1 << 32
    assert torch.equal(n[-7:], n[:7])
    del n
    joined, _ = mx4.block_join(many, many, post_weight=w)
    few, _ = mx4.block_join(many[:600], many[:600], post_weight=w)
    assert torch.equal(joined[-7:], few[:7])
